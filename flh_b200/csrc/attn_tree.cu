// Attention of drafted tokens over a KV cache whose sequences have lengths of their own, and its accumulated weights.
//
//   o[b, s, h] = sum_t p[t] v[b, h / g, t],  p = softmax over the entries t that token s sees of scale * q[b, s, h] . k[b, h / g, t]
//   weights[b, kvh, t] += sum over s and the heads of the group of p[t]
//
// Token s of sequence b sees every committed entry (t < lengths[b]) and, of the drafted ones (t = lengths[b] + j, j < S), those
// whose bit j is set in tree[b, s]; S = 1 is ordinary decode.
//
// A pass reads K and V once: 4 D bytes an entry against 4 R D operations (R = S g rows share a kv head's entries), so that up to a few
// dozen rows the memory is what bounds it.  attn_mma_kernel is built for that: every warp streams key tiles of its own through a ring
// of TMA loads in shared memory, keeps the running maximum and sum of its rows in registers and needs no other warp until its
// share of a job ends (mma.sync: 16 rows by 8 keys by 16 values; the tensor cores are at a fraction of their rate).
//
// The weights of the product with V are rounded to the tensors' type, their sum is of the unrounded ones.  float16 ends at 2^-24, so its
// weights are relative to a reference 2^14 below the maximum: the heaviest is 2^14, and of one that is 2^-26 of it nothing is lost.
// (Relative to the maximum itself 16,384 such entries beside one heavy one vanished from the result.)
#include "attn_common.cuh"
#include "tc_pair.cuh"

namespace flh {

int launch_attn_tc(const TreeAttnParams &, int, bool, const CUtensorMap &, const CUtensorMap &, cudaStream_t);
int launch_attn_weights_tc(const TreeAttnParams &, bool, const CUtensorMap &, cudaStream_t);
int attn_tc_status(int *);
int attn_tc_status_clear();

namespace {

__device__ int g_status_attn[4];

constexpr int kTile = 32;                  // keys of a tile
constexpr int kWarps = 4, kThreadsAttn = kWarps * 32;

constexpr int kRows = 16;                  // of a job
constexpr int kSlots = 3;                  // ring slots of a warp, so that two CTAs fit an SM; a slot is the K or the V part of a tile
template <bool BF16> constexpr int kRaise = BF16 ? 0 : 14;                             // powers of two that the heaviest weight of a product is
template <int D> constexpr int slot_bytes() { return kTile * D * 2; }
template <int D> constexpr int q_pitch() { return D * 2 + 16; }                       // bytes; the 16 keep ldmatrix free of conflicts
template <int D> constexpr int attn_smem() { return 1024 + kWarps * kSlots * slot_bytes<D>() + kRows * q_pitch<D>() + kWarps * 4 * 128 * 4; }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t &a, uint32_t &b, uint32_t &c, uint32_t &d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 rows of 8-byte pieces: where piece (row, 16-byte chunk) of a tile of 128-byte swizzled rows lies
template <int ROWS> __device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
    return (chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// weights += sum over the rows of 2^(score - lse), from the scores that the attention left (few rows: 8 R bytes an entry against
// 2 D for reading K again).  A thread has EACH entries, t0 and every stride-th, and fetches ROWS rows' scores of them together.
template <int ROWS, int EACH>
__device__ __forceinline__ void add_weights(const TreeAttnParams &p, int b, int bh, int len, int n, int t0, int stride, const float *lse) {
    const float *sc = p.scores + (long)bh * p.R * p.score_ld;
    float *w = p.weights + (long)bh * p.T, was[EACH], sum[EACH] = {};
    int at[EACH];                   // entries; behind the last one it stands in
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        at[k] = min(t0 + k * stride, n - 1);
        was[k] = w[at[k]];
    }
    const bool drafted = at[EACH - 1] >= len;                             // some may not be seen by every row
    const int rows = counted_rows(p, b);
    for (int r0 = 0; r0 < rows; r0 += ROWS) {
        float x[ROWS][EACH], l[ROWS];     // fetched together
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = min(r0 + i, p.R - 1);
            l[i] = lse[r];
#pragma unroll
            for (int k = 0; k < EACH; ++k) x[i][k] = sc[r * p.score_ld + at[k]];
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (r0 + i >= rows) break;
            const uint64_t bits = drafted ? drafted_bits(p, b, token_of(p, r0 + i), len) : 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const bool seen = at[k] < len || ((bits >> (at[k] - len)) & 1);
                sum[k] += seen ? exp2_approx(fmaf(x[i][k], p.scale_log2, -l[i])) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k)
        if (t0 + k * stride < n) w[at[k]] = was[k] + sum[k];
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreadsAttn, 2) attn_mma_kernel(const __grid_constant__ TreeAttnParams p, const __grid_constant__ CUtensorMap kmap,
                                                                   const __grid_constant__ CUtensorMap vmap) {
    constexpr int kNT = kTile / 8, kKS = D / 16, kDT = D / 8, kSlot = slot_bytes<D>();
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sm_q = smem + kWarps * kSlots * kSlot;
    float *sm_o = reinterpret_cast<float *>(sm_q + kRows * q_pitch<D>());      // [warp][rows][D], 512 values a warp
    __shared__ uint64_t full[kWarps][kSlots];
    __shared__ uint64_t seen[kRows];
    __shared__ unsigned long long bad;
    __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, quad = lane & 3;
    uint8_t *ring = smem + warp * kSlots * kSlot;
    const uint32_t ring_u = smem_u32(ring), full_u = smem_u32(&full[warp][0]);
    if (lane == 0)
        for (int i = 0; i < kSlots; ++i) mbar_init(full_u + 8 * i, 1);
    if (tid == 0) { abort_flag = 0; bad = 0; }
    fence_proxy_async();
    __syncthreads();
    pdl_wait();
    pdl_trigger();

    JobWalk<kTile> cur, ahead;             // the job worked on, and the one that the loads have come to
    int u0, u1;
    take_share(p, lane, cur, u0, u1);
    if (u0 >= u1) return;
    ahead = cur;

    // item i of this warp: K (i even) or V (i odd) of its tile i / 2, into slot i % kSlots
    int u_ahead = u0 + warp, item = 0;
    auto issue = [&]() {
        if (u_ahead >= u1) return;
        while (u_ahead >= ahead.begin + ahead.nt) ahead.next(p);
        if (lane == 0) {
            const uint32_t bar = full_u + 8 * (item % kSlots), dst = ring_u + (item % kSlots) * kSlot;
            const CUtensorMap *map = item & 1 ? &vmap : &kmap;
            mbar_expect_tx(bar, kSlot);
            for (int h = 0; h < D / 64; ++h)
                tma_load_tile(dst + h * (kTile * 128), map, h * 64, (u_ahead - ahead.begin) * kTile, ahead.b * p.nkv + ahead.job, bar);
        }
        if (item & 1) u_ahead += kWarps;
        ++item;
    };
    for (int i = 0; i < kSlots; ++i) issue();
    const bool few = p.R <= 8;
    int used = 0;                          // items taken from the ring
    bool alive = true;

    // rows of q of a job and what they see of its drafted entries: 16-byte piece q_c of every kQStep-th row, fetched while the job before is finished
    constexpr int kQStep = kThreadsAttn / (D / 8), kQLoads = kRows / kQStep;
    const int q_c = tid % (D / 8), q_r = tid / (D / 8);
    uint4 qv[kQLoads];
    uint64_t bits = 0;
    auto fetch_q = [&](const JobWalk<kTile> &j) {
#pragma unroll
        for (int i = 0; i < kQLoads; ++i) {
            const int row = q_r + i * kQStep;
            qv[i] = row < p.R ? ldg_v4(static_cast<const uint16_t *>(p.q) + q_offset(p, j.b, j.job, row) + q_c * 8) : make_uint4(0, 0, 0, 0);
        }
        if (tid < p.R) bits = tree_bits(p, j.b, token_of(p, tid));
    };
    fetch_q(cur);
    for (int piece = u0; piece < u1;) {
        const int piece_end = min(u1, cur.begin + cur.nt);
        const int b = cur.b, kvh = cur.job, len = cur.len, n = entries(p, len);                // one block of rows a job
        __syncthreads();                   // the piece before is written out
#pragma unroll
        for (int i = 0; i < kQLoads; ++i) *reinterpret_cast<uint4 *>(sm_q + (q_r + i * kQStep) * q_pitch<D>() + q_c * 16) = qv[i];
        if (tid < kRows) seen[tid] = tid < p.R ? bits & existing_bits(p, len) : 0;
        if (tid == 0) bad = 0;
        __syncthreads();
        float o[kDT][4], m[2], l[2];
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < kDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        int u = piece + ((u0 + warp - piece) % kWarps + kWarps) % kWarps;
        for (; u < piece_end && alive; u += kWarps) {
            const int key0 = (u - cur.begin) * kTile;
            // scores: 16 rows by 32 keys
            float sc[kNT][4];
#pragma unroll
            for (int i = 0; i < kNT; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.0f;
            int slot = used % kSlots;
            alive = mbar_wait_warp(g_status_attn, full_u + 8 * slot, (used / kSlots) & 1, &abort_flag, 31);
            if (!alive) break;
            const uint32_t ks = ring_u + slot * kSlot;
#pragma unroll
            for (int k2 = 0; k2 < kKS / 2; ++k2) {                              // 32 values of the heads at a time
                uint32_t a[8];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
                    ldsm4(smem_u32(sm_q) + (lane & 15) * q_pitch<D>() + (k2 * 4 + hh * 2 + (lane >> 4)) * 16,
                          a[4 * hh], a[4 * hh + 1], a[4 * hh + 2], a[4 * hh + 3]);
#pragma unroll
                for (int i = 0; i < kNT; ++i) {
                    uint32_t b0, b1, b2, b3;
                    ldsm4(ks + swizzled<kTile>(i * 8 + (lane & 7), k2 * 4 + (lane >> 3)), b0, b1, b2, b3);
                    mma16816<BF16>(sc[i], a[0], a[1], a[2], a[3], b0, b1);
                    mma16816<BF16>(sc[i], a[4], a[5], a[6], a[7], b2, b3);
                }
            }
            __syncwarp();
            ++used;
            issue();
            const bool tail = key0 + kTile > len;                              // drafted entries, or none at all, in this tile
            if (tail) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    // a bit for each of the 32 entries: committed, or drafted and seen
                    const uint64_t bits = seen[grp + hh * 8];
                    const int j0 = key0 - len;
                    const uint32_t vis = (j0 >= 64 ? 0u : j0 >= 0 ? (uint32_t)(bits >> j0) : ((uint32_t)bits << -j0) | ((1u << -j0) - 1)) >> (quad * 2);
#pragma unroll
                    for (int i = 0; i < kNT; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            if (!((vis >> (i * 8 + e)) & 1)) sc[i][2 * hh + e] = -INFINITY;
                }
            }
            if (p.scores) {
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const int row = grp + hh * 8;
                    if (row < p.R) {
                        float *dst = p.scores + (((long)b * p.nkv + kvh) * p.R + row) * p.score_ld + key0 + quad * 2;
#pragma unroll
                        for (int i = 0; i < kNT; ++i)
                            *reinterpret_cast<float2 *>(dst + i * 8) = make_float2(sc[i][2 * hh], sc[i][2 * hh + 1]);
                    }
                }
            }
            // running maximum and sum; the sum is of the exponentials in binary32, before they are rounded for the product
            uint32_t pr[kNT][2] = {};
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                if (hh && few) break;                                            // rows 8 and up do not exist
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < kNT; ++i) mx = fmaxf(mx, fmaxf(sc[i][2 * hh], sc[i][2 * hh + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = reference_of<kRaise<BF16>>(mx * p.scale_log2);          // scale > 0
                const float was = m[hh], now = fmaxf(was, mx), base = now == -INFINITY ? 0.0f : now;
                m[hh] = now;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < kNT; ++i) {
                    const float x = exp2_approx(fmaf(sc[i][2 * hh], p.scale_log2, -base)), y = exp2_approx(fmaf(sc[i][2 * hh + 1], p.scale_log2, -base));
                    sum += x + y;
                    pr[i][hh] = narrow<BF16>(x, y);
                }
                const float keep = exp2_approx(was - base);
                l[hh] = l[hh] * keep + sum;
                if (__any_sync(0xffffffffu, now != was)) {
#pragma unroll
                    for (int i = 0; i < kDT; ++i) { o[i][2 * hh] *= keep; o[i][2 * hh + 1] *= keep; }
                }
            }
            slot = used % kSlots;
            alive = mbar_wait_warp(g_status_attn, full_u + 8 * slot, (used / kSlots) & 1, &abort_flag, 32);
            if (!alive) break;
            const uint32_t vs = ring_u + slot * kSlot;
            if (tail) {
                // values that are not finite become zero, of drafted entries and of what lies behind the sequence's end
                const int row = max(len - key0, 0) + lane / (D / 8), chunk = lane % (D / 8);      // the rows behind the committed ones
#pragma unroll 4
                for (int r = row; r < kTile; r += 32 / (D / 8)) {
                    uint4 *at = reinterpret_cast<uint4 *>(ring + slot * kSlot + swizzled<kTile>(r, chunk));
                    const uint4 x = *at;
                    if (any_nonfinite<BF16>(x)) {
                        if (key0 + r < n) atomicOr(&bad, 1ull << (key0 + r - len));
                        *at = make_uint4(finite2<BF16>(x.x), finite2<BF16>(x.y), finite2<BF16>(x.z), finite2<BF16>(x.w));
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) {
#pragma unroll
                for (int i = 0; i < kDT; i += 2) {
                    uint32_t b0, b1, b2, b3;
                    ldsm4t(vs + swizzled<kTile>(k * 16 + (lane & 15), i + (lane >> 4)), b0, b1, b2, b3);
                    mma16816<BF16>(o[i], pr[2 * k][0], pr[2 * k][1], pr[2 * k + 1][0], pr[2 * k + 1][1], b0, b1);
                    mma16816<BF16>(o[i + 1], pr[2 * k][0], pr[2 * k][1], pr[2 * k + 1][0], pr[2 * k + 1][1], b2, b3);
                }
            }
            if (tail) fence_proxy_async();                                      // the slot was written here: TMA writes it next
            __syncwarp();
            ++used;
            issue();
        }
        // the warps' results, each relative to its own maximum, become one
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            float sum = l[hh];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (quad == 0) { sm_m[warp][grp + hh * 8] = m[hh]; sm_l[warp][grp + hh * 8] = sum; }
        }
        __syncthreads();
        // a row's factors: of every warp, and of the sum
        if (tid < kRows) {
            float top = sm_m[0][tid], sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_m[w][tid]);
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = exp2_approx(sm_m[w][tid] - base);
                sum += sm_l[w][tid] * f;
                sm_m[w][tid] = f;
            }
            const bool whole_job = piece == cur.begin && piece_end == cur.begin + cur.nt;
            sm_l[0][tid] = whole_job ? row_factor(sum, len == 0 && !seen[tid]) : 1.0f;
            sm_l[1][tid] = base;
            sm_l[2][tid] = base + log2f(sum);
            if (tid < p.R) {
                if (!whole_job) p.part_ml[(2L * blockIdx.x + (piece != u0)) * kRows + tid] = make_float2(top, sum);
                else if (p.lse) p.lse[((long)b * p.nkv + kvh) * p.R + tid] = sm_l[2][tid];
            }
        }
        JobWalk<kTile> next = cur;
        if (piece_end < u1) {
            next.next(p);
            fetch_q(next);
        }
        __syncthreads();
        const float mine[2] = {sm_m[warp][grp], sm_m[warp][grp + 8]};
        const bool whole = piece == cur.begin && piece_end == cur.begin + cur.nt;
        const long part = 2L * blockIdx.x + (piece != u0);
        constexpr int kChunk = 4 * 128 / D;                                      // rows whose sums of all warps fit the buffer (8 KB)
#pragma unroll
        for (int r0 = 0; r0 < kRows; r0 += kChunk) {
            if (r0 >= p.R) break;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int r = hh * 8 + grp;
                if (r / kChunk == r0 / kChunk) {
#pragma unroll
                    for (int i = 0; i < kDT; ++i)
                        *reinterpret_cast<float2 *>(sm_o + (warp * kChunk + r - r0) * D + i * 8 + quad * 2) = make_float2(o[i][2 * hh] * mine[hh], o[i][2 * hh + 1] * mine[hh]);
                }
            }
            __syncthreads();
            // a thread has four columns of a row
            const int r = r0 + tid / (D / 4), d = tid % (D / 4) * 4;
            if (r < p.R) {
                float4 acc = *reinterpret_cast<const float4 *>(sm_o + (r - r0) * D + d);
#pragma unroll
                for (int w = 1; w < kWarps; ++w) {
                    const float4 v = *reinterpret_cast<const float4 *>(sm_o + (w * kChunk + r - r0) * D + d);
                    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
                }
                if (bad) {
                    const float base = sm_l[1][r];
                    acc.x += nonfinite_part<BF16>(p, bad, seen[r], b, kvh, r, d, len, base);
                    acc.y += nonfinite_part<BF16>(p, bad, seen[r], b, kvh, r, d + 1, len, base);
                    acc.z += nonfinite_part<BF16>(p, bad, seen[r], b, kvh, r, d + 2, len, base);
                    acc.w += nonfinite_part<BF16>(p, bad, seen[r], b, kvh, r, d + 3, len, base);
                }
                if (whole) {
                    const float f = sm_l[0][r];
                    const int s = token_of(p, r), h = kvh * p.g + r - s * p.g;
                    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + (((long)b * p.S + s) * p.nh + h) * D + d) =
                        make_uint2(narrow<BF16>(acc.x * f, acc.y * f), narrow<BF16>(acc.z * f, acc.w * f));
                } else {
                    *reinterpret_cast<float4 *>(p.part_o + part * kRows * D + d * kRows + r * 4) = acc;
                }
            }
            if (r0 + kChunk < kRows) __syncthreads();
        }
        // no job is cut: what its rows gave its entries is added here (16 sequences of 766 .. 1,531: 51 us without weights, 55 with, 59 as a launch of its own)
        if (p.scores && p.split == kJobs)
            for (int t0 = tid; t0 < n; t0 += (p.R == 1 ? 12 : 4) * kThreadsAttn) {
                if (p.R == 1) add_weights<1, 12>(p, b, b * p.nkv + kvh, len, n, t0, kThreadsAttn, sm_l[2]);
                else add_weights<4, 4>(p, b, b * p.nkv + kvh, len, n, t0, kThreadsAttn, sm_l[2]);
            }
        piece = piece_end;
        cur = next;
    }
    if (!alive)                            // a wait ran out: what is still on its way lands before the CTA leaves
        for (int i = used; i < item; ++i)
            for (int tries = 0; tries < 10000 && !__all_sync(0xffffffffu, mbar_try_hint(full_u + 8 * (i % kSlots), (i / kSlots) & 1, 20000u)); ++tries);
}

// Jobs that several CTAs hold: their partial results in order.  A block for each job, or (kEven) for each cut between two shares where that
// is fewer: it takes the job that is cut there, if that is the job's first cut.  A thread has four columns of a row, the 8 rows next
// to one another in a warp so that it reads whole lines.
//
// CTAs c0 .. c0 + parts - 1 have the job; the first of them may have begun with another one (behind).
template <int TILE>
__device__ __forceinline__ bool find_parts(const TreeAttnParams &p, int lane, int by_job, int &b, int &job_of, int &c0, int &parts, bool &behind) {
    behind = false;
    if (p.split == kParts) {
        const int per = p.nkv * p.nrb;
        const int2 t = p.parts_of[blockIdx.x];
        b = blockIdx.x / per;
        job_of = blockIdx.x - b * per;
        c0 = t.x & ~kBehind;
        parts = t.y;
        behind = (t.x & kBehind) != 0;
        return parts > 1;
    }
    const int total = tiles_before<TILE>(p, p.B, lane), share = share_tiles(p, total);
    JobWalk<TILE> job;
    if (by_job) {
        job.at(p, blockIdx.x, lane);
    } else {
        const long cut = (blockIdx.x + 1L) * share;
        if (cut >= total) return false;
        job.seek(p, (int)cut, lane);
        if (job.begin == cut || job.begin / share != (int)blockIdx.x) return false;
    }
    b = job.b;
    job_of = job.job;
    c0 = job.begin / share;
    parts = (job.begin + job.nt - 1) / share - c0 + 1;
    behind = (long)c0 * share != job.begin;
    return parts > 1;
}
template <int D, bool BF16>
__device__ __forceinline__ void store_joined(const TreeAttnParams &p, int b, int kvh, int row, int group, float base, float sum, float4 acc) {
    const int s = token_of(p, row), h = kvh * p.g + row - s * p.g;
    float factor = 1.0f / sum;
    if (sum == 0.0f) {
        const int len = committed(p, b);
        factor = row_factor(sum, len == 0 && !drafted_bits(p, b, s, len));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + (((long)b * p.S + s) * p.nh + h) * D + group * 4) =
        make_uint2(narrow<BF16>(acc.x * factor, acc.y * factor), narrow<BF16>(acc.z * factor, acc.w * factor));
    if (group == 0 && p.lse) p.lse[((long)b * p.nkv + kvh) * p.R + row] = base + log2f(sum);
}

// A block has 1,024 / D rows and all columns.  Eight parts and their maxima and sums are fetched together, so that up to eight cost one
// wait for memory; where there are more the sum goes on relative to the larger maximum.
template <int D, int TILE, bool BF16>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ TreeAttnParams p, int by_job) {
    constexpr int kRowsOf = 1024 / D, kAhead = 8;
    const int tid = threadIdx.x, r = blockIdx.y * kRowsOf + tid % kRowsOf, group = tid / kRowsOf;
    pdl_wait();
    pdl_trigger();
    int b, job, c0, parts;
    bool behind;
    if (!find_parts<TILE>(p, tid & 31, by_job, b, job, c0, parts, behind)) return;
    const int kvh = job / p.nrb, row = (job - kvh * p.nrb) * p.rows + r;
    if (r >= p.rows || row >= p.R) return;
    float top = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0, 0, 0, 0);
    for (int i0 = 0; i0 < parts; i0 += kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = min(i0 + k, parts - 1);
            const long slot = 2L * (c0 + i) + (i == 0 && behind);
            ml[k] = p.part_ml[slot * p.rows + r];
            v[k] = *reinterpret_cast<const float4 *>(p.part_o + slot * p.rows * D + ((long)group * p.rows + r) * 4);
        }
        float now = top;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) now = fmaxf(now, ml[k].x);
        const float base = now == -INFINITY ? 0.0f : now, keep = exp2_approx(top - base);
        sum *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (i0 + k >= parts) continue;
            const float f = exp2_approx(ml[k].x - base);
            sum += ml[k].y * f;
            acc.x += v[k].x * f; acc.y += v[k].y * f; acc.z += v[k].z * f; acc.w += v[k].w * f;
        }
        top = now;
    }
    store_joined<D, BF16>(p, b, kvh, row, group, top == -INFINITY ? 0.0f : top, sum, acc);
}

// Few jobs in many parts: a block for 8 rows and 32 columns, with 16 sets of threads that share out the parts; the parts' factors come
// first, each from one thread (one sequence of 60,000 entries, 8 rows, in 268 parts: 59 -> 19 us with its attention).
constexpr int kJoinRows = 8, kMaxParts = 2 * kNumSMs;
template <int D, int TILE, bool BF16>
__global__ void __launch_bounds__(1024) attn_join_wide_kernel(const __grid_constant__ TreeAttnParams p, int by_job) {
    constexpr int GROUPS = 8, WAYS = 16;
    __shared__ float factor_of[kMaxParts][kJoinRows], reduced[GROUPS * WAYS / 4][kJoinRows];
    __shared__ float4 sm_acc[WAYS][8 * GROUPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, way = tid / (8 * GROUPS);
    const int r_in = tid & 7, r = blockIdx.y * kJoinRows + r_in, group = blockIdx.z * GROUPS + (tid >> 3) % GROUPS;
    pdl_wait();
    pdl_trigger();
    int b, job, c0, parts;
    bool behind;
    if (!find_parts<TILE>(p, lane, by_job, b, job, c0, parts, behind)) return;
    const int kvh = job / p.nrb, row = (job - kvh * p.nrb) * p.rows + r;
    const bool live = r < p.rows && row < p.R;
    auto slot = [&](int i) { return 2L * (c0 + i) + (i == 0 && behind); };
    // a row's values in lanes 8 apart, then over the warps
    auto over_block = [&](float x, bool max) {
        for (int o = 8; o < 32; o <<= 1) { const float y = __shfl_xor_sync(0xffffffffu, x, o); x = max ? fmaxf(x, y) : x + y; }
        if (lane < 8) reduced[warp][lane] = x;
        __syncthreads();
        x = reduced[0][r_in];
#pragma unroll
        for (int w = 1; w < GROUPS * WAYS / 4; ++w) x = max ? fmaxf(x, reduced[w][r_in]) : x + reduced[w][r_in];
        __syncthreads();
        return x;
    };
    // a thread for every kThreads-th part of a row
    constexpr int kThreads = GROUPS * WAYS, kEach = (kMaxParts + kThreads - 1) / kThreads;
    float2 ml[kEach];
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int i = (tid >> 3) + k * kThreads;
        ml[k] = live && i < parts ? p.part_ml[slot(i) * p.rows + r] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[k].x);
    }
    top = over_block(top, true);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int i = (tid >> 3) + k * kThreads;
        const float f = exp2_approx(ml[k].x - base);
        if (i < parts) factor_of[i][r_in] = f;
        sum += ml[k].y * f;
    }
    sum = over_block(sum, false);
    float4 acc = make_float4(0, 0, 0, 0);
    if (live) {
#pragma unroll 8
        for (int i = way; i < parts; i += WAYS) {
            const float4 v = *reinterpret_cast<const float4 *>(p.part_o + slot(i) * p.rows * D + ((long)group * p.rows + r) * 4);
            const float f = factor_of[i][r_in];
            acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        }
    }
    sm_acc[way][tid % (8 * GROUPS)] = acc;
    __syncthreads();
    if (way || !live) return;
#pragma unroll
    for (int w = 1; w < WAYS; ++w) { const float4 v = sm_acc[w][tid]; acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w; }
    store_joined<D, BF16>(p, b, kvh, row, group, base, sum, acc);
}

// The same where jobs were cut: a launch behind the join.
constexpr int kWeightThreads = 256, kWeightEach = 4;
__global__ void __launch_bounds__(kWeightThreads) attn_weights_kernel(const __grid_constant__ TreeAttnParams p) {
    const int bh = blockIdx.x, t0 = blockIdx.y * kWeightThreads * kWeightEach + threadIdx.x;
    pdl_wait();
    pdl_trigger();
    const int b = bh / p.nkv, len = committed(p, b), n = entries(p, len);
    if (t0 < n) add_weights<4, kWeightEach>(p, b, bh, len, n, t0, kWeightThreads, p.lse + (long)bh * p.R);
}

// ---- host side ------------------------------------------------------------------------------
struct Plan {
    int rows, nrb, shares, min_share;
    int split, jobs_each;
    bool scores;
    long score_ld;
    size_t part_o, part_ml, parts_of, lse, sc, total;        // offsets in the workspace
};
Plan plan_of(int B, int S, int nh, int nkv, int D, long T, bool weights) {
    Plan pl = {};
    const int R = S * (nh / nkv);
    pl.rows = R <= 16 ? 16 : R <= 128 ? 128 : 256;
    pl.nrb = (R + pl.rows - 1) / pl.rows;
    pl.shares = pl.rows >= 128 ? kNumSMs : 2 * kNumSMs;
    pl.min_share = pl.rows >= 128 ? 2 : kWarps;
    // Whole jobs where what that makes the fullest CTA work more than an even share is little, if the sequences are about as long as one another:
    // what is saved is the join and, for most CTAs, a second piece (kSecondJob tiles; one sequence of 500 entries, 32 heads: 13.7 -> 10.1
    // us; 24 sequences of 40: 31 -> 20; 4 of 2,478 .. 4,000, 32 heads of 64 rows: 57 -> 50).  The lengths are not known here: a CTA has at most
    // `most` tiles whatever they are, so that one long sequence among short ones costs little even then (8 rows, 16 sequences: 1,531 entries
    // and 15 of 20 33 us, 30 if cut; 40 rows, 18 sequences: 2,000 and 17 of 100 27 us, 18 if cut).  Else parts of the jobs, where that is
    // worked out quickly.
    const bool tc = pl.rows >= 128;
    const long jobs = (long)B * nkv * pl.nrb, tile = tc ? kTreeTcTile : kTile, nt = (T + tile - 1) / tile, each = (jobs + pl.shares - 1) / pl.shares;
    const long over = each * nt - jobs * nt / pl.shares, most = tc ? 72 : 128;
    pl.split = over <= (tc ? kSecondJob<kTreeTcTile> : kSecondJob<kTile>) && each * nt <= most ? kJobs : jobs <= pl.shares && B <= 32 ? kParts : kEven;
    pl.jobs_each = (int)each;
    if (pl.split == kJobs) pl.shares = (int)((jobs + each - 1) / each);
    pl.scores = weights && R <= 16;
    pl.score_ld = (T + kTile - 1) / kTile * kTile;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    const size_t slots = pl.split == kJobs ? 0 : (size_t)2 * pl.shares * pl.rows;
    pl.part_o = take(slots * D * 4);
    pl.part_ml = take(slots * 8);
    pl.parts_of = take((size_t)pl.shares * 8);
    pl.lse = take(weights ? (size_t)B * nkv * R * 4 : 0);
    pl.sc = take(pl.scores ? (size_t)B * nkv * R * pl.score_ld * 4 : 0);
    pl.total = at;
    return pl;
}

int make_map(CUtensorMap *map, const void *base, bool bf16, int D, long T, long heads, int rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(FLH_B200_EUNSUPPORTED, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)heads};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)T * D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1}, step[3] = {1, 1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : fail(FLH_B200_EINVAL, "the cache cannot be described to TMA (%d)", (int)r);
}

template <int D, bool BF16>
int launch_mma(const TreeAttnParams &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t stream) {
    auto kern = attn_mma_kernel<D, BF16>;
    constexpr int smem = attn_smem<D>();
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kern), smem, done);
    if (e != cudaSuccess) return cuda_status(e, "tree_attention shared memory");
    return cuda_status(launch_pdl(kern, dim3((unsigned)p.shares), kThreadsAttn, smem, stream, p, km, vm), "tree_attention launch");
}

template <int D, bool BF16>
int launch_attention(const TreeAttnParams &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t stream) {
    const unsigned heads = (unsigned)(p.B * p.nkv);
    const bool tc = p.rows >= 128;
    int rc = tc ? launch_attn_tc(p, p.rows, BF16, km, vm, stream) : launch_mma<D, BF16>(p, km, vm, stream);
    if (rc) return rc;
    const long jobs = (long)heads * p.nrb;
    if (p.split != kJobs) {
        const bool each = p.split == kParts || jobs < p.shares, wide = jobs * 16 <= p.shares;           // a block per job; 16 parts a job and more
        const int rows = p.R < p.rows ? p.R : p.rows, of = wide ? kJoinRows : 1024 / D;
        const dim3 grid(each ? (unsigned)jobs : (unsigned)p.shares - 1, (unsigned)((rows + of - 1) / of), wide ? D / 32 : 1);
        auto join = tc ? (wide ? attn_join_wide_kernel<D, kTreeTcTile, BF16> : attn_join_kernel<D, kTreeTcTile, BF16>)
                       : (wide ? attn_join_wide_kernel<D, kTile, BF16> : attn_join_kernel<D, kTile, BF16>);
        rc = cuda_status(launch_pdl(join, grid, wide ? 1024 : 256, 0, stream, p, (int)each), "tree_attention join");
    }
    if (rc || !p.weights || (p.scores && p.split == kJobs)) return rc;
    if (p.scores) {
        const int each = kWeightThreads * kWeightEach;
        return cuda_status(launch_pdl(attn_weights_kernel, dim3(heads, (unsigned)((p.T + each - 1) / each)), kWeightThreads, 0, stream, p), "tree_attention weights");
    }
    return launch_attn_weights_tc(p, BF16, km, stream);
}

}  // namespace

size_t tree_attention_workspace_bytes(int B, int S, int nh, int nkv, int D, long T, bool weights) { return plan_of(B, S, nh, nkv, D, T, weights).total; }

int launch_tree_attention(TreeAttnParams p, bool bf16, uint8_t *ws, cudaStream_t stream) {
    const Plan pl = plan_of(p.B, p.S, p.nh, p.nkv, p.D, p.T, p.weights != nullptr);
    p.g = p.nh / p.nkv;
    p.g_inverse = p.g > 1 ? (uint32_t)(((1ull << 32) + p.g - 1) / p.g) : 0;
    p.R = p.S * p.g;
    p.nrb = pl.nrb;
    p.rows = pl.rows;
    p.shares = pl.shares;
    p.min_share = pl.min_share;
    p.split = pl.split;
    p.jobs_each = pl.jobs_each;
    p.part_o = reinterpret_cast<float *>(ws + pl.part_o);
    p.part_ml = reinterpret_cast<float2 *>(ws + pl.part_ml);
    p.parts_of = reinterpret_cast<int2 *>(ws + pl.parts_of);
    p.lse = p.weights ? reinterpret_cast<float *>(ws + pl.lse) : nullptr;
    p.scores = pl.scores ? reinterpret_cast<float *>(ws + pl.sc) : nullptr;
    p.score_ld = pl.score_ld;
    CUtensorMap km, vm;
    const int tile = pl.rows >= 128 ? kTreeTcTile : kTile;
    int rc = make_map(&km, p.k, bf16, p.D, p.T, (long)p.B * p.nkv, tile);
    if (!rc) rc = make_map(&vm, p.v, bf16, p.D, p.T, (long)p.B * p.nkv, tile);
    if (rc) return rc;
    if (p.D == 128) return bf16 ? launch_attention<128, true>(p, km, vm, stream) : launch_attention<128, false>(p, km, vm, stream);
    return bf16 ? launch_attention<64, true>(p, km, vm, stream) : launch_attention<64, false>(p, km, vm, stream);
}

int attn_tree_status(int *out) {
    const int rc = attn_tc_status(out);
    return rc || out[0] ? rc : cuda_status(cudaMemcpyFromSymbol(out, g_status_attn, sizeof(int) * 4), "attn_tree_status");
}
int attn_tree_status_clear() {
    const int zero[4] = {};
    const int rc = attn_tc_status_clear();
    return rc ? rc : cuda_status(cudaMemcpyToSymbol(g_status_attn, zero, sizeof(zero)), "attn_tree_status");
}

}  // namespace flh
