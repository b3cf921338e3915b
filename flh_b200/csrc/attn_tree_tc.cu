// The attention of attn_tree.cu on the 5th-generation tensor cores, for jobs of many rows: S drafted tokens times the g query heads of a
// kv head are R rows over the same entries, and from a few dozen on the products, not the memory, are what a pass waits for.
//
// A CTA per SM.  One warp loads key tiles (128 entries) of K and V by TMA into a ring, one issues the MMAs, two groups of four warps
// have the softmax of one stream each, a thread per row.  A stream is a block of 128 rows with a tile of scores S and an accumulator
// O in tensor memory:
//   S = Q K^T        both operands in shared memory, K as it lies there
//   P = 2^(S - m)    read from tensor memory, rounded to 16 bits (half a step of each weight; their sum is of the unrounded ones) and
//                    written over S
//   O += P V         P from tensor memory, V from shared memory as it lies there, read along the entries
// While the threads of one stream work on their scores the tensor cores multiply for the other.  With more than 128 rows the two
// streams are two blocks of rows that share every tile (half the shared-memory traffic and half the reads of K and V); with up to 128
// they are the same rows over every other tile, and their results become one at the end of a piece, straight from tensor memory.
//
// The running maximum that the exponentials are relative to follows the true one only when that is 2^8 ahead: O is then read, scaled
// and written back.  P reaches 2^8 at most, far from the end of float16.
#include "attn_common.cuh"
#include "tc_pair.cuh"
#include "tc_quant_common.cuh"

namespace flh {
namespace {

__device__ int g_status_attn_tc[4];

constexpr int kTileTc = 128, kRowsTc = 128;
constexpr int kThreadsTcA = 384;           // warp 0 TMA, warp 1 MMA, warps 4 - 7 and 8 - 11 the two streams
// registers: 384 threads are launched with 168; 128 * 88 + 256 * 208 are the same 64,512
constexpr int kRegsIssue = 88, kRegsSoftmax = 208;
static_assert(128 * kRegsIssue + 256 * kRegsSoftmax <= kThreadsTcA * 168, "more registers than the CTA was launched with");
constexpr float kLag = 8.0f;               // powers of two that the true maximum may be ahead

template <int D> constexpr int item_bytes() { return kTileTc * D * 2; }                         // K or V of a tile, and a block of rows of Q
template <int D> constexpr int items_tc() { return D == 64 ? 10 : 5; }
template <int D, bool TWO> constexpr int smem_tc() { return 1024 + (items_tc<D>() + (TWO ? 2 : 1)) * item_bytes<D>(); }

template <bool A_TMEM>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    if (A_TMEM)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                     ::"r"(d), "r"((uint32_t)a), "l"(b), "r"(idesc), "r"(accum) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                   "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// TWO: the streams are two blocks of rows; otherwise they share one.
template <int D, bool TWO, bool BF16>
__global__ void __launch_bounds__(kThreadsTcA, 1) attn_tc_kernel(const __grid_constant__ TreeAttnParams p, const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap vmap) {
    constexpr int kItem = item_bytes<D>(), kItems = items_tc<D>(), kHalf = kTileTc * 128, kJobRows = TWO ? 2 * kRowsTc : kRowsTc;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sm_q = smem + kItems * kItem;
    __shared__ uint64_t full[kItems], empty[kItems], s_full[2], p_full[2], o_full[2], q_full[2];
    __shared__ float2 sm_ml[2][TWO ? 1 : kRowsTc];
    __shared__ unsigned long long bad;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kItems; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&s_full[i]), 1); mbar_init(smem_u32(&p_full[i]), 4); mbar_init(smem_u32(&o_full[i]), 1); mbar_init(smem_u32(&q_full[i]), 4); }
        abort_flag = 0;
        bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_trigger();

    const int total = tiles_before<kTileTc>(p, p.B, lane), share = share_tiles(p, total);
    const long first = (long)blockIdx.x * share;
    const int u0 = (int)min(first, (long)total), u1 = (int)min((long)total, first + share);
    bool ok = true;
    auto wait = [&](uint64_t *bar, int phase, int code) {
        if (ok) ok = mbar_wait_warp(g_status_attn_tc, smem_u32(bar), phase & 1, &abort_flag, code);
        return ok;
    };
    JobWalk<kTileTc> job;
    if (u0 < u1) job.seek(p, u0, lane);

    // Items 2 i and 2 i + 1 of the ring are K and V of the CTA's tile u0 + i, at slot item % kItems.
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == 0) {
        // ---------------------------------------------------------------------- loads
        int item = 0;
        for (int u = u0; u < u1 && ok; ++u) {
            while (u >= job.begin + job.nt) job.next(p);
            const int head = job.b * p.nkv + job.job / p.nrb, key0 = (u - job.begin) * kTileTc;
            for (int kv = 0; kv < 2 && ok; ++kv, ++item) {
                const int slot = item % kItems;
                if (item >= kItems) wait(&empty[slot], item / kItems - 1, 41);
                if (ok && elect_one()) {
                    const uint32_t bar = smem_u32(&full[slot]), dst = smem_u32(smem + slot * kItem);
                    mbar_expect_tx(bar, kItem);
                    for (int h = 0; h < D / 64; ++h)
                        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                                     ::"r"(dst + h * kHalf), "l"(kv ? &vmap : &kmap), "r"(h * 64), "r"(key0), "r"(head), "r"(bar) : "memory");
                }
                __syncwarp();
            }
        }
        // what is still in flight lands before the CTA leaves (after a wait that ran out; otherwise all of it was used)
        for (int i = max(0, item - kItems); i < item; ++i)
            for (int tries = 0; tries < 10000 && !__all_sync(0xffffffffu, mbar_try_hint(smem_u32(&full[i % kItems]), (i / kItems) & 1, 20000u)); ++tries);
    } else if (warp == 1) {
        // ---------------------------------------------------------------------- products
        const uint32_t fmt = BF16 ? 1u : 0u, base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTc >> 4) << 24);
        const uint32_t id_qk = base | ((uint32_t)(kTileTc >> 3) << 17), id_pv = base | (1u << 16) | ((uint32_t)(D >> 3) << 17);
        // slots and phases of the next K and the next V of the ring; phases of the streams' barriers, a bit each
        uint32_t ks = 0, kph = 0, vs = 1, vph = 0, qph = 0, pph = 0;
        const uint32_t ring = uniform(smem_u32(smem)), qbase = uniform(smem_u32(sm_q)), tm = uniform(tmem);
        const uint32_t fulls = smem_u32(full), empties = smem_u32(empty);
        auto wait_u = [&](uint32_t bar, uint32_t phase, int code) {
            if (ok) ok = mbar_wait_warp(g_status_attn_tc, bar, phase, &abort_flag, code);
            return ok;
        };
        for (int piece = u0; piece < u1 && ok;) {
            while (piece >= job.begin + job.nt) job.next(p);
            const int end = min(u1, job.begin + job.nt), tiles = end - piece;
            const bool second = !TWO || (job.job % p.nrb) * kJobRows + kRowsTc < p.R;
            const int live = second ? 2 : 1, steps = TWO ? tiles * live : tiles;
            // stream x: step parity where there are two
            auto qk = [&](uint32_t x) {
                if (!wait_u(fulls + 8 * ks, kph, 42)) return;
                tc_fence_after();
                const uint64_t a = make_smem_desc(qbase + (TWO ? x * kItem : 0)), b = make_smem_desc(ring + ks * kItem);
                const uint32_t d = tm + x * 128;
                const bool free = !TWO || x == (uint32_t)live - 1;
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint64_t off = ((s >> 2) * kHalf + (s & 3) * 32) >> 4;
                        mma_f16<false>(d, a + off, b + off, id_qk, s > 0);
                    }
                    tc_commit(smem_u32(&s_full[0]) + 8 * x);
                    if (free) tc_commit(empties + 8 * ks);
                }
                __syncwarp();
                if (free) { ks += 2; if (ks >= kItems) { ks -= kItems; kph ^= 1; } }
            };
            for (int x = 0; x < 2; ++x) wait_u(smem_u32(&q_full[x]), qph, 43);
            qph ^= 1;
            tc_fence_after();
            uint32_t begun = 0;                                                  // streams that have a sum in this piece, a bit each
            for (int k = 0; k < min(live, steps) && ok; ++k) qk(second ? k & 1 : 0);
            for (int k = 0; k < steps && ok; ++k) {
                const uint32_t x = second ? k & 1 : 0;
                if (!wait_u(smem_u32(&p_full[0]) + 8 * x, (pph >> x) & 1, 44) || !wait_u(fulls + 8 * vs, vph, 45)) break;
                tc_fence_after();
                const bool last = k + live >= steps, free = !TWO || x == (uint32_t)live - 1;
                const uint64_t b = umma_desc_tc(ring + vs * kItem, kHalf, 1024);
                const uint32_t d = tm + 256 + x * 128, a = tm + x * 128, more = (begun >> x) & 1;
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < kTileTc / 16; ++s) mma_f16<true>(d, a + s * 8, b + ((s * 2048) >> 4), id_pv, s > 0 ? 1 : more);
                    if (free) tc_commit(empties + 8 * vs);
                    if (last) tc_commit(smem_u32(&o_full[0]) + 8 * x);
                }
                __syncwarp();
                begun |= 1u << x;
                pph ^= 1u << x;
                if (free) { vs += 2; if (vs >= kItems) { vs -= kItems; vph ^= 1; } }
                if (!last) qk(x);
            }
            piece = end;
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ---------------------------------------------------------------------- softmax
        const int x = (warp >> 2) - 1, quarter = warp & 3, r = quarter * 32 + lane, wg = tid - 128 - x * 128;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, ts = tmem + x * 128 + lanes;
        int sn = 0, on[2] = {0, 0};
        for (int piece = u0; piece < u1;) {
            while (piece >= job.begin + job.nt) job.next(p);
            const int end = min(u1, job.begin + job.nt), tiles = end - piece;
            const int b = job.b, kvh = job.job / p.nrb, row0 = (job.job - kvh * p.nrb) * kJobRows, len = job.len, n = entries(p, len);
            const bool whole = piece == job.begin && end == job.begin + job.nt;
            const int myrow0 = row0 + (TWO ? x * kRowsTc : 0), row = myrow0 + r;
            const bool warp_live = myrow0 + quarter * 32 < p.R;
            // rows of q; what came before in this CTA is read out of shared and tensor memory
            if (tid == 128) bad = 0;
            constexpr int kStep = (TWO ? 128 : 256) / (D / 8), kLoads = kRowsTc / kStep;          // rows apart, and rows, of a thread
            const int c = wg % (D / 8), qr0 = (TWO ? wg : wg + x * 128) / (D / 8);
            uint4 qv[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int from = myrow0 + qr0 + i * kStep, at = min(from, p.R - 1);
                qv[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + q_offset(p, b, kvh, at) + c * 8);
                if (from >= p.R) qv[i] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int qr = qr0 + i * kStep;
                *reinterpret_cast<uint4 *>(sm_q + (TWO ? x * kItem : 0) + (c >> 3) * kHalf + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = qv[i];
            }
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[x]));
            const uint64_t seen = row < p.R ? drafted_bits(p, b, token_of(p, row), len) : 0;
            const bool stream = !TWO || warp_live || myrow0 < p.R;               // this stream has rows
            float m = -INFINITY, l = 0.0f;
            int mine = 0;                                                        // tiles of this stream in this piece
            for (int t = TWO ? 0 : x; stream && t < tiles; t += TWO ? 1 : 2, ++mine, ++sn) {
                const int key0 = (piece + t - job.begin) * kTileTc;
                const bool tail = key0 + kTileTc > len;
                if (!wait(&s_full[x], sn, 46)) break;
                tc_fence_after();
                if (warp_live) {
                    uint32_t s[128];
#pragma unroll
                    for (int i = 0; i < 4; ++i) tc_ld32(ts + i * 32, *reinterpret_cast<uint32_t(*)[32]>(s + i * 32));
                    tc_wait_ld();
                    if (tail) {
#pragma unroll
                        for (int c = 0; c < 128; ++c) {
                            const int j = key0 + c - len;
                            if (j >= 0 && (j >= 64 || !((seen >> j) & 1))) s[c] = 0xff800000u;
                        }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 128; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(s[c]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
                    const bool grow = mx > m + kLag || m == -INFINITY;
                    if (mine == 0) m = mx;
                    else if (__any_sync(0xffffffffu, grow && mx != m)) {
                        const float to = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : exp2_approx(m - to);
                        l *= f;
                        m = to;
#pragma unroll 1
                        for (int i = 0; i < D / 32; ++i) {
                            uint32_t o[32];
                            tc_ld32(tmem + 256 + x * 128 + lanes + i * 32, o);
                            tc_wait_ld();
#pragma unroll
                            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
                            tc_st16(tmem + 256 + x * 128 + lanes + i * 32, o);
                            tc_st16(tmem + 256 + x * 128 + lanes + i * 32 + 16, o + 16);
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : -m;
                    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), base2 = pack2(base, base);
                    uint64_t sum2[4] = {};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[16];
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float e0, e1;
                            unpack2(fma2(pack2(__uint_as_float(s[i * 32 + 2 * c]), __uint_as_float(s[i * 32 + 2 * c + 1])), scale2, base2), e0, e1);
                            e0 = exp2_approx(e0);
                            e1 = exp2_approx(e1);
                            sum2[c & 3] = add2(sum2[c & 3], pack2(e0, e1));
                            w[c] = narrow<BF16>(e0, e1);
                        }
                        tc_st16(ts + i * 16, w);
                    }
                    float a, c;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), a, c);
                    l += a + c;
                    tc_wait_st();
                }
                if (tail && (!TWO || x == 0)) {
                    // rows of V behind the sequence's end become zero, and so do values of drafted entries that are not finite
                    const int item = 2 * (piece - u0 + t) + 1, slot = item % kItems, at = key0 + wg;
                    if (wait(&full[slot], item / kItems, 47) && at >= len) {
                        uint8_t *v = smem + slot * kItem + wg * 128;
                        bool changed = false;
                        for (int c = 0; c < D / 8; ++c) {
                            uint4 *q = reinterpret_cast<uint4 *>(v + (c >> 3) * kHalf + (((c & 7) ^ (wg & 7)) << 4));
                            uint4 w = *q;
                            uint16_t *h = reinterpret_cast<uint16_t *>(&w);
                            bool here = false;
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (at >= n || nonfinite16<BF16>(h[e])) { h[e] = 0; here = true; }
                            if (here) { *q = w; changed = true; }
                        }
                        if (changed && at < n) atomicOr(&bad, 1ull << (at - len));
                        fence_proxy_async();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[x]));
            }
            // ------------------------------------------------------------------ the piece's result
            const long part = 2L * blockIdx.x + (piece != u0);
            float top = m, sum = l, f0 = 1.0f, f1 = 0.0f;
            int col0 = 0, cols = D;
            bool other = false;
            if (TWO) {
                if (mine) { wait(&o_full[x], on[x], 48); ++on[x]; }
            } else {
                other = tiles > 1;                                               // the second stream had tiles
                wait(&o_full[0], on[0], 48);
                ++on[0];
                if (other) { wait(&o_full[1], on[1], 48); ++on[1]; }
                sm_ml[x][r] = make_float2(m, l);
                bar_sync_named(1, 256);
                const float2 a = sm_ml[0][r], c = sm_ml[1][r];
                top = other ? fmaxf(a.x, c.x) : a.x;
                const float base = top == -INFINITY ? 0.0f : top;
                f0 = exp2_approx(a.x - base);
                f1 = other ? exp2_approx(c.x - base) : 0.0f;
                sum = a.y * f0 + (other ? c.y * f1 : 0.0f);
                cols = D / 2;
                col0 = x * cols;
            }
            tc_fence_after();
            const uint64_t nonfinite = bad;
            if (warp_live && ok) {
                const float factor = row_factor(sum, len == 0 && !seen), base = top == -INFINITY ? 0.0f : top;
#pragma unroll 1
                for (int c0 = col0; c0 < col0 + cols; c0 += 32) {
                    uint32_t a[32], o[32];
                    tc_ld32(tmem + 256 + (TWO ? x * 128 : 0) + lanes + c0, a);
                    if (other) tc_ld32(tmem + 384 + lanes + c0, o);
                    tc_wait_ld();
                    float v[32];
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        v[c] = __uint_as_float(a[c]) * f0;
                        if (other) v[c] += __uint_as_float(o[c]) * f1;
                    }
                    if (row < p.R) {
                        if (nonfinite)
                            for (int c = 0; c < 32; ++c) {
                                // (registers are not indexed by a variable: the sum goes to where its turn is)
                                const float add = nonfinite_part<BF16>(p, nonfinite, seen, b, kvh, row, c0 + c, len, base);
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (e == c) v[e] += add;
                            }
                        if (!whole) {
                            float *dst = p.part_o + part * kJobRows * D + ((c0 >> 2) * kJobRows + (row - row0)) * 4;
#pragma unroll
                            for (int c = 0; c < 32; c += 4) *reinterpret_cast<float4 *>(dst + c * kJobRows) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                        }
                    }
                    if (whole) {
                        // through the rows' own place in the buffer of q, which is not read any more: a warp then writes whole lines
                        uint8_t *dst = sm_q + (TWO ? x * kItem : 0) + (c0 >> 6) * kHalf + r * 128;
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            *reinterpret_cast<uint4 *>(dst + (((((c0 & 32) + c) >> 3) ^ (r & 7)) << 4)) =
                                make_uint4(narrow<BF16>(v[c] * factor, v[c + 1] * factor), narrow<BF16>(v[c + 2] * factor, v[c + 3] * factor),
                                           narrow<BF16>(v[c + 4] * factor, v[c + 5] * factor), narrow<BF16>(v[c + 6] * factor, v[c + 7] * factor));
                    }
                }
                if (whole) {
                    __syncwarp();
                    constexpr int kPieces = (TWO ? D : D / 2) / 8, kRowsAtOnce = 32 / kPieces;       // of 16 bytes, of this warp's rows
                    const int piece_of = col0 / 8 + lane % kPieces;
#pragma unroll
                    for (int i = 0; i < 32; i += kRowsAtOnce) {
                        const int rr = quarter * 32 + i + lane / kPieces, orow = myrow0 + rr, os = token_of(p, orow), oh = kvh * p.g + orow - os * p.g;
                        const uint4 w = *reinterpret_cast<const uint4 *>(sm_q + (TWO ? x * kItem : 0) + (piece_of >> 3) * kHalf + rr * 128 + (((piece_of & 7) ^ (rr & 7)) << 4));
                        if (orow < p.R) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + (((long)b * p.S + os) * p.nh + oh) * D + piece_of * 8) = w;
                    }
                }
                if (row < p.R && col0 == 0) {
                    if (!whole) p.part_ml[part * kJobRows + (row - row0)] = make_float2(top, sum);
                    else if (p.lse) p.lse[((long)b * p.nkv + kvh) * p.R + row] = base + log2f(sum);
                }
            }
            // both streams have read what the next piece overwrites: O of either, the exchanged sums, the marks of V
            bar_sync_named(2, 256);
            piece = end;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D, bool TWO, bool BF16>
int launch_tc(const TreeAttnParams &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t stream) {
    auto kern = attn_tc_kernel<D, TWO, BF16>;
    constexpr int smem = smem_tc<D, TWO>();
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_status(e, "tree_attention shared memory");
    return cuda_status(launch_pdl(kern, dim3((unsigned)p.shares), kThreadsTcA, smem, stream, p, km, vm), "tree_attention launch");
}

}  // namespace

// rows: of a job, 128 or 256
int launch_attn_tc(const TreeAttnParams &p, int rows, bool bf16, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t stream) {
    if (p.D == 128) {
        if (rows == 128) return bf16 ? launch_tc<128, false, true>(p, km, vm, stream) : launch_tc<128, false, false>(p, km, vm, stream);
        return bf16 ? launch_tc<128, true, true>(p, km, vm, stream) : launch_tc<128, true, false>(p, km, vm, stream);
    }
    if (rows == 128) return bf16 ? launch_tc<64, false, true>(p, km, vm, stream) : launch_tc<64, false, false>(p, km, vm, stream);
    return bf16 ? launch_tc<64, true, true>(p, km, vm, stream) : launch_tc<64, true, false>(p, km, vm, stream);
}

int attn_tc_status(int *out) { return cuda_status(cudaMemcpyFromSymbol(out, g_status_attn_tc, sizeof(int) * 4), "attn_tc_status"); }
int attn_tc_status_clear() {
    const int zero[4] = {};
    return cuda_status(cudaMemcpyToSymbol(g_status_attn_tc, zero, sizeof(zero)), "attn_tc_status");
}

}  // namespace flh
