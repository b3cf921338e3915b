// What happens to a KV cache around the attention of a drafted tree (attn_tree.cu):
//   * rope_kv_at_kernel     the drafted q and k turned to their depth in the tree, k and v written behind each sequence's own length;
//   * cache_accept_kernel   the accepted branch moved together behind the committed entries, in all layers by one launch;
//   * evict_select_kernel   per (layer, sequence, kv head): the most recent entries and the heaviest of the others, in order;
//   * evict_move_kernel     their rows moved together in place.
// All of them move bytes; what a pass cannot do without is each moved row read once and written once.
#include "act_common.cuh"
#include "attn_common.cuh"
#include "tc_pair.cuh"
#include <algorithm>

namespace flh {
namespace {

constexpr int kMaxLayers = FLH_B200_CACHE_MAX_LAYERS;
constexpr int kMaxDrafted = FLH_B200_TREE_MAX_TOKENS;

// ---- append ---------------------------------------------------------------------------------
struct RopeAtParams {
    const void *qkv;                       // [B * S, (nh + 2 nkv) * D]
    const float *cos, *sin;                // [P, D / 2]
    const int32_t *positions, *lengths;    // [B * S], [B]
    void *q_out, *k_cache, *v_cache;       // [B, S, nh, D], [B, nkv, T, D]
    int S, nh, nkv, D;
    long P, T;
};

template <bool BF16> __device__ __forceinline__ float2 widen2(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}

// One block per token (and part of its heads), a thread takes 16 bytes of the first half of a head and their rotation partners, as in
// rope_kv_kernel; x1 cos - x2 sin and x2 cos + x1 sin with every product and sum rounded on its own, the bits of separate tensor
// operations.  The row of the tables goes by the token's position, the row of the caches by its sequence's length: a token behind the
// end of the cache leaves it as it is, a position that the tables do not have turns q and k into NaN.
template <bool BF16>
__global__ void __launch_bounds__(256) rope_kv_at_kernel(const RopeAtParams p) {
    const int half = p.D / 2, vec = half / 8, heads = p.nh + 2 * p.nkv, items = heads * vec;
    const long token = blockIdx.x;
    const int b = (int)(token / p.S), s = (int)(token - (long)b * p.S);
    pdl_wait();
    pdl_trigger();
    const long pos = p.positions[token], slot = (long)p.lengths[b] + s;
    const bool known = pos >= 0 && pos < p.P, kept = slot >= 0 && slot < p.T;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < items; i += gridDim.y * 256) {
        const int h = i / vec, v = i - h * vec;
        const uint16_t *src = static_cast<const uint16_t *>(p.qkv) + (token * heads + h) * p.D + v * 8;
        uint4 lo = ldg_nc_v4(src), hi = ldg_nc_v4(src + half);
        if (h < p.nh + p.nkv) {
            uint32_t *a = reinterpret_cast<uint32_t *>(&lo), *c = reinterpret_cast<uint32_t *>(&hi);
            const float *ct = p.cos + pos * half + v * 8, *st = p.sin + pos * half + v * 8;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float nan = __int_as_float(0x7fffffff);
                const float2 cc = known ? *reinterpret_cast<const float2 *>(ct + 2 * e) : make_float2(nan, nan);
                const float2 ss = known ? *reinterpret_cast<const float2 *>(st + 2 * e) : make_float2(nan, nan);
                const float2 x1 = widen2<BF16>(a[e]), x2 = widen2<BF16>(c[e]);
                a[e] = narrow<BF16>(__fsub_rn(__fmul_rn(x1.x, cc.x), __fmul_rn(x2.x, ss.x)), __fsub_rn(__fmul_rn(x1.y, cc.y), __fmul_rn(x2.y, ss.y)));
                c[e] = narrow<BF16>(__fadd_rn(__fmul_rn(x2.x, cc.x), __fmul_rn(x1.x, ss.x)), __fadd_rn(__fmul_rn(x2.y, cc.y), __fmul_rn(x1.y, ss.y)));
            }
        }
        uint16_t *dst;
        if (h < p.nh) dst = static_cast<uint16_t *>(p.q_out) + (token * p.nh + h) * p.D;
        else {
            if (!kept) continue;
            const bool isk = h < p.nh + p.nkv;
            dst = static_cast<uint16_t *>(isk ? p.k_cache : p.v_cache) + (((long)b * p.nkv + (h - p.nh - (isk ? 0 : p.nkv))) * p.T + slot) * p.D;
        }
        *reinterpret_cast<uint4 *>(dst + v * 8) = lo;
        *reinterpret_cast<uint4 *>(dst + v * 8 + half) = hi;
    }
}

// ---- accept ---------------------------------------------------------------------------------
struct AcceptParams {
    void *k[kMaxLayers], *v[kMaxLayers];
    float *w[kMaxLayers];
    const int32_t *lengths, *path, *accepted;
    int32_t *now;
    int B, nkv, A, S, chunks;              // chunks of 16 bytes in a row
    long T;
    int weights;
};

// Block (layer and what of it: K, V or the weights; sequence and head).  Everything a block moves is read before anything is written,
// so that a path may name its entries in any order and more than once.  N: pieces of 16 bytes for each of the 128 threads.
template <int N>
__global__ void __launch_bounds__(128) cache_accept_kernel(const __grid_constant__ AcceptParams p) {
    const int kinds = p.weights ? 3 : 2, layer = blockIdx.y / kinds, kind = blockIdx.y - layer * kinds;
    const int b = blockIdx.x / p.nkv, tid = threadIdx.x;
    pdl_wait();
    pdl_trigger();
    const long len = p.lengths[b];
    const int n = min(max(p.accepted[b], 0), p.A);
    const int32_t *path = p.path + (long)b * p.A;
    const bool first = blockIdx.x % p.nkv == 0 && blockIdx.y == 0;
    if (first && tid == 0 && p.now) p.now[b] = (int32_t)min(max(len, 0L) + n, p.T);
    // the entry that drafted entry i is taken from; i itself where there is none to take
    auto source = [&](int i) {
        if (i >= n) return i;
        const int from = path[i];
        return from < 0 || from >= p.S || len + from >= p.T ? i : from;
    };
    if (len < 0) return;
    if (kind == 2) {
        static_assert(kMaxDrafted <= 128, "a thread per drafted entry");
        float *w = p.w[layer] + (long)blockIdx.x * p.T + len;
        const bool mine = tid < p.S && len + tid < p.T;
        const float x = mine && tid < n ? w[source(tid)] : 0.0f;
        __syncthreads();
        if (mine) w[tid] = x;
        return;
    }
    uint4 *rows = static_cast<uint4 *>(kind ? p.v[layer] : p.k[layer]) + ((long)blockIdx.x * p.T + len) * p.chunks;
    const int items = n * p.chunks;
    uint4 x[N];
    int from[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = tid + 128 * j, r = i / p.chunks;
        from[j] = i < items && len + r < p.T ? source(r) : r;
        if (from[j] != r) x[j] = rows[(long)from[j] * p.chunks + (i - r * p.chunks)];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int i = tid + 128 * j;
        if (from[j] != i / p.chunks) rows[i] = x[j];
    }
}

// ---- evict ----------------------------------------------------------------------------------
struct EvictParams {
    void *k[kMaxLayers], *v[kMaxLayers];
    const float *w[kMaxLayers];
    const int32_t *lengths;
    int32_t *kept, *now;                   // [layers, B, nkv, keep], [B]
    float *left;                           // [layers, B, nkv, T]
    int B, nkv, keep, recent, chunks;
    long T;
};

// weights in an order of unsigned numbers: NaN above +inf, -0 as 0
__device__ __forceinline__ uint32_t order_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelKeys = 45056;            // of a block in shared memory, 176 KB
constexpr int kMaxCluster = 8;
constexpr int kSelAhead = 4;               // times 32 entries that a warp has under way

__device__ __forceinline__ uint32_t cluster_size_of() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r)); return r; }
// a word of shared memory of another CTA of the cluster, at the place that `local` has in this one
__device__ __forceinline__ uint32_t peer_u32(const uint32_t *local, uint32_t rank) {
    uint32_t at, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// A block per row, or a cluster of blocks that have a stretch of it each.  The smallest key that is kept is found digit by digit, eight
// bits at a time, by counting the keys that agree with the digits found so far; then the row is walked in order, every warp over a
// part of its own, and what lies above that key is kept, of the equal ones the first few.  The keys stay in shared memory (cap: how
// many fit; the rest is read again).  Every lane counts in a histogram of its own, since weights are much alike in their leading bits;
// in small caches two or four lanes share one, since the histograms have to be cleared and added up for each digit.  (With 8 copies of
// the counters 256 rows of 8,192 took 31 us, finding the key two bits at a time by comparisons in registers 33, counting equal digits
// of a warp once 28; this 25.)
template <int THREADS, int COPIES>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const __grid_constant__ EvictParams p, int cap) {
    constexpr int kWarps = THREADS / 32, kLanes = COPIES / 8, kDigits = 256 / kWarps;            // lanes for a digit's counts, digits of a warp
    static_assert(64 * COPIES % THREADS == 0, "whole steps to clear the histogram");
    static_assert(COPIES % 8 == 0 && 32 % kLanes == 0 && kDigits % (32 / kLanes) == 0, "whole steps over a warp's digits");
    extern __shared__ uint32_t keys[];
    __shared__ __align__(16) uint32_t hist[256 * COPIES]; // [digit][lane % COPIES]
    __shared__ uint32_t digits[2][256];    // of one digit and the next, in turn: the cluster may still read the last ones
    __shared__ uint32_t total[256];
    __shared__ uint32_t found[2];          // prefix, how many of the keys that match it are to be kept
    __shared__ uint32_t above[kWarps], equal[kWarps], sides[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = cluster_size_of(), rank = cluster_rank();
    const int layer = blockIdx.y, head = blockIdx.x / blocks, b = head / p.nkv;
    pdl_wait();
    pdl_trigger();
    const long row = (long)layer * (gridDim.x / blocks) + head;
    const float *w = p.w[layer] + (long)head * p.T;
    float *left = p.left + row * p.T;
    int32_t *kept = p.kept + row * p.keep;
    const int n = (int)min(max((long)p.lengths[b], 0L), p.T), m = min(n, p.keep);
    const int all = blocks * THREADS, me = rank * THREADS + tid;
    if (me == 0 && layer == 0 && head % p.nkv == 0) p.now[b] = m;
    for (int i = m + me; i < p.keep; i += all) kept[i] = -1;
    for (long i = m + me; i < p.T; i += all) left[i] = 0.0f;
    if (n <= p.keep) {
        for (int i = me; i < n; i += all) { kept[i] = i; left[i] = w[i]; }
        return;                            // the whole cluster
    }
    const int cand = n - p.recent;         // recent <= keep < n
    uint32_t need = p.keep - p.recent, prefix = 0;
    // this block's stretch of the row (whole warps' spans), and its warps'
    const int span = ((n + blocks * kWarps - 1) / (blocks * kWarps) + 31) / 32 * 32;
    const int lo = min(rank * kWarps * span, n), hi = min(lo + kWarps * span, n), own = min(hi, cand) - lo;      // entries to choose from: may be none
    auto key = [&](int i) { return i < cap ? keys[i] : order_key(w[lo + i]); };
#pragma unroll 8
    for (int i = tid; i < min(own, cap); i += THREADS) keys[i] = order_key(w[lo + i]);
    if (need) {
        for (int shift = 24, turn = 0; shift >= 0; shift -= 8, turn ^= 1) {
#pragma unroll
            for (int i = 0; i < 64 * COPIES / THREADS; ++i) reinterpret_cast<uint4 *>(hist)[tid + i * THREADS] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
#pragma unroll 4
            for (int i = tid; i < own; i += THREADS) {
                const uint32_t u = key(i);
                if ((u & mask) == prefix) atomicAdd(&hist[((u >> shift) & 255u) * COPIES + lane % COPIES], 1u);
            }
            __syncthreads();
            // a lane has eight of a digit's counts
#pragma unroll
            for (int i = 0; i < kDigits; i += 32 / kLanes) {
                const int d = warp * kDigits + i + lane / kLanes;
                const uint32_t *h = &hist[d * COPIES + lane % kLanes * 4];
                const uint4 u = *reinterpret_cast<const uint4 *>(h), v = *reinterpret_cast<const uint4 *>(h + COPIES / 2);
                uint32_t c = u.x + u.y + u.z + u.w + v.x + v.y + v.z + v.w;
#pragma unroll
                for (int o = 1; o < kLanes; o <<= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
                if (lane % kLanes == 0) digits[turn][d] = c;
            }
            if (blocks > 1) {
                cluster_sync_all();
                for (int i = tid; i < 256; i += THREADS) {
                    uint32_t c = 0;
                    for (int r = 0; r < blocks; ++r) c += peer_u32(&digits[turn][i], r);
                    total[i] = c;
                }
            }
            __syncthreads();
            if (warp == 0) {
                // lane l: digits 255 - 8 l .. 248 - 8 l, from the largest down
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) { c[e] = blocks > 1 ? total[255 - 8 * lane - e] : digits[turn][255 - 8 * lane - e]; sum += c[e]; }
                uint32_t before = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t t = __shfl_up_sync(0xffffffffu, before, o);
                    if (lane >= o) before += t;
                }
                before -= sum;             // keys with a larger digit than this lane's
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (before < need && need <= before + c[e]) { found[0] = prefix | ((uint32_t)(255 - 8 * lane - e) << shift); found[1] = need - before; }
                    before += c[e];
                }
            }
            __syncthreads();
            prefix = found[0];
            need = found[1];
        }
    } else {
        prefix = 0xffffffffu;              // none of the others; a NaN is equal and not needed
        __syncthreads();
    }
    // a warp walks entries [from, to) of the row, 32 at a time; the recent ones are above everything
    const int from = min(lo + warp * span, hi), to = min(from + span, hi);
    auto side = [&](int i) { return i >= to ? 0 : i >= cand ? 2 : key(i - lo) > prefix ? 2 : key(i - lo) == prefix ? 1 : 0; };
    uint32_t na = 0, ne = 0;
    for (int i = from; i < to; i += 32 * kSelAhead) {
#pragma unroll
        for (int k = 0; k < kSelAhead; ++k) {
            const int s = side(i + k * 32 + lane);
            na += __popc(__ballot_sync(0xffffffffu, s == 2));
            ne += __popc(__ballot_sync(0xffffffffu, s == 1));
        }
    }
    if (lane == 0) { above[warp] = na; equal[warp] = ne; }
    __syncthreads();
    uint32_t a0 = 0, e0 = 0;               // what lies before this warp's stretch
    for (int i = 0; i < warp; ++i) { a0 += above[i]; e0 += equal[i]; }
    if (blocks > 1) {
        if (warp == kWarps - 1 && lane == 0) { sides[0] = a0 + na; sides[1] = e0 + ne; }
        cluster_sync_all();
        for (int r = 0; r < rank; ++r) { a0 += peer_u32(&sides[0], r); e0 += peer_u32(&sides[1], r); }
    }
    for (int i = from; i < to; i += 32 * kSelAhead) {
        float x[kSelAhead];                // fetched together
#pragma unroll
        for (int k = 0; k < kSelAhead; ++k) x[k] = i + k * 32 + lane < to ? w[i + k * 32 + lane] : 0.0f;
#pragma unroll
        for (int k = 0; k < kSelAhead; ++k) {
            const int s = side(i + k * 32 + lane);
            const uint32_t ba = __ballot_sync(0xffffffffu, s == 2), be = __ballot_sync(0xffffffffu, s == 1), low = (1u << lane) - 1;
            const uint32_t ea = e0 + __popc(be & low);
            if (s == 2 || (s == 1 && ea < need)) {
                const uint32_t at = a0 + __popc(ba & low) + min(ea, need);
                kept[at] = i + k * 32 + lane;
                left[at] = x[k];
            }
            a0 += __popc(ba);
            e0 += __popc(be);
        }
    }
    if (blocks > 1) cluster_sync_all();     // the others have read this block's counts
}

// Rows kept[0 .. m) of K and V to rows 0 .. m - 1, in place.  kept rises, so kept[d] >= d: rows that a batch writes are read by
// that batch and by earlier ones only.  A block owns a column of a row's 16-byte pieces; while it has one batch of rows to write it
// reads the next one and the indices of the one after that, and it writes when all its threads have read theirs.
template <int THREADS, int PIECES>
__global__ void __launch_bounds__(THREADS) evict_move_kernel(const __grid_constant__ EvictParams p, int slab) {
    const int layer = blockIdx.y, unit = blockIdx.x, slabs = p.chunks / slab;
    const int bh = unit / (2 * slabs), sub = unit - bh * 2 * slabs, isv = sub / slabs, c0 = (sub - isv * slabs) * slab;
    pdl_wait();
    pdl_trigger();
    const int rows = THREADS / slab, r = threadIdx.x / slab, c = c0 + threadIdx.x - r * slab;
    const int heads = gridDim.x / (2 * slabs), b = bh / p.nkv;
    const int n = (int)min(max((long)p.lengths[b], 0L), p.T);
    if (n <= p.keep) return;               // the whole block
    const int end = r < rows ? p.keep : 0; // threads that a slab of odd width leaves over have nothing to move
    const int32_t *kept = p.kept + ((long)layer * heads + bh) * p.keep;
    uint4 *base = static_cast<uint4 *>(isv ? p.v[layer] : p.k[layer]) + (long)bh * p.T * p.chunks + c;
    const int batch = rows * PIECES;
    uint4 x[PIECES], y[PIECES];
    int fx[PIECES], fy[PIECES], fz[PIECES];
    auto indices = [&](int d0, int (&f)[PIECES]) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int d = d0 + r + j * rows;
            f[j] = d < end ? kept[d] : d;
        }
    };
    auto load = [&](int d0, const int (&f)[PIECES], uint4 (&v)[PIECES]) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
            if (f[j] != d0 + r + j * rows) v[j] = base[(long)f[j] * p.chunks];
    };
    indices(0, fx);
    indices(batch, fy);
    load(0, fx, x);
    for (int d0 = 0; d0 < p.keep; d0 += batch) {
        indices(d0 + 2 * batch, fz);
        load(d0 + batch, fy, y);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int d = d0 + r + j * rows;
            if (fx[j] != d) base[(long)d * p.chunks] = x[j];
            x[j] = y[j];
            fx[j] = fy[j];
            fy[j] = fz[j];
        }
    }
}

}  // namespace

int launch_rope_kv_at(const void *qkv, int dtype, const float *cos, const float *sin, long P, const int32_t *positions, const int32_t *lengths,
                      void *q_out, void *k_cache, void *v_cache, int B, int S, int nh, int nkv, int D, long T, cudaStream_t stream) {
    RopeAtParams p;
    p.qkv = qkv; p.cos = cos; p.sin = sin; p.positions = positions; p.lengths = lengths;
    p.q_out = q_out; p.k_cache = k_cache; p.v_cache = v_cache;
    p.S = S; p.nh = nh; p.nkv = nkv; p.D = D; p.P = P; p.T = T;
    const long tokens = (long)B * S, items = (long)(nh + 2 * nkv) * (D / 16), parts = std::min((items + 255) / 256, 65535L);
    const dim3 grid((unsigned)tokens, (unsigned)(tokens >= 4L * kNumSMs ? 1 : parts));
    return cuda_status(launch_pdl(dtype == FLH_B200_BF16 ? rope_kv_at_kernel<true> : rope_kv_at_kernel<false>, grid, 256, 0, stream, p), "rope_kv_at launch");
}

int launch_cache_accept(void *const *k, void *const *v, float *const *w, int layers, const int32_t *lengths, const int32_t *path, const int32_t *accepted,
                        int32_t *now, int B, int nkv, int D, long T, int A, int S, cudaStream_t stream) {
    AcceptParams p;
    for (int i = 0; i < layers; ++i) { p.k[i] = k[i]; p.v[i] = v[i]; p.w[i] = w ? w[i] : nullptr; }
    p.lengths = lengths; p.path = path; p.accepted = accepted; p.now = now;
    p.B = B; p.nkv = nkv; p.A = A; p.S = S; p.chunks = D / 8; p.T = T; p.weights = w != nullptr;
    const dim3 grid((unsigned)(B * nkv), (unsigned)(layers * (w ? 3 : 2)));
    const int pieces = (A * p.chunks + 127) / 128;
    auto kern = pieces <= 1 ? cache_accept_kernel<1> : pieces <= 4 ? cache_accept_kernel<4> : cache_accept_kernel<16>;
    return cuda_status(launch_pdl(kern, grid, 128, 0, stream, p), "cache_accept launch");
}

int launch_cache_evict(void *const *k, void *const *v, const float *const *w, int layers, const int32_t *lengths, int32_t *kept, float *left, int32_t *now,
                       int B, int nkv, int D, long T, int keep, int recent, cudaStream_t stream) {
    EvictParams p;
    for (int i = 0; i < layers; ++i) { p.k[i] = k[i]; p.v[i] = v[i]; p.w[i] = w[i]; }
    p.lengths = lengths; p.kept = kept; p.now = now; p.left = left;
    p.B = B; p.nkv = nkv; p.keep = keep; p.recent = recent; p.chunks = D / 8; p.T = T;
    // One block per row; a cluster of up to 8 where the rows do not fill the GPU and are long (16 rows of 24,000: 29 -> 18 us).  Short rows
    // take blocks of 256 threads, of which more fit an SM; caches of up to 4,096 entries half the histograms (32 rows of 2,047 of 2,111
    // entries 15.7 -> 14.8 us, 256 of 4,090 of 4,096 21.3 -> 19.9).  What counts is the cache's size: the lengths are not known here.
    const long rows = (long)B * nkv * layers;
    int blocks = 1;
    while (blocks < kMaxCluster && rows * blocks * 2 <= kNumSMs && T >= 4096L * blocks) blocks *= 2;
    const bool few = T <= 2048, medium = T <= 4096;
    const long each = (T + blocks - 1) / blocks + 2048;                  // a block's stretch, rounded up to whole spans
    const int cap = (int)(each < kSelKeys ? each : kSelKeys);
    auto select = few ? evict_select_kernel<256, 8> : medium ? evict_select_kernel<512, 16> : evict_select_kernel<512, 32>;
    static std::atomic<uint64_t> done[3];
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(select), kSelKeys * 4, done[few ? 0 : medium ? 1 : 2]);
    if (e != cudaSuccess) return cuda_status(e, "cache_evict shared memory");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = blocks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(B * nkv * blocks), (unsigned)layers); cfg.blockDim = dim3(few ? 256 : 512);
    cfg.dynamicSmemBytes = (size_t)cap * 4; cfg.stream = stream; cfg.attrs = attr; cfg.numAttrs = blocks > 1 ? 2 : 1;
    int rc = cuda_status(cudaLaunchKernelEx(&cfg, select, p, cap), "cache_evict select");
    if (rc) return rc;
    // A block per half of a row's pieces (128 bytes of a head of 128), so that one layer of one sequence already spreads over the GPU:
    // 256 threads with 8 pieces each (512 MB: 95 us; with 4 pieces 126).  Where that is a block for half of the SMs or less and each has
    // much to move, quarters and 512 threads (16 heads, 24,000 -> 15,600 entries: 105 -> 71 us in all); where it is little, 128 threads with 4
    // pieces, of which more fit an SM (1,536 heads, 700 -> 197 entries: 130 -> 82 us with the smaller blocks of the selection).
    const bool much = rows * 4 <= kNumSMs / 2 && keep > 2048 && p.chunks % 4 == 0 && p.chunks >= 8, little = keep <= 512;
    const int slabs = much ? 4 : p.chunks % 2 == 0 && p.chunks >= 8 ? 2 : 1, slab = p.chunks / slabs;
    const dim3 grid((unsigned)(B * nkv * 2 * slabs), (unsigned)layers);
    if (much) return cuda_status(launch_pdl(evict_move_kernel<512, 8>, grid, 512, 0, stream, p, slab), "cache_evict move");
    if (little) return cuda_status(launch_pdl(evict_move_kernel<128, 4>, grid, 128, 0, stream, p, slab), "cache_evict move");
    return cuda_status(launch_pdl(evict_move_kernel<256, 8>, grid, 256, 0, stream, p, slab), "cache_evict move");
}

}  // namespace flh
