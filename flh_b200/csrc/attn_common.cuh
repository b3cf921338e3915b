// What the kernels of the attention over a cache with drafted entries share: the order of the work, the visibility of entries, and
// the join of partial results.
//
// Rows: the S drafted tokens of a sequence times the g query heads that share a kv head are R = S g rows over the same keys;
// row r is token r / g, head r % g of the group.  A job is a block of rows of one (sequence, kv head); its keys come in tiles.  The
// lengths are read on the device, so that a recorded launch follows them, and so is the division of the work among the CTAs:
//   kEven   all tiles of all jobs in a row (sequence, then head, then block of rows) are cut into equal shares, wherever the cuts fall:
//           a batch of uneven lengths is as balanced as one long sequence.  For more jobs than CTAs, or many sequences.
//   kParts  every job is cut into parts of nearly the same size, as many as its length is worth, a CTA for each: no CTA has
//           parts of two jobs, whose second one costs it what several tiles do (q, the ramp of the rings, the result).  Where that
//           makes the fullest CTA work longer than equal shares and a second part would (one long sequence among many short ones,
//           each of which takes a CTA a head), the CTAs take equal shares instead: 60,000 entries beside 31 sequences of 500, 8 rows,
//           8 heads: 429 us in parts, 44 in equal shares.
//   kJobs   each CTA has as many whole jobs as the next; nothing is cut.
// A job that lies within one CTA is finished there; of a job that was cut each CTA writes a partial result (sum of exponentials,
// maximum, weighted sum of V) to a slot of its own and the join kernel adds them in order.
#pragma once
#include "tc_common.cuh"

namespace flh {

enum { kEven, kParts, kJobs };
constexpr int kTreeTcTile = 64;            // entries of a key tile of attn_tc_kernel
constexpr int kBehind = 1 << 30;           // the first CTA of a job began with another one
// What a second job costs a CTA, in tiles of 32 (attn_mma_kernel), 64 (attn_tc_kernel) and 128 entries (attn_weights_tc_kernel).
template <int TILE> constexpr int kSecondJob = TILE == 32 ? 24 : TILE == 64 ? 12 : 2;

struct TreeAttnParams {
    const void *q;
    long q_sb, q_ss, q_sh;                 // strides in elements; the head's values are contiguous
    const int32_t *lengths;
    const int64_t *tree;                   // ancestor bits [S] or [B, S]; null: a chain
    long tree_sb;
    const void *k, *v;                     // [B, nkv, T, D]
    void *out;                             // [B, S, nh, D]
    float *weights;                        // [B, nkv, T], added to; or null
    const int32_t *counted;                // [B]: tokens of each sequence whose weights are added; null: all
    int B, S, nh, nkv, g, D, R, nrb, rows; // nrb: blocks of `rows` rows
    uint32_t g_inverse;                    // 2^32 / g, rounded up (g > 1)
    int T;
    float scale_log2;                      // scale * log2(e): scores live in powers of two
    int shares, min_share;                 // CTAs, tiles that a share has at least
    int split, jobs_each;                  // kEven, kParts, kJobs; jobs of a CTA (kJobs)
    float *part_o;                         // [2 shares][D / 4][rows of a block][4]: 32 rows of a thread each write whole lines
    float2 *part_ml;                       // [2 shares][rows of a block]: maximum, sum
    int2 *parts_of;                        // [jobs] (kParts), or null: first CTA (and kBehind), number of parts, for the join
    float *lse;                            // [B, nkv, R]: log2 of the sum of powers (with weights), or null
    float *scores;                         // [B, nkv, R, score_ld] (with weights and few rows), or null
    long score_ld;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ int committed(const TreeAttnParams &p, int b) { return min(max(p.lengths[b], 0), p.T); }
__device__ __forceinline__ int entries(const TreeAttnParams &p, int len) { return min(len + p.S, p.T); }    // len <= T < 2^30

// row / g: exact for row < 64 g with g <= 4096, where row * (g_inverse * g - 2^32) < 64 g * g < 2^32
__device__ __forceinline__ int token_of(const TreeAttnParams &p, int row) { return p.g == 1 ? row : (int)__umulhi((uint32_t)row, p.g_inverse); }
// rows of a sequence whose weights are added
__device__ __forceinline__ int counted_rows(const TreeAttnParams &p, int b) { return p.counted ? min(max(p.counted[b], 0), p.S) * p.g : p.R; }
// element offset of a row of q
__device__ __forceinline__ long q_offset(const TreeAttnParams &p, int b, int kvh, int row) {
    const int s = token_of(p, row);
    return b * p.q_sb + s * p.q_ss + (long)(kvh * p.g + row - s * p.g) * p.q_sh;
}
// A value that is the same in all lanes, where the compiler knows it too: what MMAs and TMA loads are issued with has to be in uniform
// registers, and a value out of a shuffle or a load is moved there anew for every instruction (measured: 900 clocks for eight MMAs).
__device__ __forceinline__ int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }

// The reference of a row's exponentials: RAISE powers of two below its largest score x, so that the heaviest weight is 2^RAISE.  Where x is so
// large that its last place is a power of two and more, what the reference is rounded by would push weights over the end of float16: there it
// is x itself.
template <int RAISE> __device__ __forceinline__ float reference_of(float x) {
    if (RAISE == 0) return x;
    return x - (fabsf(x) < 0x1p22f ? (float)RAISE : 0.0f);
}

// The drafted entries that a token sees, as bits; those behind the end of the cache do not exist.
__device__ __forceinline__ uint64_t tree_bits(const TreeAttnParams &p, int b, int s) { return p.tree ? (uint64_t)p.tree[b * p.tree_sb + s] : ~0ull >> (63 - s); }
__device__ __forceinline__ uint64_t existing_bits(const TreeAttnParams &p, int len) {
    const int n = entries(p, len) - len;
    return n >= 64 ? ~0ull : (1ull << n) - 1;
}
__device__ __forceinline__ uint64_t drafted_bits(const TreeAttnParams &p, int b, int s, int len) { return existing_bits(p, len) & tree_bits(p, b, s); }

// Tiles of all jobs up to sequence b (exclusive); warp-uniform.  upto = B: all of them.
template <int TILE>
__device__ __forceinline__ int tiles_before(const TreeAttnParams &p, int upto, int lane) {
    int sum = 0;
    for (int i = lane; i < upto; i += 32) sum += (entries(p, committed(p, i)) + TILE - 1) / TILE;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return uniform(sum) * p.nkv * p.nrb;
}
__device__ __forceinline__ int share_tiles(const TreeAttnParams &p, int total) { return max((total + p.shares - 1) / p.shares, p.min_share); }

// A walk over jobs in order: the job that holds a tile.
template <int TILE>
struct JobWalk {
    int b, job, nt, len, begin;            // sequence; job within the sequence (head * nrb + block of rows); its tiles; first tile
    // job `index` in order; warp-uniform
    __device__ void at(const TreeAttnParams &p, int index, int lane) {
        const int per = p.nkv * p.nrb;
        b = index / per;
        job = index - b * per;
        len = uniform(committed(p, b));
        nt = (entries(p, len) + TILE - 1) / TILE;
        begin = tiles_before<TILE>(p, b, lane) + job * nt;
    }
    // from the start of the order to the job of tile u (u < total); warp-uniform
    __device__ void seek(const TreeAttnParams &p, int u, int lane) {
        const int per = p.nkv * p.nrb;
        int base = 0, b0 = 0;
        for (;;) {                         // 32 sequences at a time
            const int i = b0 + lane;
            const int mine = i < p.B ? (entries(p, committed(p, i)) + TILE - 1) / TILE * per : 0;
            int incl = mine;
            for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += t; }
            const unsigned over = __ballot_sync(0xffffffffu, base + incl > u);
            if (over || b0 + 32 >= p.B) {
                const int l = over ? __ffs(over) - 1 : 31;
                b = min(b0 + l, p.B - 1);
                base += __shfl_sync(0xffffffffu, incl - mine, l);
                break;
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
            b0 += 32;
        }
        b = uniform(b);
        base = uniform(base);
        len = uniform(committed(p, b));
        nt = (entries(p, len) + TILE - 1) / TILE;
        job = (u - base) / nt;
        begin = base + job * nt;
    }
    __device__ __forceinline__ void next(const TreeAttnParams &p) {
        begin += nt;
        if (++job == p.nkv * p.nrb) {
            job = 0;
            if (++b < p.B) {
                len = uniform(committed(p, b));
                nt = (entries(p, len) + TILE - 1) / TILE;
            } else {
                b = p.B;                   // behind the last job: no tile comes here
                nt = 1 << 30;
            }
        }
    }
};

// kParts: the parts that the jobs of a sequence are cut into.  Lane l has those of sequence l (at most 32, and no more jobs than CTAs).
template <int TILE>
struct Parts {
    int nt, parts, size, first;            // tiles of a job, its parts, tiles of a part (the last may have fewer), first CTA of the sequence
    int total;                             // tiles of all jobs
    // false: no size that is at most kSecondJob tiles over an even share has CTAs enough
    __device__ __forceinline__ bool find(const TreeAttnParams &p, int lane) {
        static_assert(kSecondJob<TILE> < 32, "a lane for every size");
        const int per = p.nkv * p.nrb;
        nt = lane < p.B ? (entries(p, committed(p, lane)) + TILE - 1) / TILE : 0;
        total = nt;
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        total *= per;
        // a lane tries a size: the smallest for which there are CTAs enough
        const int tried = share_tiles(p, total) + lane;
        // ceil(nt / tried) as a truncated product: a little less than the quotient, by more than its rounding (2^-22) and less than the
        // distance to the next whole number (1 / tried, nt < 2^17), and one more
        const float inverse = (1.0f - 0x1p-19f) / (float)tried;
        int count = 0;
#pragma unroll 8
        for (int i = 0; i < p.B; ++i) {
            const int other = __shfl_sync(0xffffffffu, nt, i);
            count += (int)((float)other * inverse) + (other > 0);
        }
        const unsigned fits = __ballot_sync(0xffffffffu, lane <= kSecondJob<TILE> && (long)count * per <= p.shares);
        if (!fits) return false;
        size = __shfl_sync(0xffffffffu, tried, __ffs(fits) - 1);
        parts = (nt + size - 1) / size;
        size = nt ? (nt + parts - 1) / parts : 1;
        parts = (nt + size - 1) / size;
        int incl = parts * per;
        for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += t; }
        first = incl - parts * per;
        return true;
    }
};

// Tiles [u0, u1) of this CTA, and the walk at the first of them (u0 < u1)
template <int TILE>
__device__ __forceinline__ void take_share(const TreeAttnParams &p, int lane, JobWalk<TILE> &job, int &u0, int &u1) {
    if (p.split == kJobs) {
        const int per = p.nkv * p.nrb, first = blockIdx.x * p.jobs_each, count = min(p.jobs_each, p.B * per - first);
        job.b = first / per;
        job.job = first - job.b * per;
        job.len = uniform(committed(p, job.b));
        job.nt = (entries(p, job.len) + TILE - 1) / TILE;
        job.begin = 0;                     // its own count of tiles
        JobWalk<TILE> last = job;
        for (int i = 1; i < count; ++i) last.next(p);
        u0 = 0;
        u1 = last.begin + last.nt;
        return;
    }
    int total;
    if (p.split == kParts) {
        Parts<TILE> c;
        if (c.find(p, lane)) {
            const int per = p.nkv * p.nrb, cta = blockIdx.x;
            const unsigned at = __ballot_sync(0xffffffffu, lane < p.B && cta < c.first + c.parts * per);
            u0 = u1 = 0;
            if (!at) return;
            const int b = __ffs(at) - 1;
            const int first = uniform(__shfl_sync(0xffffffffu, c.first, b)), parts = uniform(__shfl_sync(0xffffffffu, c.parts, b)), size = uniform(__shfl_sync(0xffffffffu, c.size, b));
            job.b = b;
            job.job = (cta - first) / parts;
            job.len = uniform(committed(p, b));
            job.nt = (entries(p, job.len) + TILE - 1) / TILE;
            job.begin = 0;                 // its own count of tiles
            u0 = (cta - first - job.job * parts) * size;
            u1 = min(u0 + size, job.nt);
            if (u0 == 0 && threadIdx.x == 0 && p.parts_of) p.parts_of[b * per + job.job] = make_int2(cta, parts);
            return;
        }
        total = uniform(c.total);
    } else {
        total = tiles_before<TILE>(p, p.B, lane);
    }
    const int share = share_tiles(p, total);
    const long first = (long)blockIdx.x * share;
    u0 = (int)min(first, (long)total);
    u1 = (int)min((long)total, first + share);
    if (u0 >= u1) return;
    job.seek(p, u0, lane);
    if (p.split == kParts && p.parts_of && threadIdx.x < 32) {                   // the jobs that begin here
        JobWalk<TILE> at = job;
        if (at.begin < u0) at.next(p);
        for (; at.begin < u1 && at.b < p.B; at.next(p))
            if (threadIdx.x == 0)
                p.parts_of[at.b * p.nkv * p.nrb + at.job] = make_int2(blockIdx.x | (at.begin != u0 ? kBehind : 0), (at.begin + at.nt - 1) / share - (int)blockIdx.x + 1);
    }
}

// A box of a cache's tensor map [heads, entries, values], from (c2, c1, c0) to shared memory
__device__ __forceinline__ void tma_load_tile(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

// Two values rounded to the tensors' type; one value of it.
template <bool BF16> __device__ __forceinline__ uint32_t narrow(float lo, float hi) {
    if (BF16) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <bool BF16> __device__ __forceinline__ float load16(const void *p, long i) {
    if (BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
// whether one of eight 16-bit values is not finite: then its exponent, all ones, carries into the sign's place
template <bool BF16> __device__ __forceinline__ bool any_nonfinite(const uint4 x) {
    const uint32_t e = BF16 ? 0x7f807f80u : 0x7c007c00u, one = BF16 ? 0x00800080u : 0x04000400u;
    return (((x.x & e) + one) | ((x.y & e) + one) | ((x.z & e) + one) | ((x.w & e) + one)) & 0x80008000u;
}
// 16-bit values of a word that are not finite, as zero
template <bool BF16> __device__ __forceinline__ uint32_t finite2(uint32_t w) {
    const uint32_t e = BF16 ? 0x7f807f80u : 0x7c007c00u;
    return w & ~__vcmpeq2(w & e, e);
}

// 1 / l of a row whose exponentials sum to l, as the factor of its weighted sum.  A row that sees nothing is zero; one whose scores
// are all -inf is NaN, as a softmax has it.
__device__ __forceinline__ float row_factor(float l, bool empty) { return l == 0.0f && empty ? 0.0f : 1.0f / l; }

// What the values of drafted entries that are not finite add to one element of the weighted sum of a row: they are kept out of
// the matrix product, where a weight of zero would still make them NaN for rows that do not see them.  bad: those entries; m: the
// maximum that the sum is relative to.
template <bool BF16>
__device__ __noinline__ float nonfinite_part(const TreeAttnParams &p, uint64_t bad, uint64_t seen, int b, int kvh, int row, int d, int len, float m) {
    const long q0 = q_offset(p, b, kvh, row);
    float sum = 0.0f;
    for (uint64_t left = bad & seen; left; left &= left - 1) {
        const long at = (((long)b * p.nkv + kvh) * p.T + len + __ffsll((long long)left) - 1) * p.D;
        const float x = load16<BF16>(p.v, at + d);
        if (fabsf(x) <= 3.4e38f) continue;
        float dot = 0.0f;
        for (int i = 0; i < p.D; ++i) dot = fmaf(load16<BF16>(p.q, q0 + i), load16<BF16>(p.k, at + i), dot);
        sum += exp2_approx(fmaf(dot, p.scale_log2, -m)) * x;
    }
    return sum;
}

}  // namespace flh
