// The attention of attn_tree.cu on the 5th-generation tensor cores, for jobs of many rows: S drafted tokens times the g query heads of a
// kv head are R rows over the same entries, and from a few dozen on the products, not the memory, are what a pass waits for.
//
// A CTA per SM.  One warp loads key tiles (64 entries) of K and V by TMA into a ring; two streams, each a warp that issues its MMAs and
// a group of four warps that has its softmax, a thread per row, work through them.  A stream is a block of 128 rows with two tiles of
// scores S and an accumulator O in tensor memory:
//   S = Q K^T        both operands in shared memory, K as it lies there
//   P = 2^(S - m)    read from tensor memory, rounded to 16 bits (half a step of each weight; their sum is of the unrounded ones) and
//                    written over S
//   O += P V         P from tensor memory, V from shared memory as it lies there, read along the entries
// The scores of the next tile are made while the threads are at this one, so that they wait for a product only when the tensor cores are
// what bounds the pass.  What goes from the softmax to the products is a named barrier (56 clocks there and back; a wait on an
// mbarrier is 120 - 160 even where it does not have to wait, so those that remain are asked before their time has come).
// With more than 128 rows the two streams are two blocks of rows that share every tile (half the shared-memory traffic and half
// the reads of K and V); with up to 128 they are the same rows over every other tile, and their results become one at the end of a
// piece, straight from tensor memory.
//
// The reference m that the exponentials are relative to follows the true maximum only when that is 2^8 ahead: O is then read, scaled and
// written back.  In float16, which ends at 2^-24 and at 2^16, m is 2^7 below the maximum that it was taken from: P reaches 2^15 at most, and
// what is 2^-26 of the heaviest keeps five bits and more of itself (relative to the maximum it vanished from O, not from the sum).
#include "attn_common.cuh"
#include "tc_pair.cuh"
#include "tc_quant_common.cuh"
#include <type_traits>

namespace flh {
namespace {

__device__ int g_status_attn_tc[4];

constexpr int kTileTc = kTreeTcTile, kRowsTc = 128;
constexpr int kThreadsTcA = 384;           // warp 0 TMA, warps 1 and 2 MMA, warps 4 - 7 and 8 - 11 softmax
// registers: 384 threads are launched with 168; 128 * 112 + 256 * 192 are less than those 64,512
constexpr int kRegsIssue = 112, kRegsSoftmax = 192;
static_assert(128 * kRegsIssue + 256 * kRegsSoftmax <= kThreadsTcA * 168, "more registers than the CTA was launched with");
constexpr float kLag = 8.0f;               // powers of two that the true maximum may be ahead of the one that m was taken from
template <bool BF16> constexpr int kRaise = BF16 ? 0 : 7;                              // and that m lies below that one

template <int D> constexpr int item_bytes() { return kTileTc * D * 2; }                         // K or V of a tile
template <int D> constexpr int q_bytes() { return kRowsTc * D * 2; }                            // a block of rows of Q
// Slots of the ring.  Streams that take turns need a multiple of four: then a slot is always the same stream's, and a wait on it is never
// two phases away from what the barrier is at.
template <int D, bool TWO> constexpr int items_tc() { return (TWO ? 160 : 192) * 1024 / item_bytes<D>(); }
template <int D, bool TWO> constexpr int smem_tc() { return 1024 + items_tc<D, TWO>() * item_bytes<D>() + (TWO ? 2 : 1) * q_bytes<D>(); }

__device__ __forceinline__ void bar_arrive_named(int id, int nthreads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory"); }
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
__device__ __forceinline__ void tc_st2(uint32_t taddr, uint32_t a, uint32_t b) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1,%2};" ::"r"(taddr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void tc_ld2(uint32_t taddr, uint32_t &a, uint32_t &b) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(a), "=r"(b) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// TWO: the streams are two blocks of rows; otherwise they share one.
template <int D, bool TWO, bool BF16>
__global__ void __launch_bounds__(kThreadsTcA, 1) attn_tc_kernel(const __grid_constant__ TreeAttnParams p, const __grid_constant__ CUtensorMap kmap,
                                                                 const __grid_constant__ CUtensorMap vmap) {
    static_assert(TWO || items_tc<D, TWO>() % 4 == 0, "a slot of the ring belongs to one stream");
    constexpr int kItem = item_bytes<D>(), kItems = items_tc<D, TWO>(), kHalf = kTileTc * 128, kQ = q_bytes<D>(), kQHalf = kRowsTc * 128, kJobRows = TWO ? 2 * kRowsTc : kRowsTc;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sm_q = smem + kItems * kItem;
    __shared__ uint64_t full[kItems], empty[kItems], s_full[2][2], o_full[2][2], q_full[2];  // [stream][its tiles in turn]
    __shared__ unsigned long long bad[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < kItems; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), TWO ? 2 : 1); }
        for (int i = 0; i < 2; ++i) {
            for (int j = 0; j < 2; ++j) { mbar_init(smem_u32(&s_full[i][j]), 1); mbar_init(smem_u32(&o_full[i][j]), 1); }
            mbar_init(smem_u32(&q_full[i]), TWO ? 4 : 8);
        }
        abort_flag = 0;
        bad[0] = bad[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();
    pdl_trigger();

    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t phase, int code) {
        if (ok) ok = mbar_wait_warp(g_status_attn_tc, bar, phase & 1, &abort_flag, code);
        return ok;
    };
    const uint32_t fulls = smem_u32(full), empties = smem_u32(empty);
    JobWalk<kTileTc> job;
    int u0, u1;
    take_share(p, lane, job, u0, u1);

    // Items 2 i and 2 i + 1 of the ring are K and V of the CTA's tile u0 + i, in slot item % kItems.
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp == 0) {
        // ---------------------------------------------------------------------- loads
        int item = 0, slot = 0;
        uint32_t phase = 1;
        const uint32_t ring = uniform(smem_u32(smem));
        for (int u = u0; u < u1 && ok; ++u) {
            while (u >= job.begin + job.nt) job.next(p);
            const int head = job.b * p.nkv + job.job / p.nrb, key0 = (u - job.begin) * kTileTc;
            for (int kv = 0; kv < 2 && ok; ++kv) {
                wait(empties + 8 * slot, phase, 41);
                const uint32_t bar = fulls + 8 * slot, dst = ring + slot * kItem;
                const CUtensorMap *map = kv ? &vmap : &kmap;
                if (ok && elect_one()) {
                    mbar_expect_tx(bar, kItem);
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) tma_load_tile(dst + h * kHalf, map, h * 64, key0, head, bar);
                }
                __syncwarp();
                item += ok;
                if (++slot == kItems) { slot = 0; phase ^= 1; }
            }
        }
        // what is still in flight lands before the CTA leaves (after a wait that ran out; otherwise all of it was used)
        for (int i = max(0, item - kItems); i < item; ++i)
            for (int tries = 0; tries < 10000 && !__all_sync(0xffffffffu, mbar_try_hint(fulls + 8 * (i % kItems), (i / kItems) & 1, 20000u)); ++tries);
    } else if (warp < 3) {
        // ---------------------------------------------------------------------- products of stream x
        const int x = warp - 1;
        const uint32_t fmt = BF16 ? 1u : 0u, base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRowsTc >> 4) << 24);
        const uint32_t id_qk = base | ((uint32_t)(kTileTc >> 3) << 17), id_pv = base | (1u << 16) | ((uint32_t)(D >> 3) << 17);
        const uint32_t ring = uniform(smem_u32(smem)), qbase = uniform(smem_u32(sm_q) + (TWO ? x * kQ : 0)), tm = uniform(tmem + x * 128);
        const uint32_t s_bar = uniform(smem_u32(&s_full[x][0])), o_bar = uniform(smem_u32(&o_full[x][0]));
        // the stream's next K and next V: slots 2 i and 2 i + 1 of the ring's kItems, i counting its tiles
        constexpr int kAdvance = TWO ? 2 : 4;
        uint32_t ks = TWO ? 0 : 2 * x, kph = 0, vs = ks + 1, vph = 0, qph = 0, nk = 0, nv = 0;           // nk, nv: tiles so far
        auto advance = [](uint32_t &slot, uint32_t &phase, uint32_t by) { slot += by; if (slot >= kItems) { slot -= kItems; phase ^= 1; } };
        for (int piece = u0; piece < u1;) {
            while (piece >= job.begin + job.nt) job.next(p);
            const int end = min(u1, job.begin + job.nt), tiles = end - piece;
            // the second block of rows may not exist; with one block the streams take turns, beginning with the tile at u0
            const bool live = !TWO || x == 0 || (job.job % p.nrb) * kJobRows + kRowsTc < p.R;
            const int mine = TWO ? tiles : (tiles + (((piece - u0) & 1) == x)) / 2;
            wait(smem_u32(&q_full[TWO ? x : 0]), qph, 43);
            qph ^= 1;
            tc_fence_after();
            if (!live) {                                                         // the other stream's tiles: they are not waited for here
                for (int i = 0; i < 2 * tiles; ++i) {
                    wait(fulls + 8 * (i & 1 ? vs : ks), i & 1 ? vph : kph, 42);
                    if (ok && elect_one()) mbar_arrive(empties + 8 * (i & 1 ? vs : ks));
                    __syncwarp();
                    if (i & 1) advance(vs, vph, kAdvance);
                    else advance(ks, kph, kAdvance);
                }
                bar_arrive_named(2, 320);
                piece = end;
                continue;
            }
            // the tile's K is there
            auto qk = [&]() {
                tc_fence_after();
                const uint64_t a = make_smem_desc(qbase), b = make_smem_desc(ring + ks * kItem);
                const uint32_t d = tm + (nk & 1) * kTileTc;
                if (ok && elect_one()) {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s)
                        mma_f16<false>(d, a + (((s >> 2) * kQHalf + (s & 3) * 32) >> 4), b + (((s >> 2) * kHalf + (s & 3) * 32) >> 4), id_qk, s > 0);
                    tc_commit(s_bar + 8 * (nk & 1));
                    tc_commit(empties + 8 * ks);
                }
                __syncwarp();
                ++nk;
                advance(ks, kph, kAdvance);
            };
            for (int i = 0; i < min(mine, 2); ++i) {
                wait(fulls + 8 * ks, kph, 42);
                qk();
            }
            // whether a load is there is asked before the products that come first are issued, and the answer looked at behind them
            bool v_there = mine > 0 && mbar_test(fulls + 8 * vs, vph), k_there = true;
            for (int i = 0; i < mine; ++i) {
                if (!__all_sync(0xffffffffu, v_there)) wait(fulls + 8 * vs, vph, 45);
                if (i + 2 < mine) k_there = mbar_test(fulls + 8 * ks, kph);
                bar_sync_named(3 + 2 * x + (nv & 1), 160);                       // the weights are written
                tc_fence_after();
                const uint64_t b = umma_desc_tc(ring + vs * kItem, kHalf, 1024);
                const uint32_t d = tm + 256, a = tm + (nv & 1) * kTileTc, more = i > 0;
                if (ok && elect_one()) {
#pragma unroll
                    for (int s = 0; s < kTileTc / 16; ++s) mma_f16<true>(d, a + s * 8, b + ((s * 2048) >> 4), id_pv, s > 0 ? 1 : more);
                    tc_commit(o_bar + 8 * (nv & 1));
                    tc_commit(empties + 8 * vs);
                }
                __syncwarp();
                ++nv;
                advance(vs, vph, kAdvance);
                if (i + 1 < mine) v_there = mbar_test(fulls + 8 * vs, vph);
                if (i + 2 < mine) {
                    if (!__all_sync(0xffffffffu, k_there)) wait(fulls + 8 * ks, kph, 42);
                    qk();
                }
            }
            bar_arrive_named(2, 320);                                            // this warp has seen the piece's q: the next may come (also after a wait that ran out)
            piece = end;
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ---------------------------------------------------------------------- softmax of stream x
        const int x = (warp >> 2) - 1, quarter = warp & 3, r = quarter * 32 + lane, wg = tid - 128 - x * 128;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, ts = tmem + x * 128 + lanes, to = tmem + 256 + x * 128 + lanes;
        const uint32_t s_bar = smem_u32(&s_full[x][0]), o_bar = smem_u32(&o_full[x][0]);
        uint32_t count = 0, which = 0;                                           // this stream's tiles so far; piece parity
        for (int piece = u0; piece < u1; which ^= 1) {
            while (piece >= job.begin + job.nt) job.next(p);
            const int end = min(u1, job.begin + job.nt), tiles = end - piece;
            const int b = job.b, kvh = job.job / p.nrb, row0 = (job.job - kvh * p.nrb) * kJobRows, len = job.len, n = entries(p, len);
            const bool whole = piece == job.begin && end == job.begin + job.nt;
            const int myrow0 = row0 + (TWO ? x * kRowsTc : 0), row = myrow0 + r;
            const bool warp_live = myrow0 + quarter * 32 < p.R;
            // rows of q; what came before in this CTA is read out of shared and tensor memory
            if (tid == 128) bad[which ^ 1] = 0;                                  // the next piece's; the one before it has been read
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
                *reinterpret_cast<uint4 *>(sm_q + (TWO ? x * kQ : 0) + (c >> 3) * kQHalf + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = qv[i];
            }
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[TWO ? x : 0]));
            const uint64_t seen = row < p.R ? drafted_bits(p, b, token_of(p, row), len) : 0;
            // tiles of this piece that stream 0 and stream 1 have, and the first one of this stream
            const int odd = (piece - u0) & 1;
            const int t0 = TWO ? tiles : (tiles + !odd) / 2, t1 = TWO ? (row0 + kRowsTc < p.R ? tiles : 0) : (tiles + odd) / 2;
            const int mine = x ? t1 : t0, first_tile = TWO ? 0 : x ^ odd;
            float m = -INFINITY, l = 0.0f;
            int i = 0;
            for (; i < mine; ++i, ++count) {
                const int t = TWO ? i : first_tile + 2 * i, key0 = (piece + t - job.begin) * kTileTc;
                const bool tail = key0 + kTileTc > len;
                const uint32_t tile = ts + (count & 1) * kTileTc;
                wait(s_bar + 8 * (count & 1), count >> 1, 46);
                tc_fence_after();
                if (warp_live) {
                    uint32_t s[64];
#pragma unroll
                    for (int j = 0; j < 2; ++j) tc_ld32(tile + j * 32, *reinterpret_cast<uint32_t(*)[32]>(s + j * 32));
                    tc_wait_ld();
                    if (tail) {
                        // a bit for each of 32 entries: committed, or drafted and seen
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int j0 = key0 + j * 32 - len;
                            const uint32_t vis = j0 <= -32 ? ~0u : j0 >= 64 ? 0u : j0 >= 0 ? (uint32_t)(seen >> j0) : ((uint32_t)seen << -j0) | ((1u << -j0) - 1);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(vis & (1u << e))) s[j * 32 + e] = 0xff800000u;
                        }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 64; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(s[e]));
                    const float mx = reference_of<kRaise<BF16>>(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2);
                    if (i == 0) m = mx;
                    else if (__any_sync(0xffffffffu, (mx > m + kLag || m == -INFINITY) && mx != m)) {
                        // the product before this one has to be done (the one before that is: these scores were made behind it)
                        wait(o_bar + 8 * ((count - 1) & 1), (count - 1) >> 1, 49);
                        tc_fence_after();
                        const float up = fmaxf(m, mx), f = m == -INFINITY ? 0.0f : exp2_approx(m - up);
                        l *= f;
                        m = up;
#pragma unroll 1
                        for (int j = 0; j < D / 32; ++j) {
                            uint32_t o[32];
                            tc_ld32(to + j * 32, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tc_st16(to + j * 32, o);
                            tc_st16(to + j * 32 + 16, o + 16);
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : -m;
                    const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2), base2 = pack2(base, base);
                    uint64_t sum2[4] = {};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float e0, e1;
                            unpack2(fma2(pack2(__uint_as_float(s[j * 32 + 2 * e]), __uint_as_float(s[j * 32 + 2 * e + 1])), scale2, base2), e0, e1);
                            e0 = exp2_approx(e0);
                            e1 = exp2_approx(e1);
                            sum2[e & 3] = add2(sum2[e & 3], pack2(e0, e1));
                            w[e] = narrow<BF16>(e0, e1);
                        }
                        tc_st16(tile + j * 16, w);
                    }
                    float a, d;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), a, d);
                    l += a + d;
                    tc_wait_st();
                }
                if (tail) {
                    // values of V that are not finite become zero, of drafted entries and of what lies behind the sequence's end: half a row
                    // a thread, or a quarter where both streams are at this tile.  Then they share the work and wait for one another: each
                    // thread makes its own writes known to the async proxy, and no product begins before all have.
                    const bool both = TWO && row0 + kRowsTc < p.R;
                    const int item = 2 * (piece - u0 + t) + 1, slot = item % kItems, of = both ? 4 : 2, mate = both ? wg + x * 128 : wg, vr = mate / of, at = key0 + vr;
                    const int first_ch = (mate % of) * (D / 8 / of), chunks = D / 8 / of;
                    if (wait(fulls + 8 * slot, item / kItems, 47) && at >= len) {
                        uint8_t *v = smem + slot * kItem + vr * 128;
                        uint32_t odd = 0;                                        // pieces with such a value, a bit each
#pragma unroll
                        for (int j = 0; j < D / 16; ++j) {
                            const int ch = first_ch + j;
                            if (j < chunks) odd |= (uint32_t)any_nonfinite<BF16>(*reinterpret_cast<const uint4 *>(v + (ch >> 3) * kHalf + (((ch & 7) ^ (vr & 7)) << 4))) << j;
                        }
                        if (odd) {
                            if (at < n) atomicOr(&bad[which], 1ull << (at - len));
                            for (int j = 0; j < chunks; ++j) {
                                const int ch = first_ch + j;
                                uint4 *q = reinterpret_cast<uint4 *>(v + (ch >> 3) * kHalf + (((ch & 7) ^ (vr & 7)) << 4));
                                const uint4 w = *q;
                                *q = make_uint4(finite2<BF16>(w.x), finite2<BF16>(w.y), finite2<BF16>(w.z), finite2<BF16>(w.w));
                            }
                            fence_proxy_async();
                        }
                    }
                    if (both) bar_sync_named(1, 256);                            // (reached by both for every such tile, also after a wait that ran out)
                }
                tc_fence_before();
                bar_arrive_named(3 + 2 * x + (count & 1), 160);
            }
            // ------------------------------------------------------------------ the piece's result
            const long part = 2L * blockIdx.x + (piece != u0);
            float top = m, sum = l, f0 = 1.0f, f1 = 0.0f;
            int col0 = 0, cols = D;
            bool have0 = true, have1 = false;
            // the stream's last product; the one before it on the same barrier is done, its scores were made behind that
            if (mine) wait(o_bar + 8 * ((count - 1) & 1), (count - 1) >> 1, 48);
            if (!TWO) {
                have0 = t0 > 0;
                have1 = t1 > 0;
                // each thread's maximum and sum to the other stream's thread of the same row, through the tile of scores in tensor memory
                tc_st2(ts, __float_as_uint(m), __float_as_uint(l));
                tc_wait_st();
                tc_fence_before();
                bar_sync_named(1, 256);
                tc_fence_after();
                uint32_t ml[4];
                tc_ld2(tmem + lanes, ml[0], ml[1]);
                tc_ld2(tmem + 128 + lanes, ml[2], ml[3]);
                tc_wait_ld();
                const float2 a = make_float2(__uint_as_float(ml[0]), __uint_as_float(ml[1])), d = make_float2(__uint_as_float(ml[2]), __uint_as_float(ml[3]));
                top = fmaxf(a.x, d.x);
                const float base = top == -INFINITY ? 0.0f : top;
                f0 = exp2_approx(a.x - base);
                f1 = exp2_approx(d.x - base);
                sum = a.y * f0 + d.y * f1;
                cols = D / 2;
                col0 = x * cols;
            }
            tc_fence_after();
            const uint64_t nonfinite = bad[which];
            if (warp_live && ok) {
                const float factor = row_factor(sum, len == 0 && !seen), base = top == -INFINITY ? 0.0f : top;
#pragma unroll 1
                for (int c0 = col0; c0 < col0 + cols; c0 += 32) {
                    uint32_t a[32], o[32];
                    if (have0) tc_ld32((TWO ? to : tmem + 256 + lanes) + c0, a);
                    if (have1) tc_ld32(tmem + 384 + lanes + c0, o);
                    tc_wait_ld();
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        v[e] = have0 ? __uint_as_float(a[e]) * f0 : 0.0f;
                        if (have1) v[e] += __uint_as_float(o[e]) * f1;
                    }
                    if (nonfinite && row < p.R)
                        for (int d = 0; d < 32; ++d) {
                            // (registers are not indexed by a variable: the sum goes to where its turn is)
                            const float add = nonfinite_part<BF16>(p, nonfinite, seen, b, kvh, row, c0 + d, len, base);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (e == d) v[e] += add;
                        }
                    if (!whole) {
                        float *dst = p.part_o + part * kJobRows * D + ((c0 >> 2) * kJobRows + (row - row0)) * 4;
                        if (row < p.R) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4 *>(dst + e * kJobRows) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                        }
                    } else {
                        // through the rows' own place in the buffer of q, which is not read any more: a warp then writes whole lines
                        uint8_t *dst = sm_q + (TWO ? x * kQ : 0) + (c0 >> 6) * kQHalf + r * 128;
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            *reinterpret_cast<uint4 *>(dst + (((((c0 & 32) + e) >> 3) ^ (r & 7)) << 4)) =
                                make_uint4(narrow<BF16>(v[e] * factor, v[e + 1] * factor), narrow<BF16>(v[e + 2] * factor, v[e + 3] * factor),
                                           narrow<BF16>(v[e + 4] * factor, v[e + 5] * factor), narrow<BF16>(v[e + 6] * factor, v[e + 7] * factor));
                    }
                }
                if (whole) {
                    __syncwarp();
                    constexpr int kPieces = (TWO ? D : D / 2) / 8, kRowsAtOnce = 32 / kPieces;       // of 16 bytes, of this warp's rows
                    const int piece_of = col0 / 8 + lane % kPieces;
#pragma unroll
                    for (int i = 0; i < 32; i += kRowsAtOnce) {
                        const int rr = quarter * 32 + i + lane / kPieces, orow = myrow0 + rr, os = token_of(p, orow), oh = kvh * p.g + orow - os * p.g;
                        const uint4 w = *reinterpret_cast<const uint4 *>(sm_q + (TWO ? x * kQ : 0) + (piece_of >> 3) * kQHalf + rr * 128 + (((piece_of & 7) ^ (rr & 7)) << 4));
                        if (orow < p.R) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + (((long)b * p.S + os) * p.nh + oh) * D + piece_of * 8) = w;
                    }
                }
                if (row < p.R && col0 == 0) {
                    if (!whole) p.part_ml[part * kJobRows + (row - row0)] = make_float2(top, sum);
                    else if (p.lse) p.lse[((long)b * p.nkv + kvh) * p.R + row] = base + log2f(sum);
                }
            }
            // both streams have read what the next piece overwrites: O of either, the exchanged sums, the marks of V
            tc_fence_before();
            bar_sync_named(2, 320);
            piece = end;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// weights += sum over the rows of 2^(score - lse) for more rows than leave their scores (attn_tree.cu), from K and q again: S^T = K Q^T, an
// entry per lane of tensor memory and a row per column, so that a thread adds up its entry's weights with nothing to exchange.  A
// CTA (two an SM) has some of the heads' tiles of 128 entries, divided by the lengths as those of the attention are, 128 rows at a time; K is
// loaded, multiplied and added up in a pipeline of two tiles.  What bounds it is one exponential for each score, 16 a clock and SM, or K; as mma.sync, where every warp reads all
// rows for its 16 entries, 64 rows x 254,000 entries took 28 us (17 so, of which K's 65 MB are 10).
constexpr int kWeightTile = 128, kThreadsWeights = 256, kWeightGroup = 8;
template <int D> constexpr int smem_weights() { return 1024 + (2 * kWeightTile + kRowsTc) * D * 2; }
// COUNTED: of p.counted rows only (the number of rows in a register instead of a constant costs 0.5 us).
template <int D, bool BF16, bool COUNTED>
__global__ void __launch_bounds__(kThreadsWeights, 2) attn_weights_tc_kernel(const __grid_constant__ TreeAttnParams p, const __grid_constant__ CUtensorMap kmap) {
    constexpr int kTileBytes = kWeightTile * D * 2, kHalf = kWeightTile * 128, kBox = kTreeTcTile * 128;         // a box of the map is 64 entries high
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023), *sm_q = smem + 2 * kTileBytes;
    __shared__ uint64_t full[2], empty[2], s_full[2], s_free[2];
    __shared__ uint32_t seen[64][kRowsTc / 32];                                  // of drafted entry j: the rows that see it, a bit each
    __shared__ __align__(16) float lse[kRowsTc];
    __shared__ float so_far[kWeightGroup][kWeightTile];                          // an entry's sum over the rows before, its thread's own
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&full[i]), 1); mbar_init(smem_u32(&empty[i]), 1); mbar_init(smem_u32(&s_full[i]), 1); mbar_init(smem_u32(&s_free[i]), 4); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // the lengths may be read here: the kernel before this one is the attention or the join of the same call, which lets this one start when
    // it has itself waited for all that came before the call
    JobWalk<kWeightTile> job;
    int u0, u1;
    take_share(p, lane, job, u0, u1);
    pdl_wait();
    pdl_trigger();
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t phase, int code) {
        if (ok) ok = mbar_wait_warp(g_status_attn_tc, smem_u32(bar), phase & 1, &abort_flag, code);
    };
    uint32_t it = 0;                                                             // tiles so far, of all rows
    for (int piece = u0, piece_end; piece < u1; piece = piece_end) {
    while (piece >= job.begin + job.nt) job.next(p);
    piece_end = min(u1, job.begin + job.nt);
    const int b = job.b, kvh = job.job, bh = b * p.nkv + kvh, len = job.len, n = entries(p, len), first = piece - job.begin, last = piece_end - job.begin;
    // with more rows than 128 a few tiles at a time, so that an entry's sum over all of them is added to its weight once
    const int rows = COUNTED ? counted_rows(p, b) : p.R, group = rows > kRowsTc ? kWeightGroup : 1 << 20;
    for (int g0 = first; g0 < last; g0 += group)
    for (int row0 = 0; row0 < rows; row0 += kRowsTc) {
        const int g1 = min(g0 + group, last);
        __syncthreads();                                                         // the rows before have been multiplied and looked at
        constexpr int kStep = kThreadsWeights / (D / 8), kLoads = kRowsTc / kStep;
        const int c = tid % (D / 8), r_of = tid / (D / 8);
        uint4 q[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            q[i] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + q_offset(p, b, kvh, min(row0 + r_of + i * kStep, p.R - 1)) + c * 8);
        if (tid < kRowsTc) {
            const int row = row0 + tid;
            const uint64_t bits = row < rows ? drafted_bits(p, b, token_of(p, row), len) : 0;
            if (last * kWeightTile > len) {                                      // some of the drafted entries are this CTA's
#pragma unroll 8
                for (int j = 0; j < 64; ++j) {
                    const uint32_t seeing = __ballot_sync(0xffffffffu, (bits >> j) & 1);
                    if (lane == 0) seen[j][warp] = seeing;
                }
            }
            // rows that do not count or see nothing have no weight anywhere
            lse[tid] = row >= rows || (len == 0 && !bits) ? INFINITY : p.lse[(long)bh * p.R + row];
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = r_of + i * kStep;
            *reinterpret_cast<uint4 *>(sm_q + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = q[i];
        }
        fence_proxy_async();
        __syncthreads();
        const int cols = (min(rows - row0, kRowsTc) + 15) / 16 * 16;
        if (warp == 0) {
            for (int tile = g0; tile < g1; ++tile, ++it) {
                const int slot = it & 1;
                wait(&empty[slot], (it >> 1) ^ 1, 61);
                if (ok && elect_one()) {
                    const uint32_t bar = smem_u32(&full[slot]), dst = smem_u32(smem + slot * kTileBytes);
                    mbar_expect_tx(bar, kTileBytes);
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
                        tma_load_tile(dst + (i >> 1) * kHalf + (i & 1) * kBox, &kmap, (i >> 1) * 64, tile * kWeightTile + (i & 1) * kTreeTcTile, bh, bar);
                }
                __syncwarp();
            }
        } else if (warp == 1) {
            const uint32_t fmt = BF16 ? 1u : 0u, idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(kWeightTile >> 4) << 24);
            for (int tile = g0; tile < g1; ++tile, ++it) {
                const int slot = it & 1;
                wait(&full[slot], it >> 1, 62);
                wait(&s_free[slot], (it >> 1) ^ 1, 63);
                tc_fence_after();
                const uint64_t a = make_smem_desc(smem_u32(smem + slot * kTileBytes)), bq = make_smem_desc(smem_u32(sm_q));
                if (ok && elect_one()) {
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint64_t off = ((s >> 2) * kHalf + (s & 3) * 32) >> 4;
                        mma_f16<false>(tmem + slot * kRowsTc, a + off, bq + off, idesc, s > 0);
                    }
                    tc_commit(smem_u32(&s_full[slot]));
                    tc_commit(smem_u32(&empty[slot]));
                }
                __syncwarp();
            }
        } else if (warp >= 4) {
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            float *w = p.weights + (long)bh * p.T;
            for (int tile = g0; tile < g1; ++tile, ++it) {
                const int slot = it & 1, t = tile * kWeightTile + (warp & 3) * 32 + lane, j = t - len;
                const bool done = row0 + kRowsTc >= rows;
                const float was = done && t < n ? w[t] : 0.0f;
                wait(&s_full[slot], it >> 1, 64);
                tc_fence_after();
                float sum[4] = {};
                if (ok) {
#pragma unroll 1
                    for (int c0 = 0; c0 < cols; c0 += 32) {
                        uint32_t s[32];
                        tc_ld32(tmem + slot * kRowsTc + lanes + c0, s);          // (columns behind the rows' are not looked at)
                        tc_wait_ld();
                        const uint32_t hidden = j < 0 ? 0u : j >= 64 ? ~0u : ~seen[j][c0 >> 5];
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 l4 = *reinterpret_cast<const float4 *>(&lse[c0 + e]);
                            const float l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float x = exp2_approx(fmaf(__uint_as_float(s[e + i]), p.scale_log2, -l[i]));
                                sum[i] += l[i] == INFINITY || (hidden & (1u << (e + i))) ? 0.0f : x;
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_free[slot]));
                float &before = so_far[row0 || !done ? tile - g0 : 0][(warp & 3) * 32 + lane];
                const float now = (row0 ? before : 0.0f) + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                if (!done) before = now;
                else if (t < n && ok) w[t] = was + now;
            }
        }
    }
    }
    __syncwarp();
    if (warp == 0)                                                               // as in attn_tc_kernel: nothing is on its way when the CTA leaves
        for (uint32_t i = it > 2 ? it - 2 : 0; i < it && abort_flag; ++i)
            for (int tries = 0; tries < 10000 && !__all_sync(0xffffffffu, mbar_try_hint(smem_u32(&full[i & 1]), (i >> 1) & 1, 20000u)); ++tries);
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
}

template <int D, bool BF16, bool COUNTED>
int launch_weights(const TreeAttnParams &p, const CUtensorMap &km, cudaStream_t stream) {
    auto kern = attn_weights_tc_kernel<D, BF16, COUNTED>;
    constexpr int smem = smem_weights<D>();
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kern), smem, done);
    if (e != cudaSuccess) return cuda_status(e, "tree_attention shared memory");
    // Two CTAs for every SM, but none without a tile; a job is a head here.  Whole heads, as plan_of has whole jobs, where a CTA has few
    // tiles whatever the lengths are (37 sequences of 511 .. 1,000, 8 heads of 40 rows: 51 us with the attention, 57 in equal shares).
    const long heads = (long)p.B * p.nkv, nt = (p.T + kWeightTile - 1) / kWeightTile;
    TreeAttnParams q = p;
    q.nrb = 1;
    q.shares = heads * nt < 2L * kNumSMs ? (int)(heads * nt) : 2 * kNumSMs;
    q.min_share = 1;
    const long each = (heads + q.shares - 1) / q.shares;
    q.split = each * nt - heads * nt / q.shares <= kSecondJob<kWeightTile> && each * nt <= 20 ? kJobs : heads <= q.shares && p.B <= 32 ? kParts : kEven;
    q.jobs_each = (int)each;
    if (q.split == kJobs) q.shares = (int)((heads + each - 1) / each);
    q.parts_of = nullptr;
    return cuda_status(launch_pdl(kern, dim3((unsigned)q.shares), kThreadsWeights, smem, stream, q, km), "tree_attention weights");
}

template <int D, bool TWO, bool BF16>
int launch_tc(const TreeAttnParams &p, const CUtensorMap &km, const CUtensorMap &vm, cudaStream_t stream) {
    auto kern = attn_tc_kernel<D, TWO, BF16>;
    constexpr int smem = smem_tc<D, TWO>();
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(reinterpret_cast<const void *>(kern), smem, done);
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

int launch_attn_weights_tc(const TreeAttnParams &p, bool bf16, const CUtensorMap &km, cudaStream_t stream) {
    auto launch = [&](auto counted) {
        constexpr bool COUNTED = decltype(counted)::value;
        if (p.D == 128) return bf16 ? launch_weights<128, true, COUNTED>(p, km, stream) : launch_weights<128, false, COUNTED>(p, km, stream);
        return bf16 ? launch_weights<64, true, COUNTED>(p, km, stream) : launch_weights<64, false, COUNTED>(p, km, stream);
    };
    return p.counted ? launch(std::true_type()) : launch(std::false_type());
}

int attn_tc_status(int *out) { return cuda_status(cudaMemcpyFromSymbol(out, g_status_attn_tc, sizeof(int) * 4), "attn_tc_status"); }
int attn_tc_status_clear() {
    const int zero[4] = {};
    return cuda_status(cudaMemcpyToSymbol(g_status_attn_tc, zero, sizeof(zero)), "attn_tc_status");
}

}  // namespace flh
