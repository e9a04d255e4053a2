// window_attention_mma_bwd.cu -- gradients of the windowed attention on the tensor cores (bf16, sm_100a).
//
// With P = exp(s - lse) (attention.cuh: RowWeight) and dS = P (dO V^T - delta), delta_i = dO_i . O_i:
//     dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,   dbias[b] = sum of dS over the pairs in bucket b.
// Two kernels, each without atomics: one CTA per 128 queries streams the keys they see (dQ, delta, the
// bucket sums); one CTA per 128 keys streams the queries that see them (dK, dV). Either recomputes S and dP;
// 7 products instead of 5, for results that do not depend on scheduling. TMEM lane r is row r of the CTA;
// two warpgroups share a tile of 64 columns, 32 each (no row statistics are left to find), and go on
// independently: while one waits for its products, the other computes.
// P and dS are rounded to bf16 as operands of the products (the bucket sums take dS before it); against 64 bits
// dQ, dK and dV are then off by 0.0023 to 0.0025, where a result's own rounding alone makes 0.0017.
// Bound, like the forward, by the instructions of the softmax threads (31 to a pair of rows in dQ, 29 in dK and dV, at
// 49 and 45 % of the issue rate; tensor pipe 12 and 17 %; counters of an earlier build). 131072 points, 4 heads of 64,
// window 513, 32 buckets: 1195 us, of which dQ and the bucket sums 600 and dK and dV 576 in a trace.
#include "attention_sinks.cuh"

namespace gdl {
namespace {

using namespace tc;

constexpr int kBwdSoft = 256;               // softmax threads: 8 warps
constexpr int kBwdThreads = kBwdSoft + 32;  // and the warp that loads and issues the products
constexpr int kCols = 32;                   // columns of a tile that one thread handles

__device__ __forceinline__ float dot8(const uint4 &x, const uint4 &y) {
    const uint32_t p[4] = {x.x, x.y, x.z, x.w}, q[4] = {y.x, y.y, y.z, y.w};
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        s = fmaf(__uint_as_float(p[i] << 16), __uint_as_float(q[i] << 16), s);
        s = fmaf(__uint_as_float(p[i] & 0xffff0000u), __uint_as_float(q[i] & 0xffff0000u), s);
    }
    return s;
}

// ------------------------------------------------------------------------------------ dQ, delta, dbias
template <int DP>
struct DqShape {
    static constexpr int panels = DP / 64;
    static constexpr int kstages = 3, vstages = 2;  // (K of the tile before is read until this one's S is done)
    static constexpr uint32_t row_bytes = panels * 128 * 128;      // Q or dO of the CTA
    static constexpr uint32_t tile_bytes = panels * kMmaKeys * 128;  // K or V of one tile
    static constexpr uint32_t q = 0, d = row_bytes, k = 2 * row_bytes, v = k + kstages * tile_bytes;
    static constexpr uint32_t table = v + vstages * tile_bytes;
    static constexpr uint32_t s_col = 0, dp_col = 64, acc_col = 128, tmem_cols = 256;
    static uint32_t smem(int buckets, bool hist) {
        return table + 1024 + buckets * 128 + (hist ? buckets * kBwdSoft * 4 : 0) + 2 * 3 * kMmaKeys * 4 + 256;
    }
};

// Four columns c .. c + 3 of a tile, one row: dS from S (s) and dP (g), and the bucket sums. `bits`: the columns that
// the row sees, where `part` holds. FAR: some row's inv is not 1.
template <bool BIAS, bool HIST, bool FAR>
__device__ __forceinline__ void dq_step(const uint32_t *s, const uint32_t *g, int c, unsigned bits, bool part,
                                        const float *kp, uint64_t scale2, const RowBias &rb, RowWeight rw, float de,
                                        uint32_t mine, uint32_t *pk) {
    const uint64_t up = pack2(rw.shift, rw.shift), dd = pack2(-de, -de);
    unsigned u[4];
    if (BIAS) buckets4(rb, kp, c, u);
    uint64_t x[2];
    logits4<BIAS>(s, scale2, rb, u, x[0], x[1]);
    float ds[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        float p0, p1;
        unpack2(add2(x[e / 2], up), p0, p1);
        if (FAR) {
            p0 = not_above_0(p0);
            p1 = not_above_0(p1);
        }
        unpack2(mul2(pack2(ex2(p0), ex2(p1)), add2(pair(g[e], g[e + 1]), dd)), ds[e], ds[e + 1]);
    }
    if (FAR) {
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[e] *= rw.inv;
    }
    if (part) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(bits >> e & 1)) ds[e] = 0.0f;
    }
    if (HIST) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at = mad(u[e], kBwdSoft * 4, mine);
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v + ds[e]));
        }
    }
    pk[0] = pack_bf16(ds[0], ds[1]);
    pk[1] = pack_bf16(ds[2], ds[3]);
}

template <int DP, bool BIAS, bool HIST>
__global__ void __launch_bounds__(kBwdThreads, DP == 64 ? 2 : 1)
    attn_dq_mma_kernel(const __grid_constant__ gdl_attention a, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_d, const uint16_t *__restrict__ out,
                       const float *__restrict__ lse, const uint16_t *__restrict__ rest, const uint16_t *__restrict__ dout, uint16_t *__restrict__ dq,
                       const RowStats stats, float *__restrict__ part) {
    using S = DqShape<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_addr(smem_raw) & 1023);  // (through no integer: it stays a shared pointer)
    float *table = (float *)(smem + S::table);                      // [buckets][32]
    float *hist = table + (BIAS ? a.buckets : 0) * 32;              // [buckets][256]: a column for each thread
    float *kpos = hist + (HIST ? a.buckets * kBwdSoft : 0);  // [vstages][3][64]
    uint64_t *bars = (uint64_t *)(kpos + 2 * 3 * kMmaKeys);
    __shared__ uint32_t tmem_slot;
    __shared__ int dead, redo;
    __shared__ uint32_t bad_rows[6];
    __shared__ float half_sum[2][128];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x % a.heads;
    const int64_t slot = blockIdx.x / a.heads;
    const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, kMmaRows, slot);
    const int rows = t.cloud == -2 ? 0 : (int)(t.n - t.first < kMmaRows ? t.n - t.first : kMmaRows);
    const int64_t row0 = t.start + t.first;
    int64_t k0 = 0, nk = 0;
    if (t.cloud >= 0) {
        k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
        const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2);
        nk = k1 > k0 ? k1 - k0 : 0;
    }
    const KeyTiles kt = key_tiles(a, t.first + nk - t.n, t.first + rows - 1 + nk - t.n, nk);
    if (t.cloud < 0 || kt.count == 0) {  // nothing to weigh: no gradient
        for (int r = tid; r < rows; r += kBwdThreads) stats.put((int64_t)h * a.n_query + row0 + r, 0.0f, near_weight(neg_inf()));
        zero_rows(dq + (row0 * a.heads + h) * a.dim, (int64_t)a.heads * a.dim, rows, a.dim);
        if (HIST)
            for (int b = tid; b < a.buckets; b += kBwdThreads) part[(slot * a.heads + h) * a.buckets + b] = 0.0f;
        return;
    }

    // barriers: rows (Q, dO), k[stage], v[stage], s[half] (S and dP are done), end (the last product is done),
    // pos[stage] (key positions written), p[half] (dS is written), fix (a tile's values that are not finite
    // replaced), sum (half sums written)
    const uint32_t bar_q = smem_addr(bars), bar_k = bar_q + 8, bar_v = bar_k + 8 * S::kstages,
                   bar_s = bar_v + 8 * S::vstages, bar_end = bar_s + 16, bar_pos = bar_end + 8, bar_p = bar_pos + 16,
                   bar_fix = bar_p + 16, bar_sum = bar_fix + 8;
    if (warp == 8) {
        if (lane == 0) {
            for (uint32_t i = bar_q; i < bar_pos; i += 8) mbar_init(i, 1);
            for (uint32_t i = bar_pos; i < bar_p; i += 8) mbar_init(i, 32);
            for (uint32_t i = bar_p; i < bar_fix; i += 8) mbar_init(i, 128);
            mbar_init(bar_fix, kBwdSoft);
            mbar_init(bar_sum, kBwdSoft);
            mbar_init_fence();
            dead = redo = 0;
            for (int i = 0; i < 6; ++i) bad_rows[i] = 0;
        }
        __syncwarp();
        tmem_alloc(smem_addr(&tmem_slot), S::tmem_cols);
        fence_before();
    }
    if (BIAS) {
        for (int i = tid; i < a.buckets * 32; i += kBwdThreads)
            table[i] = bias2_at(a, (int64_t)h * a.buckets + (i >> 5));
        if (HIST)
            for (int i = tid; i < a.buckets * kBwdSoft; i += kBwdThreads) hist[i] = 0.0f;
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int *vdead = &dead, *vredo = &redo;

    // A second pass, as in the forward: a key that a row does not see may hold what is not finite (0 * NaN in
    // dS K). It is taken for 0; rows that see one get NaN throughout.
    int pass = 0;
    Ring<S::kstages> ring_k;  // every thread's own places in the rings; they go on through a second pass
    Ring<S::vstages> ring_v;
    uint32_t parity = 0;  // of the barriers that turn once a tile
    do {
        if (warp == 8) {
            {
                const bool issue = elect_one();
                const uint32_t base = smem_addr(smem);
                const int hk = h / (a.heads / a.kv_heads);
                const int ksteps = (a.dim + 15) / 16;
                const uint32_t id_s = mma_desc(kCols, false), id_o = mma_desc(ksteps * 16, true);
                Ring<S::kstages> fill_k = ring_k;  // next to load
                Ring<S::vstages> fill_v = ring_v, fill_pos = ring_v;
                KeyTile next_k(kt), next_v(kt);
                auto load = [&](const CUtensorMap *map, uint32_t ring, uint32_t bar, auto &st, KeyTile &t) {
                    if (issue) {
                        mbar_expect(bar + 8 * st.at, S::tile_bytes);
#pragma unroll
                        for (int p = 0; p < S::panels; ++p)
                            tma_load(ring + st.at * S::tile_bytes + p * kMmaKeys * 128, map, bar + 8 * st.at, 64 * p, hk,
                                     (int)k0 + t.j);
                    }
                    st.next();
                    t.next(kt);
                };
                if (pass == 0 && issue) {
                    mbar_expect(bar_q, 2 * S::row_bytes);
#pragma unroll
                    for (int p = 0; p < S::panels; ++p) {
                        tma_load(base + S::q + p * 128 * 128, &map_q, bar_q, 64 * p, h, (int)row0);
                        tma_load(base + S::d + p * 128 * 128, &map_d, bar_q, 64 * p, h, (int)row0);
                    }
                }
                // positions of a tile's keys: two to a lane, read when its V is asked for, written a step later
                float pos[2][3];
                const float *kpos_g = a.pos_k + 3 * k0;
                auto read_pos = [&](const KeyTile &t) {
#pragma unroll
                    for (int e = 0; e < (BIAS ? 2 : 0); ++e) {
                        const int j = t.j + lane + 32 * e;
                        const float *p = kpos_g + 3 * (int64_t)(j < (int)nk ? j : (int)nk - 1);
#pragma unroll
                        for (int x = 0; x < 3; ++x) pos[e][x] = p[x];
                    }
                };
                auto write_pos = [&]() {
                    if (!BIAS) return;
                    float *w = kpos + fill_pos.at * 3 * kMmaKeys + lane;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int x = 0; x < 3; ++x) w[x * kMmaKeys + 32 * e] = pos[e][x];
                    mbar_arrive(bar_pos + 8 * fill_pos.at);
                    fill_pos.next();
                };
                for (int i = 0; i < S::kstages && i < kt.count; ++i) load(&map_k, base + S::k, bar_k, fill_k, next_k);
                for (int i = 0; i < S::vstages && i < kt.count; ++i) {
                    read_pos(next_v);
                    load(&map_v, base + S::v, bar_v, fill_v, next_v);
                    write_pos();
                }
                int out_k = 0, out_v = 0;  // tiles whose K, V have been waited for
                bool ok = mbar_wait(bar_q, 0), pending = false;
                const uint64_t dq_desc = smem_desc(base + S::q), dd_desc = smem_desc(base + S::d);
                Ring<S::kstages> sk = ring_k;  // of the tile whose S and dP come next
                auto products = [&](int half) {  // S and dP of a tile's half
                    if (half == 0) {
                        ok = ok && mbar_wait(bar_k + 8 * sk.at, sk.parity);
                        out_k += ok;
                        ok = ok && mbar_wait(bar_v + 8 * ring_v.at, ring_v.parity);
                        out_v += ok;
                    }
                    if (!ok) return;
                    fence_after();
                    const uint64_t kd = smem_desc(base + S::k + sk.at * S::tile_bytes + half * kCols * 128),
                                   vd = smem_desc(base + S::v + ring_v.at * S::tile_bytes + half * kCols * 128);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + S::s_col + kCols * half, dq_desc + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                               kd + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, id_s, k > 0, issue && k < ksteps);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + S::dp_col + kCols * half, dd_desc + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                               vd + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, id_s, k > 0, issue && k < ksteps);
                    mma_commit(bar_s + 8 * half, issue);
                    if (half == 1) {
                        sk.next();
                        ring_v.next();
                    }
                };
                products(0);
                products(1);
                for (int i = 0; i < kt.count && ok; ++i) {
                    if (pending) write_pos();
                    pending = false;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        ok = ok && mbar_wait(bar_p + 8 * half, parity);
                        if (!ok) break;
                        fence_after();
                        const uint64_t kmn = smem_desc(base + S::k + ring_k.at * S::tile_bytes + half * kCols * 128, kMmaKeys * 128);
#pragma unroll
                        for (int k = 0; k < kCols / 16; ++k)
                            mma_ts(tmem + S::acc_col, tmem + S::s_col + kCols * half + 8 * k, kmn + k * (2048 / 16), id_o,
                                   i > 0 || half > 0 || k > 0, issue);
                        // The products run in the order of their issue: S and dP of the next tile go over this one's
                        if (i + 1 < kt.count) products(half);
                    }
                    if (!ok) break;
                    // Both halves are through with this tile: its V and positions may be overwritten, and the K of the
                    // tile before it, whose last product came before this one's S.
                    if (next_v.i < kt.count) {
                        read_pos(next_v);
                        load(&map_v, base + S::v, bar_v, fill_v, next_v);
                        pending = true;
                    }
                    if (i > 0 && next_k.i < kt.count) load(&map_k, base + S::k, bar_k, fill_k, next_k);
                    ring_k.next();
                    parity ^= 1;
                }
                if (ok) mma_commit(bar_end, issue);
                if (!ok) {  // a wait gave up: let the copies in flight land, then leave
                    *vdead = 1;
                    mbar_wait(bar_q, 0);
                    drain<S::kstages>(bar_k, fill_k, next_k.i - out_k);
                    drain<S::vstages>(bar_v, fill_v, next_v.i - out_v);
                }
            }
            __syncwarp();
        } else {
            const int r = tid & 127, half = tid >> 7;
            const bool live = r < rows;
            const int64_t qi = row0 + (live ? r : rows - 1);
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
            const KeyRange vis = visible_keys(a, qi - t.start + nk - t.n, nk);
            const uint64_t scale2 = pack2(a.scale * kLog2e, a.scale * kLog2e);
            RowBias rb;
            if (BIAS) rb = row_bias(a, a.pos_q + 3 * qi, table);
            const uint32_t mine = smem_addr(hist) + tid * 4 - (HIST ? rb.low : 0) * (kBwdSoft * 4);
            if (HIST && pass > 0)
                for (int e = 0; e < a.buckets; ++e) hist[e * kBwdSoft + tid] = 0.0f;
            const int vis_lo = (int)vis.lo, vis_hi = live ? (int)vis.hi : 0;
            // delta: each of the row's two threads takes every other 8 values
            bool ok = true;
            if (pass == 0) {
                const uint16_t *op = out + (qi * a.heads + h) * a.dim, *gp = dout + (qi * a.heads + h) * a.dim;
                float s = 0.0f;
                for (int d = 8 * half; d < a.dim; d += 16)
                    s += dot8(*reinterpret_cast<const uint4 *>(op + d), *reinterpret_cast<const uint4 *>(gp + d));
                if (rest) {
                    const uint16_t *rp = rest + (qi * a.heads + h) * a.dim;
                    for (int d = 8 * half; d < a.dim; d += 16)
                        s += dot8(*reinterpret_cast<const uint4 *>(rp + d), *reinterpret_cast<const uint4 *>(gp + d));
                }
                half_sum[half][r] = s;
                mbar_arrive(bar_sum);
                ok = mbar_wait(bar_sum, 0);
            }
            const float de = half_sum[0][r] + half_sum[1][r];
            const float ls = lse[(int64_t)h * a.n_query + qi];
            RowWeight rw = near_weight(ls);
            unsigned far = __ballot_sync(0xffffffffu, live && far_lse(ls));
            const bool any_far = far != 0;
            for (; far; far &= far - 1) {
                const RowWeight f = far_weight<uint16_t>(a, h, t.start, t.n, k0, nk, t.first + (warp & 3) * 32 + __ffs(far) - 1);
                if (lane == __ffs(far) - 1) rw = f;
            }
            if (pass == 0 && half == 0 && live) stats.put((int64_t)h * a.n_query + qi, ls == neg_inf() ? 0.0f : de, rw);
            bool sees_bad = false;
            for (KeyTile t_now(kt); t_now.i < kt.count && ok; t_now.next(kt), parity ^= 1, ring_k.next(), ring_v.next()) {
                const float *kp = kpos + ring_v.at * 3 * kMmaKeys;
                if (BIAS) ok = mbar_wait(bar_pos + 8 * ring_v.at, ring_v.parity);
                ok = ok && mbar_wait(bar_s + 8 * half, parity);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (pass > 0) {
                    const uint32_t tile = smem_addr(smem) + S::k + ring_k.at * S::tile_bytes;
                    // the tile is changed under neither half's products: S of both has to be done
                    ok = mbar_wait(bar_k + 8 * ring_k.at, ring_k.parity) && mbar_wait(bar_s + 8 * (half ^ 1), parity);
                    const uint2 bad = zero_nonfinite<S::panels>(tile, bad_rows, bar_fix, t_now.i, tid, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    sees_bad |= ((bad.x & t_now.mask(0, vis_lo, vis_hi, a.num_sinks)) |
                                 (bad.y & t_now.mask(32, vis_lo, vis_hi, a.num_sinks))) != 0;
                }
                unsigned mask = 0xffffffffu;
                ChunkSets cs = {3, 3};
                if (rows < kMmaRows || !t_now.full(kt, a.num_sinks)) {
                    mask = t_now.mask(kCols * half, vis_lo, vis_hi, a.num_sinks);
                    cs = chunk_sets(mask);
                }
                // dS goes over columns of S that this thread alone reads, and has read
                const uint32_t ts = tmem + lane_base + S::s_col + kCols * half, tg = tmem + lane_base + S::dp_col + kCols * half;
                if (any_far) {  // (rare: as little code as it takes)
#pragma unroll 1
                    for (int c = 0; c < kCols; c += 4) {
                        uint32_t s[4], g[4], pk[2];
                        tmem_ld4(ts + c, s);
                        tmem_ld4(tg + c, g);
                        wait_ld();
                        dq_step<BIAS, HIST, true>(s, g, kCols * half + c, mask >> c, true, kp, scale2, rb, rw, de, mine, pk);
                        tmem_st2(ts + c / 2, pk);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kCols / kChunk; ++k) {
                        uint32_t pk[kChunk / 2];
                        if (!(cs.any >> k & 1)) {
#pragma unroll
                            for (int c = 0; c < kChunk / 2; ++c) pk[c] = 0;
                            tmem_st8(ts + kChunk / 2 * k, pk);
                            continue;
                        }
                        uint32_t s[kChunk], g[kChunk];
                        tmem_ld16(ts + kChunk * k, s);
                        tmem_ld16(tg + kChunk * k, g);
                        wait_ld();
                        const unsigned bits = mask >> (kChunk * k);
                        const bool part_seen = !(cs.all >> k & 1);
#pragma unroll
                        for (int c = 0; c < kChunk; c += 4)
                            dq_step<BIAS, HIST, false>(s + c, g + c, kCols * half + kChunk * k + c, bits >> c, part_seen, kp,
                                                       scale2, rb, rw, de, mine, pk + c / 2);
                        tmem_st8(ts + kChunk / 2 * k, pk);
                    }
                }
                wait_st();
                fence_before();
                mbar_arrive(bar_p + 8 * half);
            }
            ok = ok && mbar_wait(bar_end, pass);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) *vdead = 1;
            fence_after();
            // a row's two threads each write half of its groups of 16
            float bad = 0.0f;
            uint16_t *dp = dq + ((row0 + r) * a.heads + h) * a.dim;
            for (int d = 16 * half; d < a.dim; d += 32) {
                uint32_t o[16], w[8];
                tmem_ld16(tmem + lane_base + S::acc_col + d, o);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = __uint_as_float(o[2 * e]) * a.scale, y = __uint_as_float(o[2 * e + 1]) * a.scale;
                    if (d + 2 * e < a.dim) bad = fmaf(x, 0.0f, fmaf(y, 0.0f, bad));
                    if (!ok || sees_bad) x = y = __int_as_float(0x7fc00000);
                    w[e] = pack_bf16(x, y);
                }
                if (live) {
                    *reinterpret_cast<uint4 *>(dp + d) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (d + 8 < a.dim) *reinterpret_cast<uint4 *>(dp + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
            if (live && !(bad == 0.0f)) *vredo = 1;
            fence_before();
        }
        __syncthreads();
        fence_after();
    } while (*vredo && !*vdead && pass++ == 0);
    if (warp == 8) tmem_free(tmem, S::tmem_cols);
    if (HIST) {
        for (int b = warp; b < a.buckets; b += kBwdThreads / 32) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < kBwdSoft / 32; ++k) s += hist[b * kBwdSoft + 32 * k + lane];
            s = warp_sum(s);
            if (lane == 0) part[(slot * a.heads + h) * a.buckets + b] = *vdead ? __int_as_float(0x7fc00000) : s;
        }
    }
    if (tid == 0 && *vdead && a.status) *a.status = GDL_ERR_TIMEOUT;
}

// ------------------------------------------------------------------------------------ dK, dV
template <int DP>
struct DkvShape {
    static constexpr int panels = DP / 64;
    static constexpr int stages = 3;
    static constexpr uint32_t row_bytes = panels * 128 * 128;        // K or V of the CTA
    static constexpr uint32_t tile_bytes = panels * kMmaKeys * 128;  // Q or dO of one tile
    static constexpr uint32_t k = 0, v = row_bytes, q = 2 * row_bytes, d = q + stages * tile_bytes;
    static constexpr uint32_t table = d + stages * tile_bytes;
    static constexpr uint32_t s_col = 0, dp_col = 64, dk_col = 128, dv_col = 128 + DP, tmem_cols = DP == 64 ? 256 : 512;
    static uint32_t smem(int buckets) { return table + 1024 + 2 * buckets * 128 + 2 * 6 * kMmaKeys * 4 + 256; }
};

// Four columns (queries) c .. c + 3 of a tile, one row (key): P and dS from S (s) and dP (g). FAR: some query's inv is
// not 1.
template <bool BIAS, bool FAR>
__device__ __forceinline__ void dkv_step(const uint32_t *s, const uint32_t *g, int c, unsigned bits, bool part,
                                         const float *cp, uint64_t scale2, const RowBias &rb, uint32_t *pk, uint32_t *gk) {
    unsigned u[4];
    if (BIAS) buckets4(rb, cp, c, u);
    uint64_t x[2];
    logits4<BIAS>(s, scale2, rb, u, x[0], x[1]);
    const ulonglong2 ls = *reinterpret_cast<const ulonglong2 *>(cp + 3 * kMmaKeys + c);
    const ulonglong2 de = *reinterpret_cast<const ulonglong2 *>(cp + 4 * kMmaKeys + c);
    float p[4], q[4];
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
        unpack2(add2(x[e / 2], e ? ls.y : ls.x), p[e], p[e + 1]);
        if (FAR) {
            const float i0 = cp[5 * kMmaKeys + c + e], i1 = cp[5 * kMmaKeys + c + e + 1];
            p[e] = ex2(i0 != 1.0f ? not_above_0(p[e]) : p[e]) * i0;
            p[e + 1] = ex2(i1 != 1.0f ? not_above_0(p[e + 1]) : p[e + 1]) * i1;
        } else {
            p[e] = ex2(p[e]);
            p[e + 1] = ex2(p[e + 1]);
        }
        unpack2(mul2(pack2(p[e], p[e + 1]), add2(pair(g[e], g[e + 1]), e ? de.y : de.x)), q[e], q[e + 1]);
    }
    if (part) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(bits >> e & 1)) p[e] = q[e] = 0.0f;
    }
    pk[0] = pack_bf16(p[0], p[1]);
    pk[1] = pack_bf16(p[2], p[3]);
    gk[0] = pack_bf16(q[0], q[1]);
    gk[1] = pack_bf16(q[2], q[3]);
}

template <int DP, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, DP == 64 ? 2 : 1)
    attn_dkv_mma_kernel(const __grid_constant__ gdl_attention a, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ CUtensorMap map_d, const RowStats stats,
                        uint16_t *__restrict__ dk, uint16_t *__restrict__ dv,
                        const SinkPlan sp, int64_t main_ctas) {
    using S = DkvShape<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_addr(smem_raw) & 1023);  // (through no integer: it stays a shared pointer)
    float *table = (float *)(smem + S::table);          // [2][buckets][32], of two heads in turn
    float *cols = table + (BIAS ? 2 * a.buckets : 0) * 32;  // [2][6][64]: x, y, z, shift, -delta, inv of a tile's queries
    uint64_t *bars = (uint64_t *)(cols + 2 * 6 * kMmaKeys);
    __shared__ uint32_t tmem_slot;
    __shared__ int dead, redo;
    __shared__ uint32_t bad_rows[2][6];
    __shared__ int far_tile[2];  // some query's inv is not 1

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.heads / a.kv_heads;
    const SinkUnit u = sink_unit(a, sp, main_ctas, kMmaRows);
    if (u.skip) return;
    const int hk = u.hk, rows = u.rows, first_out = u.first_out;
    const int64_t q0 = u.q0, nq = u.nq, k0 = u.k0, nk = u.nk, j0 = u.j0, lo = u.lo, hi = u.hi;
    float *partial = u.partial;
    const int per_head = hi > lo ? (int)((hi - lo + kMmaKeys - 1) / kMmaKeys) : 0;
    const int count = per_head * group;
    if (count == 0) {
        const int64_t at = ((k0 + j0 + first_out) * a.kv_heads + hk) * a.dim;
        zero_rows(dk + at, (int64_t)a.kv_heads * a.dim, rows - first_out, a.dim);
        zero_rows(dv + at, (int64_t)a.kv_heads * a.dim, rows - first_out, a.dim);
        for (int i = tid; i < first_out * 2 * a.dim; i += kBwdThreads) partial[i] = 0.0f;
        return;
    }

    // barriers: rows (K, V), q[stage], d[stage], s[half] (S and dP are done), end (the last product is done),
    // col[2] (a tile's column values written), p[half] (P and dS are written), fix (two: Q's tile, dO's)
    const uint32_t bar_r = smem_addr(bars), bar_q = bar_r + 8, bar_d = bar_q + 8 * S::stages,
                   bar_s = bar_d + 8 * S::stages, bar_end = bar_s + 16, bar_col = bar_end + 8, bar_p = bar_col + 16,
                   bar_fix = bar_p + 16;
    if (warp == 8) {
        if (lane == 0) {
            for (uint32_t i = bar_r; i < bar_col; i += 8) mbar_init(i, 1);
            for (uint32_t i = bar_col; i < bar_p; i += 8) mbar_init(i, 32);
            for (uint32_t i = bar_p; i < bar_fix; i += 8) mbar_init(i, 128);
            mbar_init(bar_fix, kBwdSoft);
            mbar_init(bar_fix + 8, kBwdSoft);
            mbar_init_fence();
            dead = redo = 0;
            for (int i = 0; i < 12; ++i) bad_rows[i / 6][i % 6] = 0;
        }
        __syncwarp();
        tmem_alloc(smem_addr(&tmem_slot), S::tmem_cols);
        fence_before();
    }
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int *vdead = &dead, *vredo = &redo;

    int pass = 0;  // the second one: as for dQ, with what is not finite in Q and dO taken for 0
    Ring<S::stages> ring;
    Ring<2> ring_col;
    uint32_t parity = 0;  // of the barriers that turn once a tile
    do {
        if (warp == 8) {
            {
                const bool issue = elect_one();
                const uint32_t base = smem_addr(smem);
                const int ksteps = (a.dim + 15) / 16;
                const uint32_t id_s = mma_desc(kCols, false), id_o = mma_desc(ksteps * 16, true);
                Ring<S::stages> fill = ring;
                Ring<2> fill_col = ring_col;
                int loaded = 0, load_c = 0, load_h = hk * group;
                auto load = [&]() {
                    const int z = (int)(q0 + lo) + load_c * kMmaKeys;
                    if (issue) {
                        mbar_expect(bar_q + 8 * fill.at, S::tile_bytes);
                        mbar_expect(bar_d + 8 * fill.at, S::tile_bytes);
#pragma unroll
                        for (int p = 0; p < S::panels; ++p) {
                            const uint32_t at = base + fill.at * S::tile_bytes + p * kMmaKeys * 128;
                            tma_load(at + S::q, &map_q, bar_q + 8 * fill.at, 64 * p, load_h, z);
                            tma_load(at + S::d, &map_d, bar_d + 8 * fill.at, 64 * p, load_h, z);
                        }
                    }
                    fill.next();
                    ++loaded;
                    if (++load_c == per_head) {
                        load_c = 0;
                        ++load_h;
                    }
                };
                if (pass == 0 && issue) {
                    mbar_expect(bar_r, 2 * S::row_bytes);
#pragma unroll
                    for (int p = 0; p < S::panels; ++p) {
                        tma_load(base + S::k + p * 128 * 128, &map_k, bar_r, 64 * p, hk, (int)(k0 + j0));
                        tma_load(base + S::v + p * 128 * 128, &map_v, bar_r, 64 * p, hk, (int)(k0 + j0));
                    }
                }
                // A tile's columns (two queries to a lane) and, with a new head, its table: read a step before they
                // are written, two tiles ahead of their use.
                float val[2][6];
                int read_c = 0, read_h = hk * group;
                const float *pos_g = a.pos_q + 3 * q0;
                auto read_cols = [&]() {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int64_t qc = lo + (int64_t)read_c * kMmaKeys + lane + 32 * e, qi = qc < nq ? qc : nq - 1;
                        const int64_t at = (int64_t)read_h * a.n_query + q0 + qi;
                        val[e][3] = stats.shift(at);
                        val[e][4] = -stats.delta(at);
                        val[e][5] = stats.inv(at);
                        if (BIAS)
#pragma unroll
                            for (int x = 0; x < 3; ++x) val[e][x] = pos_g[3 * qi + x];
                    }
                };
                auto write_cols = [&]() {
                    float *w = cols + fill_col.at * 6 * kMmaKeys + lane;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int x = BIAS ? 0 : 3; x < 6; ++x) w[x * kMmaKeys + 32 * e] = val[e][x];
                    const bool far = __any_sync(0xffffffffu, val[0][5] != 1.0f || val[1][5] != 1.0f);
                    if (lane == 0) far_tile[fill_col.at] = far;
                    if (BIAS && read_c == 0) {
                        float *tw = table + (read_h & 1) * a.buckets * 32 + lane;
#pragma unroll 4
                        for (int e = 0; e < a.buckets; ++e) tw[e * 32] = bias2_at(a, (int64_t)read_h * a.buckets + e);
                    }
                    mbar_arrive(bar_col + 8 * fill_col.at);
                    fill_col.next();
                    if (++read_c == per_head) {
                        read_c = 0;
                        ++read_h;
                    }
                };
                int got = 0, written = 0;  // tiles that have been waited for; tiles whose columns are written
                while (loaded < S::stages && loaded < count) load();
                for (; written < 2 && written < count; ++written) {
                    read_cols();
                    write_cols();
                }
                bool ok = mbar_wait(bar_r, 0), pending = false;
                const uint64_t kd = smem_desc(base + S::k), vd = smem_desc(base + S::v);
                Ring<S::stages> sr = ring;  // of the tile whose S and dP come next
                auto products = [&](int half) {
                    if (half == 0) {
                        ok = ok && mbar_wait(bar_q + 8 * sr.at, sr.parity) && mbar_wait(bar_d + 8 * sr.at, sr.parity);
                        got += ok;
                    }
                    if (!ok) return;
                    fence_after();
                    const uint64_t qd = smem_desc(base + S::q + sr.at * S::tile_bytes + half * kCols * 128),
                                   dd = smem_desc(base + S::d + sr.at * S::tile_bytes + half * kCols * 128);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + S::s_col + kCols * half, kd + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                               qd + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, id_s, k > 0, issue && k < ksteps);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + S::dp_col + kCols * half, vd + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                               dd + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, id_s, k > 0, issue && k < ksteps);
                    mma_commit(bar_s + 8 * half, issue);
                    if (half == 1) sr.next();
                };
                products(0);
                products(1);
                for (int i = 0; i < count && ok; ++i) {
                    if (pending) write_cols();
                    pending = false;
                    const uint32_t tq = base + S::q + ring.at * S::tile_bytes, td = base + S::d + ring.at * S::tile_bytes;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        ok = ok && mbar_wait(bar_p + 8 * half, parity);
                        if (!ok) break;
                        fence_after();
                        const uint64_t qmn = smem_desc(tq + half * kCols * 128, kMmaKeys * 128),
                                       dmn = smem_desc(td + half * kCols * 128, kMmaKeys * 128);
#pragma unroll
                        for (int k = 0; k < kCols / 16; ++k)
                            mma_ts(tmem + S::dv_col, tmem + S::s_col + kCols * half + 8 * k, dmn + k * (2048 / 16), id_o,
                                   i > 0 || half > 0 || k > 0, issue);
#pragma unroll
                        for (int k = 0; k < kCols / 16; ++k)
                            mma_ts(tmem + S::dk_col, tmem + S::dp_col + kCols * half + 8 * k, qmn + k * (2048 / 16), id_o,
                                   i > 0 || half > 0 || k > 0, issue);
                        if (i + 1 < count) products(half);
                    }
                    if (!ok) break;
                    // Both halves are through with this tile's columns, and the last product of the tile before it came
                    // before this one's S: that stage may be refilled.
                    if (written < count) {
                        read_cols();
                        pending = true;
                        ++written;
                    }
                    if (i > 0 && loaded < count) load();
                    ring.next();
                    parity ^= 1;
                }
                ring_col = fill_col;  // (all columns are written: a second pass goes on from there, as their readers do)
                if (ok) mma_commit(bar_end, issue);
                if (!ok) {
                    *vdead = 1;
                    mbar_wait(bar_r, 0);
                    drain<S::stages>(bar_q, fill, loaded - got);
                    drain<S::stages>(bar_d, fill, loaded - got);
                }
            }
            __syncwarp();
        } else {
            const int r = tid & 127, half = tid >> 7;
            const bool live = r < rows;
            const bool idle_warp = (warp & 3) * 32 >= rows;  // no row of this warp is live: its results are not read
            const int64_t j = j0 + (live ? r : rows - 1), kj = k0 + j;
            const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
            const QueryRange vis = visible_queries(a, j, nq, nk);
            const int vis_lo = (int)vis.lo, vis_hi = !live ? 0 : (int)(vis.hi < hi ? vis.hi : hi);
            // queries that every key of this CTA sees: a key behind the sinks may see less than they do
            const int all_lo = (int)visible_queries(a, j0 + rows - 1, nq, nk).lo;
            const int64_t j2 = j0 < a.num_sinks ? (a.num_sinks < j0 + rows - 1 ? a.num_sinks : j0 + rows - 1) : j0;
            const int64_t all = visible_queries(a, j2, nq, nk).hi;
            const int all_hi = (int)(all < hi ? all : hi);
            const uint64_t scale2 = pack2(a.scale * kLog2e, a.scale * kLog2e);
            RowBias rb;
            if (BIAS) rb = row_bias(a, a.pos_k + 3 * kj, table);
            int c0 = (int)lo, head = hk * group;  // first query and head of the tile
            const int lo_i = (int)lo, hi_i = (int)hi;
            const uint32_t tab0 = BIAS ? rb.tab : 0;
            bool ok = true, sees_bad = false;
            for (int i = 0; i < count && ok; ++i, parity ^= 1, ring.next(), ring_col.next()) {
                const float *cp = cols + ring_col.at * 6 * kMmaKeys;
                if (BIAS) rb.tab = tab0 + (head & 1) * a.buckets * 128;
                ok = mbar_wait(bar_col + 8 * ring_col.at, ring_col.parity) && mbar_wait(bar_s + 8 * half, parity);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (pass > 0) {
                    const uint32_t at = smem_addr(smem) + ring.at * S::tile_bytes;
                    // the tiles are changed under neither half's products: S and dP of both have to be done
                    ok = mbar_wait(bar_q + 8 * ring.at, ring.parity) && mbar_wait(bar_d + 8 * ring.at, ring.parity) &&
                         mbar_wait(bar_s + 8 * (half ^ 1), parity);
                    const uint2 bq = zero_nonfinite<S::panels>(at + S::q, bad_rows[0], bar_fix, i, tid, ok);
                    const uint2 bd = zero_nonfinite<S::panels>(at + S::d, bad_rows[1], bar_fix + 8, i, tid, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        sees_bad |= ((w ? bq.y | bd.y : bq.x | bd.x) & bits_below(vis_hi - c0 - 32 * w) &
                                     ~bits_below(vis_lo - c0 - 32 * w)) != 0;
                }
                const bool far = *(volatile int *)&far_tile[ring_col.at] != 0;
                unsigned mask = 0xffffffffu;
                ChunkSets cs = {3, 3};
                if (c0 < all_lo || c0 + kMmaKeys > all_hi) {
                    const int at = c0 + kCols * half;
                    mask = bits_below(vis_hi - at) & ~bits_below(vis_lo - at);
                    cs = chunk_sets(mask);
                }
                if (!idle_warp) {
                    // P and dS go over columns of S and dP that this thread alone reads, and has read
                    const uint32_t ts = tmem + lane_base + S::s_col + kCols * half, tg = tmem + lane_base + S::dp_col + kCols * half;
                    if (far) {  // (rare: as little code as it takes)
#pragma unroll 1
                        for (int c = 0; c < kCols; c += 4) {
                            uint32_t s[4], g[4], pk[2], gk[2];
                            tmem_ld4(ts + c, s);
                            tmem_ld4(tg + c, g);
                            wait_ld();
                            dkv_step<BIAS, true>(s, g, kCols * half + c, mask >> c, true, cp, scale2, rb, pk, gk);
                            tmem_st2(ts + c / 2, pk);
                            tmem_st2(tg + c / 2, gk);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < kCols / kChunk; ++k) {
                            uint32_t pk[kChunk / 2], gk[kChunk / 2];
                            if (!(cs.any >> k & 1)) {
#pragma unroll
                                for (int c = 0; c < kChunk / 2; ++c) pk[c] = 0;
                                tmem_st8(ts + kChunk / 2 * k, pk);
                                tmem_st8(tg + kChunk / 2 * k, pk);
                                continue;
                            }
                            uint32_t s[kChunk], g[kChunk];
                            tmem_ld16(ts + kChunk * k, s);
                            tmem_ld16(tg + kChunk * k, g);
                            wait_ld();
                            const unsigned bits = mask >> (kChunk * k);
                            const bool part_seen = !(cs.all >> k & 1);
#pragma unroll
                            for (int c = 0; c < kChunk; c += 4)
                                dkv_step<BIAS, false>(s + c, g + c, kCols * half + kChunk * k + c, bits >> c, part_seen, cp,
                                                      scale2, rb, pk + c / 2, gk + c / 2);
                            tmem_st8(ts + kChunk / 2 * k, pk);
                            tmem_st8(tg + kChunk / 2 * k, gk);
                        }
                    }
                    wait_st();
                }
                fence_before();
                mbar_arrive(bar_p + 8 * half);
                c0 += kMmaKeys;
                if (c0 >= hi_i) {
                    c0 = lo_i;
                    ++head;
                }
            }
            ok = ok && mbar_wait(bar_end, pass);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) *vdead = 1;
            fence_after();
            // the row's first thread writes dK, the second dV
            const float f = half ? 1.0f : a.scale;
            const uint32_t col = half ? S::dv_col : S::dk_col;
            uint16_t *op = (half ? dv : dk) + ((k0 + j0 + r) * a.kv_heads + hk) * a.dim;
            float bad = 0.0f;
            for (int d = 0; d < a.dim; d += 16) {
                uint32_t o[16], w[8];
                tmem_ld16(tmem + lane_base + col + d, o);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float x = __uint_as_float(o[e]) * f;
                    if (d + e < a.dim) bad = fmaf(x, 0.0f, bad);
                    if (!ok || sees_bad) x = __int_as_float(0x7fc00000);
                    o[e] = __float_as_uint(x);
                }
                if (live && r < first_out) {
                    float *pp = partial + ((int64_t)r * 2 + half) * a.dim + d;
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (d + e < a.dim) pp[e] = __uint_as_float(o[e]);
                } else if (live) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = pack_bf16(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                    *reinterpret_cast<uint4 *>(op + d) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (d + 8 < a.dim) *reinterpret_cast<uint4 *>(op + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
            if (live && !(bad == 0.0f)) *vredo = 1;
            fence_before();
        }
        __syncthreads();
        fence_after();
    } while (*vredo && !*vdead && pass++ == 0);
    if (warp == 8) tmem_free(tmem, S::tmem_cols);
    if (tid == 0 && *vdead && a.status) *a.status = GDL_ERR_TIMEOUT;
}

}  // namespace

// stats of each row; part: the bucket sums of each slot of 128 query rows (nullable); sink_ws: the partial sums of
// chunks of `chunk` queries
int attention_backward_mma(const gdl_attention &a, const uint16_t *out, const float *lse, const uint16_t *rest,
                           const uint16_t *dout, uint16_t *dq, uint16_t *dk, uint16_t *dv, const RowStats stats, float *part, float *sink_ws,
                           int chunk, cudaStream_t st) {
    const int nb = a.bias ? a.buckets : 0;
    const int64_t dh = a.dim, dr = (int64_t)a.heads * a.dim;
    CUtensorMap mq, mk, mv, md;
    if (!head_map(&mq, a.q, a.dim, a.heads, a.n_query, a.q_head, a.q_row, kMmaRows) ||
        !head_map(&mk, a.k, a.dim, a.kv_heads, a.n_key, a.k_head, a.k_row, kMmaKeys) ||
        !head_map(&mv, a.v, a.dim, a.kv_heads, a.n_key, a.v_head, a.v_row, kMmaKeys) ||
        !head_map(&md, dout, a.dim, a.heads, a.n_query, dh, dr, kMmaRows))
        return GDL_ERR_CUDA;
    const int64_t q_ctas = ragged_slots(a.n_query, a.num_clouds, kMmaRows) * a.heads;
    const SinkPlan sp = sink_plan(a, sink_ws, kMmaRows, chunk);
    const int64_t k_ctas = ragged_slots(a.n_key, a.num_clouds, kMmaRows) * a.kv_heads;
    const int64_t s_ctas = sp.tiles * sp.slots * a.kv_heads, top = ((int64_t)1 << 31) - 1;
    GDL_RETURN_IF(q_ctas > top || k_ctas + s_ctas > top, GDL_ERR_OVERFLOW);
    auto go_q = [&](auto kernel, uint32_t smem) -> int {
        GDL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kernel<<<(unsigned)q_ctas, kBwdThreads, smem, st>>>(a, mq, mk, mv, md, out, lse, rest, dout, dq, stats, part);
        GDL_CUDA_TRY(cudaGetLastError());
        return GDL_OK;
    };
    int rc;
    if (a.dim <= 64)
        rc = a.bias ? go_q(part ? attn_dq_mma_kernel<64, true, true> : attn_dq_mma_kernel<64, true, false>,
                           DqShape<64>::smem(nb, part != nullptr))
                    : go_q(attn_dq_mma_kernel<64, false, false>, DqShape<64>::smem(0, false));
    else
        rc = a.bias ? go_q(part ? attn_dq_mma_kernel<128, true, true> : attn_dq_mma_kernel<128, true, false>,
                           DqShape<128>::smem(nb, part != nullptr))
                    : go_q(attn_dq_mma_kernel<128, false, false>, DqShape<128>::smem(0, false));
    if (rc != GDL_OK) return rc;
    if (!head_map(&mq, a.q, a.dim, a.heads, a.n_query, a.q_head, a.q_row, kMmaKeys) ||
        !head_map(&mk, a.k, a.dim, a.kv_heads, a.n_key, a.k_head, a.k_row, kMmaRows) ||
        !head_map(&mv, a.v, a.dim, a.kv_heads, a.n_key, a.v_head, a.v_row, kMmaRows) ||
        !head_map(&md, dout, a.dim, a.heads, a.n_query, dh, dr, kMmaKeys))
        return GDL_ERR_CUDA;
    auto go_k = [&](auto kernel, uint32_t smem) -> int {
        GDL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kernel<<<(unsigned)(k_ctas + s_ctas), kBwdThreads, smem, st>>>(a, mq, mk, mv, md, stats, dk, dv, sp, k_ctas);
        GDL_CUDA_TRY(cudaGetLastError());
        return GDL_OK;
    };
    if (a.dim <= 64)
        rc = a.bias ? go_k(attn_dkv_mma_kernel<64, true>, DkvShape<64>::smem(nb))
                    : go_k(attn_dkv_mma_kernel<64, false>, DkvShape<64>::smem(0));
    else
        rc = a.bias ? go_k(attn_dkv_mma_kernel<128, true>, DkvShape<128>::smem(nb))
                    : go_k(attn_dkv_mma_kernel<128, false>, DkvShape<128>::smem(0));
    if (rc != GDL_OK) return rc;
    return join_sinks<uint16_t>(a, sp, kMmaRows, dk, dv, st);
}

}  // namespace gdl
