// window_attention_mma.cu -- windowed attention on the tensor cores (bf16, sm_100a).
//
// Forward. A CTA owns 128 queries of one head: TMEM lane r and softmax thread r hold query r. One thread
// loads tiles of 64 keys by TMA and issues the products; S = Q K^T goes to TMEM, the softmax threads read
// their row, add the bias, mask, take the running maximum and the sum, and write P over S as the A operand
// of O += P V. P is rounded to bf16 for that product, as the instruction takes two operands of one type; the sum is
// of P before it. The output's error against 64 bits is then 0.0023, where its own rounding alone makes 0.0017. (P in two
// parts, EXACT below, makes it 0.0017 in inference too, for 249 instead of 236 us over 8 ragged scenes and 484 instead
// of 431 in the last case below: not taken there.)
// Only the tiles that some query of the CTA sees are visited: first the sinks', then the span of the windows.
//
// With the bias the kernel is bound by the instructions of the softmax threads (distance, bucket, lookup,
// exponent: 12.6 to a pair of rows in the inner step, 24 in all, at 62 % of the issue rate), not by products
// (13 % of the tensor pipe) or memory: S goes by 32 columns in two buffers, which lets 4 CTAs share an SM. 131072
// points, 4 heads of 64, window 513, 32 buckets: 331 us in inference (the counters are of an earlier build of that),
// 377 in a training step (EXACT, and what rounding the output left over is kept). 2 x 16384 rows, 16 heads of 128 over 4,
// causal window 1024, no bias: 399 us.
#include "attention_mma.cuh"

namespace gdl {
namespace {

using namespace tc;

constexpr int kFwdThreads = 160;  // 4 warps of softmax, 1 warp that loads and issues the products

template <int DP>
struct FwdShape {
    static constexpr int panels = DP / 64;
    static constexpr int stages = 2;                  // tiles of 64 keys (K, V, positions) in flight
    static constexpr int cols = DP == 64 ? 32 : 64;   // keys of one S
    static constexpr int subs = kMmaKeys / cols;      // S's of a tile
    static constexpr int ctas = DP == 64 ? 4 : 2;     // resident CTAs of one SM
    static constexpr uint32_t tmem_cols = DP == 64 ? 128 : 256;
    static constexpr uint32_t o_col = 2 * cols;       // two S's, then O
    static constexpr uint32_t q_bytes = panels * 128 * 128;
    static constexpr uint32_t kv_bytes = panels * kMmaKeys * 128;  // K or V of one tile
    static constexpr uint32_t table = q_bytes + stages * 2 * kv_bytes;
    static uint32_t smem(int buckets) { return table + 1024 + buckets * 128 + stages * 3 * kMmaKeys * 4 + 128; }
};

// EXACT: P goes into the product in two parts, its rounding to bf16 and the rounding of what that left over, so that
// O is as exact as P in 24 bits would make it. A training step with a bias takes it, for delta = dO . O: the bias
// gradient sums dS = P (dP - delta) over all rows, where most of it cancels, and with P in one part delta's error
// is most of what is left (13645 points, 12 heads of 64 over 6, window 1401, 12 buckets: dbias off by 0.0084 instead of 0.0018).
template <int DP, bool BIAS, bool EXACT>
__global__ void __launch_bounds__(kFwdThreads, FwdShape<DP>::ctas)
    attn_fwd_mma_kernel(const __grid_constant__ gdl_attention a, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        uint16_t *__restrict__ out, float *__restrict__ lse, uint16_t *__restrict__ rest) {
    using S = FwdShape<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_addr(smem_raw) & 1023);  // (through no integer: it stays a shared pointer)
    float *table = (float *)(smem + S::table);                 // [buckets][32]: a copy for each lane's bank
    float *kpos = table + (BIAS ? a.buckets : 0) * 32;         // [stages][3][64]
    uint64_t *bars = (uint64_t *)(kpos + S::stages * 3 * kMmaKeys);
    __shared__ uint32_t tmem_slot;
    __shared__ int dead, redo;
    __shared__ uint32_t bad_rows[6];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.x % a.heads;
    const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, kMmaRows, blockIdx.x / a.heads);
    if (t.cloud == -2) return;
    const int rows = (int)(t.n - t.first < kMmaRows ? t.n - t.first : kMmaRows);
    const int64_t row0 = t.start + t.first;  // first global query row
    if (t.cloud == -1) {
        zero_rows(out + (row0 * a.heads + h) * a.dim, (int64_t)a.heads * a.dim, rows, a.dim);
        if (rest) zero_rows(rest + (row0 * a.heads + h) * a.dim, (int64_t)a.heads * a.dim, rows, a.dim);
        if (lse)
            for (int r = tid; r < rows; r += kFwdThreads) lse[(int64_t)h * a.n_query + row0 + r] = neg_inf();
        return;
    }
    const int64_t k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
    const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2);
    const int64_t nk = k1 > k0 ? k1 - k0 : 0;
    const KeyTiles kt = key_tiles(a, t.first + nk - t.n, t.first + rows - 1 + nk - t.n, nk);

    // barriers: q, k[stage], v[stage], pos[stage] (key positions written), s[2] (S is done), p[2] (P is written),
    // o (a product P V is done; all but the last, which a thread that skips its columns could take for the one
    // before it), end (the last one), fix (a tile's values that are not finite replaced)
    const uint32_t bar_q = smem_addr(bars), bar_k = bar_q + 8, bar_v = bar_k + 8 * S::stages, bar_s = bar_v + 8 * S::stages,
                   bar_o = bar_s + 16, bar_end = bar_o + 8, bar_pos = bar_end + 8, bar_p = bar_pos + 8 * S::stages, bar_fix = bar_p + 16;
    if (warp == 4) {
        if (lane == 0) {
            for (uint32_t i = bar_q; i < bar_pos; i += 8) mbar_init(i, 1);
            for (uint32_t i = bar_pos; i < bar_p; i += 8) mbar_init(i, 32);
            for (uint32_t i = bar_p; i <= bar_fix; i += 8) mbar_init(i, 128);
            mbar_init_fence();
            dead = redo = 0;
            for (int i = 0; i < 6; ++i) bad_rows[i] = 0;
        }
        __syncwarp();
        tmem_alloc(smem_addr(&tmem_slot), S::tmem_cols);
        fence_before();
    }
    if (BIAS)
        for (int i = tid; i < a.buckets * 32; i += kFwdThreads)
            table[i] = bias2_at(a, (int64_t)h * a.buckets + (i >> 5));
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int *vdead = &dead, *vredo = &redo;

    // A second pass runs only if a row came out not finite: a value that the row does not see may have done
    // it (0 * NaN in P V). It takes such values of V for 0, and what sees one is computed row by row.
    int pass = 0;
    // every thread's own places in the rings; they go on through a second pass
    Ring<S::stages> ring_k, ring_v;
    Ring<2> ring_s, ring_p;
    do {
    uint32_t parity_o = pass * ((kt.count * S::subs - 1) & 1);  // all but one of a pass turn bar_o
    if (warp == 4) {
        if (kt.count > 0) {
            const uint32_t sq = smem_addr(smem), sk = sq + S::q_bytes, sv = sk + S::stages * S::kv_bytes;
            const int hk = h / (a.heads / a.kv_heads);
            const int ksteps = (a.dim + 15) / 16;
            const uint32_t id_s = mma_desc(S::cols, false), id_o = mma_desc(ksteps * 16, true);
            Ring<S::stages> fill_k = ring_k, fill_v = ring_v, fill_pos = ring_k;  // next to load
            KeyTile next_k(kt), next_v(kt);
            auto load = [&](const CUtensorMap *map, uint32_t ring, uint32_t bar, Ring<S::stages> &st, KeyTile &t) {
                if (lane == 0) {
                    mbar_expect(bar + 8 * st.at, S::kv_bytes);
#pragma unroll
                    for (int p = 0; p < S::panels; ++p)
                        tma_load(ring + st.at * S::kv_bytes + p * kMmaKeys * 128, map, bar + 8 * st.at, 64 * p, hk,
                                 (int)k0 + t.j);
                }
                st.next();
                t.next(kt);
            };
            // positions of a tile's keys: two to a lane, read when its K is asked for, written a step later
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
            if (pass == 0 && lane == 0) {
                mbar_expect(bar_q, S::q_bytes);
#pragma unroll
                for (int p = 0; p < S::panels; ++p) tma_load(sq + p * 128 * 128, &map_q, bar_q, 64 * p, h, (int)row0);
            }
            for (int i = 0; i < S::stages && i < kt.count; ++i) {
                read_pos(next_k);
                load(&map_k, sk, bar_k, fill_k, next_k);
                load(&map_v, sv, bar_v, fill_v, next_v);
                write_pos();
            }
            bool ok = mbar_wait(bar_q, 0), pending = false;
            int out_k = 0, out_v = 0;  // tiles whose K, V have been waited for
            const uint64_t desc_q = smem_desc(sq);
            const bool issue = elect_one();
            const int total = kt.count * S::subs;
            auto scores = [&](int n) {  // S of sub-tile n: Q K^T
                const int sub = n % S::subs;
                if (sub == 0) {
                    ok = ok && mbar_wait(bar_k + 8 * ring_k.at, ring_k.parity);
                    out_k += ok;
                }
                if (ok) {
                    fence_after();
                    const uint64_t db = smem_desc(sk + ring_k.at * S::kv_bytes + sub * S::cols * 128);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        mma_ss(tmem + ring_s.at * S::cols, desc_q + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                               db + (k >> 2) * (kMmaKeys * 128 / 16) + (k & 3) * 2, id_s, k > 0, issue && k < ksteps);
                    mma_commit(bar_s + 8 * ring_s.at, issue);
                }
                if (sub == S::subs - 1) ring_k.next();
                ring_s.next();
            };
            scores(0);
            for (int n = 0; n < total && ok; ++n) {
                const int sub = n % S::subs;
                // The products run in the order of their issue, so S may go over the P that the last P V reads.
                if (n + 1 < total) scores(n + 1);
                if (pending) write_pos();
                pending = false;
                ok = ok && mbar_wait(bar_p + 8 * ring_p.at, ring_p.parity);
                if (ok && sub == 0) {
                    ok = mbar_wait(bar_v + 8 * ring_v.at, ring_v.parity);
                    out_v += ok;
                }
                if (!ok) break;
                fence_after();
                const uint64_t db = smem_desc(sv + ring_v.at * S::kv_bytes + sub * S::cols * 128, kMmaKeys * 128);
#pragma unroll
                for (int k = 0; k < S::cols / 16; ++k) {
                    const uint32_t p = tmem + ring_p.at * S::cols + (EXACT ? (k >> 1) * 32 + (k & 1) * 8 : k * 8);
                    mma_ts(tmem + S::o_col, p, db + k * (2048 / 16), id_o, n > 0 || k > 0, issue);
                    if (EXACT) mma_ts(tmem + S::o_col, p + 16, db + k * (2048 / 16), id_o, true, issue);
                }
                if (sub == S::subs - 1) {
                    // The softmax is done with this tile: its K and positions may be overwritten; so may V of the tile
                    // before it, once the last P V but this one is done.
                    if (next_k.i < kt.count) {
                        read_pos(next_k);
                        load(&map_k, sk, bar_k, fill_k, next_k);
                        pending = true;
                    }
                    if (n >= S::subs && next_v.i < kt.count) {
                        ok = mbar_wait(bar_o, parity_o ^ 1);
                        if (!ok) break;
                        load(&map_v, sv, bar_v, fill_v, next_v);
                    }
                    ring_v.next();
                }
                mma_commit(n + 1 < total ? bar_o : bar_end, issue);
                parity_o ^= 1;
                ring_p.next();
            }
            if (!ok) {  // a wait gave up: let the copies in flight land, then leave
                *vdead = 1;
                mbar_wait(bar_q, 0);
                drain<S::stages>(bar_k, fill_k, next_k.i - out_k);
                drain<S::stages>(bar_v, fill_v, next_v.i - out_v);
            }
        }
        __syncwarp();
    } else {
        const int r = tid;
        const bool live = r < rows;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const KeyRange vis = visible_keys(a, t.first + (live ? r : rows - 1) + nk - t.n, nk);
        const int vis_lo = (int)vis.lo, vis_hi = (int)vis.hi;
        const uint64_t scale2 = pack2(a.scale * kLog2e, a.scale * kLog2e);
        RowBias rb;
        if (BIAS) rb = row_bias(a, a.pos_q + 3 * (row0 + (live ? r : rows - 1)), table);
        float m = neg_inf(), l = 0.0f;
        bool ok = true, sees_bad = false;
        for (KeyTile tile(kt); tile.i < kt.count && ok; tile.next(kt), ring_k.next()) {
            const float *kp = kpos + ring_k.at * 3 * kMmaKeys;
            const bool whole = tile.full(kt, a.num_sinks);
            if (BIAS) ok = mbar_wait(bar_pos + 8 * ring_k.at, ring_k.parity);
#pragma unroll 1  // (half the code: 184 instead of 212 us at 65536 points, the instruction cache)
            for (int sub = 0; sub < S::subs; ++sub) {
                const uint32_t ts = tmem + lane_base + ring_s.at * S::cols;
                ok = ok && mbar_wait(bar_s + 8 * ring_s.at, ring_s.parity);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (pass > 0 && sub == 0) {
                    ok = mbar_wait(bar_v + 8 * ring_k.at, ring_k.parity);
                    const uint2 bad = zero_nonfinite<S::panels>(
                        smem_addr(smem) + S::q_bytes + (S::stages + ring_k.at) * S::kv_bytes, bad_rows, bar_fix, tile.i, r, ok);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    sees_bad |= ((bad.x & tile.mask(0, vis_lo, vis_hi, a.num_sinks)) |
                                 (bad.y & tile.mask(32, vis_lo, vis_hi, a.num_sinks))) != 0;
                }
                // By 32 columns; where no row of the warp sees anything, P = 0. P takes 16 TMEM columns (EXACT: the
                // rest of it the next 16).
#pragma unroll
                for (int w = 0; w < S::cols / 32; ++w) {
                    const int off = sub * S::cols + 32 * w;
                    uint32_t seen = 0xffffffffu, pk[16];
                    const uint32_t tp = ts + (EXACT ? 32 : 16) * w;
                    bool all = true;
                    if (!whole) {
                        seen = tile.mask(off, vis_lo, vis_hi, a.num_sinks);
                        all = __all_sync(0xffffffffu, seen == 0xffffffffu);
                        if (!__any_sync(0xffffffffu, seen != 0)) {
#pragma unroll
                            for (int c = 0; c < 16; ++c) pk[c] = 0;
                            tmem_st16(tp, pk);
                            if (EXACT) tmem_st16(tp + 16, pk);
                            continue;
                        }
                    }
                    uint32_t sr[32];
                    tmem_ld32(ts + 32 * w, sr);
                    wait_ld();
                    uint64_t x[16];
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        unsigned u[4];
                        if (BIAS) buckets4(rb, kp, off + c, u);
                        logits4<BIAS>(sr + c, scale2, rb, u, x[c / 2], x[c / 2 + 1]);
                    }
                    if (!all) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float x0, x1;
                            unpack2(x[c], x0, x1);
                            x[c] = pack2(seen >> (2 * c) & 1 ? x0 : neg_inf(), seen >> (2 * c + 1) & 1 ? x1 : neg_inf());
                        }
                    }
                    float mx[2] = {neg_inf(), neg_inf()};
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        float x0, x1;
                        unpack2(x[c], x0, x1);
                        mx[c & 1] = max3(mx[c & 1], x0, x1);
                    }
                    const float mt = fmaxf(mx[0], mx[1]);
                    // The reference m of the exponents moves only when a row outgrows it by 2^8: P stays below 2^8,
                    // sums stay exact to f32, and O is seldom rescaled. It is a whole number, so that rescaling is
                    // exact.
                    const bool grow = mt > m + 8.0f;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float mn = grow ? (mt < 3.0e38f ? ceilf(mt) : mt) : m;
                        const float f = m == neg_inf() ? 0.0f : ex2(m - mn);
                        l *= f;
                        m = mn;
                        wait_st();  // the half before may have stored P and a rescaled O: both are read back here
                        if (w > 0) {  // the other half's P, already written
#pragma unroll 1
                            for (int part = 0; part < (EXACT ? 2 : 1); ++part) {  // f is a power of two: exact
                                uint32_t q[16];
                                tmem_ld16(ts + 16 * part, q);
                                wait_ld();
#pragma unroll
                                for (int c = 0; c < 16; ++c)
                                    q[c] = pack_bf16(__uint_as_float(q[c] << 16) * f, __uint_as_float(q[c] & 0xffff0000u) * f);
                                tmem_st16(ts + 16 * part, q);
                            }
                        }
                        if (tile.i > 0 || sub > 0) {
                            ok = mbar_wait(bar_o, parity_o ^ 1);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            fence_after();
                            for (int d = 0; d < a.dim; d += 16) {
                                uint32_t o[16];
                                tmem_ld16(tmem + lane_base + S::o_col + d, o);
                                wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st16(tmem + lane_base + S::o_col + d, o);
                            }
                        }
                    }
                    const float base = m == neg_inf() ? 0.0f : m;
                    const uint64_t down = pack2(-base, -base);
                    uint64_t ls[2] = {0, 0};
                    uint32_t pl[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        float p0, p1;
                        unpack2(add2(x[c], down), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        ls[c & 1] = add2(ls[c & 1], pack2(p0, p1));
                        pk[c] = pack_bf16(p0, p1);
                        if (EXACT) {
                            unpack2(fma2(pair(pk[c] << 16, pk[c] & 0xffff0000u), pack2(-1.0f, -1.0f), pack2(p0, p1)), p0, p1);
                            pl[c] = pack_bf16(p0, p1);
                        }
                    }
                    tmem_st16(tp, pk);
                    if (EXACT) tmem_st16(tp + 16, pl);
                    float l0, l1;
                    unpack2(add2(ls[0], ls[1]), l0, l1);
                    l += l0 + l1;
                }
                if (!ok) break;
                wait_st();
                fence_before();
                mbar_arrive(bar_p + 8 * ring_s.at);
                ring_s.next();
                parity_o ^= 1;
            }
        }
        // ------------------------------------------------------------ epilogue
        if (ok && kt.count > 0) ok = mbar_wait(bar_end, pass);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) *vdead = 1;
        fence_after();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float bad = l - l;  // NaN once anything is not finite
        uint16_t *op = out + ((row0 + r) * a.heads + h) * a.dim;
        if (kt.count == 0 || !ok) {
            if (live)
                for (int d = 0; d < a.dim; ++d) {
                    op[d] = ok ? 0 : 0x7fc0;
                    if (rest) rest[((row0 + r) * a.heads + h) * a.dim + d] = 0;
                }
        } else {
            for (int d = 0; d < a.dim; d += 16) {
                uint32_t o[16];
                tmem_ld16(tmem + lane_base + S::o_col + d, o);
                wait_ld();
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = __uint_as_float(o[2 * e]) * inv, y = __uint_as_float(o[2 * e + 1]) * inv;
                    if (d + 2 * e < a.dim) bad = fmaf(x, 0.0f, fmaf(y, 0.0f, bad));
                    w[e] = pack_bf16(x, y);
                }
                if (live) {  // dim is a multiple of 8
                    *reinterpret_cast<uint4 *>(op + d) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (d + 8 < a.dim) *reinterpret_cast<uint4 *>(op + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
                if (live && rest) {
                    uint16_t *rp = rest + ((row0 + r) * a.heads + h) * a.dim + d;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        w[e] = pack_bf16(fmaf(__uint_as_float(o[2 * e]), inv, -__uint_as_float(w[e] << 16)),
                                         fmaf(__uint_as_float(o[2 * e + 1]), inv, -__uint_as_float(w[e] & 0xffff0000u)));
                    *reinterpret_cast<uint4 *>(rp) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (d + 8 < a.dim) *reinterpret_cast<uint4 *>(rp + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
        }
        if (live && lse)
            lse[(int64_t)h * a.n_query + row0 + r] =
                !ok ? __int_as_float(0x7fc00000) : l == 0.0f ? neg_inf() : (m + log2f(l)) * kLn2;
        const bool odd = ok && live && kt.count > 0 && (!(bad == 0.0f) || sees_bad);
        unsigned again = __ballot_sync(0xffffffffu, odd);
        if (pass == 0) {
            if (again && lane == 0) *vredo = 1;
        } else {
            float *strip = (float *)smem + warp * kAttnMaxDim;  // Q's place: the products are done
            while (again) {
                const int e = __ffs(again) - 1;
                again &= again - 1;
                attention_row<uint16_t>(a, h, t.start, t.n, k0, nk, t.first + warp * 32 + e, strip, out, lse, rest);
            }
        }
        fence_before();
    }
    __syncthreads();
    fence_after();
    } while (*vredo && !*vdead && pass++ == 0);
    __syncthreads();
    if (warp == 4) tmem_free(tmem, S::tmem_cols);
    if (tid == 0 && *vdead && a.status) *a.status = GDL_ERR_TIMEOUT;
}

}  // namespace

int attention_forward_mma(const gdl_attention &a, uint16_t *out, float *lse, uint16_t *rest, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    if (!head_map(&mq, a.q, a.dim, a.heads, a.n_query, a.q_head, a.q_row, kMmaRows) ||
        !head_map(&mk, a.k, a.dim, a.kv_heads, a.n_key, a.k_head, a.k_row, kMmaKeys) ||
        !head_map(&mv, a.v, a.dim, a.kv_heads, a.n_key, a.v_head, a.v_row, kMmaKeys))
        return GDL_ERR_CUDA;
    const int64_t ctas = ragged_slots(a.n_query, a.num_clouds, kMmaRows) * a.heads;
    GDL_RETURN_IF(ctas > ((int64_t)1 << 31) - 1, GDL_ERR_OVERFLOW);
    auto go = [&](auto kernel, uint32_t smem) -> int {
        GDL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kernel<<<(unsigned)ctas, kFwdThreads, smem, st>>>(a, mq, mk, mv, out, lse, rest);
        GDL_CUDA_TRY(cudaGetLastError());
        return GDL_OK;
    };
    const int nb = a.bias ? a.buckets : 0;
    if (a.dim <= 64)
        return a.bias ? go(rest ? attn_fwd_mma_kernel<64, true, true> : attn_fwd_mma_kernel<64, true, false>, FwdShape<64>::smem(nb))
                      : go(attn_fwd_mma_kernel<64, false, false>, FwdShape<64>::smem(nb));
    return a.bias ? go(rest ? attn_fwd_mma_kernel<128, true, true> : attn_fwd_mma_kernel<128, true, false>, FwdShape<128>::smem(nb))
                  : go(attn_fwd_mma_kernel<128, false, false>, FwdShape<128>::smem(nb));
}

}  // namespace gdl
