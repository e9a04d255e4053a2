// window_attention_simt.cu -- windowed attention and its gradients in f32 arithmetic, by tiles (sm_100a): f32
// inputs, and bf16 ones in layouts that TMA cannot read.
//
// f32 products have no tensor-core form of their precision, so these kernels are bound by FFMA: a CTA of 128
// threads holds 64 rows against tiles of 32 columns, each thread a 4 x 4 block of the products (two 16-byte
// shared-memory reads to 16 FFMA) and 4 x (dim / 8) of the outputs. Tiles lie transposed ([dim][row]) where
// they are summed over dim, as they are where they are summed over rows. What is not finite does not go into a
// tile (0 times it would reach other rows): a row of the CTA that has such a value, or that sees a column (a key; in
// the dK, dV kernel a query) with one, is computed again, by itself, from what it sees.
// 6 ragged clouds up to 1023 rows, 4 heads of 24 over 2, window 129, 16 buckets, f32: 48 us forward, 62 us dQ, 94 us dK and dV, far from what the FFMA take: 232 CTAs of 4 warps.
#include "attention_sinks.cuh"

namespace gdl {
namespace {

constexpr int kRows = 64, kCols = 32, kThreads = 128;
constexpr int kRowLd = kRows + 4, kColLd = kCols + 4;  // (16-byte rows, odd multiple of 16 bytes)

// 32 rows of a [rows][heads][dim] tensor on their way into tiles: all loads of a thread first, then the stores.
// Rows from n on are 0, and so are values that are not finite, whose rows are marked.
template <typename T, int D>
struct Load {
    float v[D / 4];
    __device__ __forceinline__ void read(const T *p, int64_t row_stride, int n, int dim) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const T *row = p + lane * row_stride + warp;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) v[i] = lane < n && warp + 4 * i < dim ? load1(row + 4 * i) : 0.0f;
    }
    // into [D][ld] (across) and / or [32][D + 4] (along)
    __device__ __forceinline__ void write(float *across, int ld, float *along, uint32_t *bad) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
            const int d = warp + 4 * i;
            float x = v[i];
            if (!(fabsf(x) <= 3.4028234e38f)) {
                odd = true;
                x = 0.0f;
            }
            if (across) across[d * ld + lane] = x;
            if (along) along[lane * (D + 4) + d] = x;
        }
        if (odd) atomicOr(bad, 1u << lane);
    }
};
// The CTA's own rows; bad[2] takes those that are not finite.
template <typename T, int D>
__device__ __forceinline__ void load_rows(const T *p, int64_t row_stride, int n, int dim, float *across, uint32_t *bad) {
#pragma unroll 1
    for (int half = 0; half < kRows / 32; ++half) {
        Load<T, D> l;
        l.read(p + half * 32 * row_stride, row_stride, n - half * 32, dim);
        l.write(across + half * 32, kRowLd, nullptr, bad + half);
    }
}
// Positions of the n columns of a tile: a value to a thread.
__device__ __forceinline__ float read_point(const float *p, int n) {
    const int i = threadIdx.x;
    return i < 3 * kCols && i / 3 < n ? __ldg(p + i) : 0.0f;
}
__device__ __forceinline__ void write_point(float v, float *pos) {
    const int i = threadIdx.x;
    if (i < 3 * kCols) pos[i % 3 * kCols + i / 3] = v;
}
// Whether a tile is read while the one before it is computed: where the registers hold both.
template <int D>
constexpr bool kAhead = D <= 32;

// acc[4][4] += A^T B over dim: rows ty * 4 .., columns tx * 4 ..
__device__ __forceinline__ void product(const float *A, const float *B, int DPAD, int ty, int tx, float (&acc)[4][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
#pragma unroll 16
    for (int d = 0; d < DPAD; ++d) {
        const float4 x = *reinterpret_cast<const float4 *>(A + d * kRowLd + ty * 4);
        const float4 y = *reinterpret_cast<const float4 *>(B + d * kColLd + tx * 4);
        const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[i], ys[j], acc[i][j]);
    }
}

// out[4][D / 8] += P^T V over the tile's columns: P [kCols][kRowLd], V [kCols][D + 4]; values tx * 4 + 32 g ..
template <int D>
__device__ __forceinline__ void gather(const float *P, const float *V, int ty, int tx, float (&out)[4][D / 8]) {
#pragma unroll 8
    for (int c = 0; c < kCols; ++c) {
        const float4 x = *reinterpret_cast<const float4 *>(P + c * kRowLd + ty * 4);
        const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int g = 0; g < D / 32; ++g) {
            const float4 y = *reinterpret_cast<const float4 *>(V + c * (D + 4) + tx * 4 + 32 * g);
            const float ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) out[i][4 * g + j] = fmaf(xs[i], ys[j], out[i][4 * g + j]);
        }
    }
}

__device__ __forceinline__ float sum8(float v) {  // over the 8 threads of a row block
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float max8(float v) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// keys (or queries) of a loop over tiles of kCols: first [0, sinks), then [lo, hi)
struct Span {
    int64_t sinks, lo, hi, j, end;
    __device__ __forceinline__ Span(int64_t s, int64_t l, int64_t h) : sinks(s), lo(l), hi(h), j(s > 0 ? 0 : l), end(s > 0 ? s : h) {}
    __device__ __forceinline__ bool more() const { return j < end; }
    __device__ __forceinline__ void next() {
        j += kCols;
        if (j >= end && end == sinks && sinks > 0) {
            j = lo;
            end = hi;
            sinks = 0;
        }
    }
};

template <int D>
constexpr size_t fwd_smem(int nb) {
    return (size_t)(D * kRowLd + D * kColLd + kCols * (D + 4) + kCols * kRowLd + nb) * 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_simt_kernel(const __grid_constant__ gdl_attention a, T *__restrict__ out,
                                                             float *__restrict__ lse, T *__restrict__ rest) {
    extern __shared__ __align__(16) float sm[];
    float *Q = sm, *K = Q + D * kRowLd, *V = K + D * kColLd, *P = V + kCols * (D + 4), *table = P + kCols * kRowLd;
    __shared__ uint32_t bad;
    __shared__ uint32_t again[2];
    __shared__ float pos[3 * kCols];
    const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
    const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, kRows, blockIdx.x);
    if (t.cloud == -2) return;
    const int rows = (int)(t.n - t.first < kRows ? t.n - t.first : kRows);
    const int64_t row0 = t.start + t.first;
    if (t.cloud == -1) {
        for (int i = tid; i < rows * a.dim; i += kThreads) {
            const int64_t at = ((row0 + i / a.dim) * a.heads + h) * a.dim + i % a.dim;
            store_rest(out + at, rest ? rest + at : nullptr, 0.0f);
        }
        if (lse)
            for (int r = tid; r < rows; r += kThreads) lse[(int64_t)h * a.n_query + row0 + r] = neg_inf();
        return;
    }
    const int64_t k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
    const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2), nk = k1 > k0 ? k1 - k0 : 0;
    const int64_t off = nk - t.n;
    if (tid < 2) again[tid] = 0;
    __syncthreads();
    load_rows<T, D>((const T *)a.q + row0 * a.q_row + (int64_t)h * a.q_head, a.q_row, rows, a.dim, Q, again);
    if (a.bias)
        for (int i = tid; i < a.buckets; i += kThreads) table[i] = bias2_at(a, (int64_t)h * a.buckets + i);
    int vis_lo[4], vis_hi[4];  // places within a cloud fit 32 bits
    float m[4], l[4], o[4][D / 8], px[4], py[4], pz[4];
    bool seen_bad[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i < rows ? ty * 4 + i : rows - 1;
        const KeyRange vis = visible_keys(a, t.first + r + off, nk);
        vis_lo[i] = (int)vis.lo;
        vis_hi[i] = ty * 4 + i < rows ? (int)vis.hi : 0;
        m[i] = neg_inf();
        l[i] = 0.0f;
        seen_bad[i] = false;
        px[i] = py[i] = pz[i] = 0.0f;
        if (a.bias) {
            px[i] = a.pos_q[3 * (row0 + r)];
            py[i] = a.pos_q[3 * (row0 + r) + 1];
            pz[i] = a.pos_q[3 * (row0 + r) + 2];
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[i][d] = 0.0f;
    }
    const KeyRange first = visible_keys(a, t.first + off, nk), last = visible_keys(a, t.first + rows - 1 + off, nk);
    int64_t sinks = a.num_sinks < first.lo ? a.num_sinks : first.lo;
    if (sinks > last.hi) sinks = last.hi;
    const float scale2 = a.scale * kLog2e;
    Load<T, D> lk, lv;
    float lp = 0.0f;
    auto read = [&](const Span &s) {
        const int n = (int)(s.end - s.j < kCols ? s.end - s.j : kCols);
        lk.read((const T *)a.k + (k0 + s.j) * a.k_row + (int64_t)hk * a.k_head, a.k_row, n, a.dim);
        lv.read((const T *)a.v + (k0 + s.j) * a.v_row + (int64_t)hk * a.v_head, a.v_row, n, a.dim);
        if (a.bias) lp = read_point(a.pos_k + 3 * (k0 + s.j), n);
    };
    Span s(sinks, first.lo, last.hi);
    if (kAhead<D> && s.more()) read(s);
    for (Span ahead = s; s.more(); s = ahead) {
        const int n = (int)(s.end - s.j < kCols ? s.end - s.j : kCols);
        ahead.next();
        __syncthreads();
        if (tid == 0) bad = 0;
        __syncthreads();
        if (!kAhead<D>) read(s);
        lk.write(K, kColLd, nullptr, &bad);
        lv.write(nullptr, 0, V, &bad);
        write_point(lp, pos);
        if (kAhead<D> && ahead.more()) read(ahead);
        __syncthreads();
        float x[4][4];
        product(Q, K, D, ty, tx, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mt = neg_inf();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = tx * 4 + j;
                const int key = (int)s.j + c;
                bool see = c < n && key < vis_hi[i] && (key >= vis_lo[i] || key < a.num_sinks);
                if (see && (bad >> c & 1)) {
                    seen_bad[i] = true;
                    see = false;
                }
                float v = x[i][j] * scale2;
                if (a.bias && see) {
                    v += table[distance_bucket(a, px[i], py[i], pz[i], pos[c], pos[kCols + c], pos[2 * kCols + c])];
                }
                x[i][j] = see ? v : neg_inf();
                mt = fmaxf(mt, x[i][j]);
            }
            mt = max8(mt);
            const float mn = fmaxf(m[i], mt), base = mn == neg_inf() ? 0.0f : mn, f = ex2(m[i] - base);
            m[i] = mn;
            float ps = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = ex2(x[i][j] - base);
                ps += x[i][j];
            }
            l[i] = l[i] * f + sum8(ps);
#pragma unroll
            for (int d = 0; d < D / 8; ++d) o[i][d] *= f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4 *>(P + (tx * 4 + j) * kRowLd + ty * 4) = make_float4(x[0][j], x[1][j], x[2][j], x[3][j]);
        __syncthreads();
        gather<D>(P, V, ty, tx, o);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        if (r >= rows) continue;
        const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
        const int64_t at = ((row0 + r) * a.heads + h) * a.dim + tx * 4;
#pragma unroll
        for (int g = 0; g < D / 32; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (tx * 4 + 32 * g + j < a.dim)
                    store_rest(out + at + 32 * g + j, rest ? rest + at + 32 * g + j : nullptr, o[i][4 * g + j] * inv);
        if (tx == 0 && lse) lse[(int64_t)h * a.n_query + row0 + r] = l[i] == 0.0f ? neg_inf() : (m[i] + log2f(l[i])) * kLn2;
        if (seen_bad[i]) atomicOr(again + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int r = tid >> 5; r < rows; r += kThreads / 32)
        if (again[r >> 5] >> (r & 31) & 1)
            attention_row<T>(a, h, t.start, t.n, k0, nk, t.first + r, P + (tid >> 5) * kAttnMaxDim, out, lse, rest);
}

template <int D>
constexpr size_t dq_smem(int nb, bool hist) {
    return (size_t)(2 * D * kRowLd + 2 * D * kColLd + kCols * (D + 4) + kCols * kRowLd + nb + (hist ? nb * kThreads : 0)) * 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
    attn_simt_dq_kernel(const __grid_constant__ gdl_attention a, const T *__restrict__ out, const float *__restrict__ lse,
                        const T *__restrict__ rest, const T *__restrict__ dout, T *__restrict__ dq, const RowStats stats,
                        float *__restrict__ part) {
    extern __shared__ __align__(16) float sm[];
    float *Q = sm, *G = Q + D * kRowLd, *K = G + D * kRowLd, *V = K + D * kColLd, *Kr = V + D * kColLd,
          *P = Kr + kCols * (D + 4), *table = P + kCols * kRowLd, *hist = table + (a.bias ? a.buckets : 0);
    __shared__ uint32_t bad;
    __shared__ uint32_t again[2];
    __shared__ float row_delta[kRows], row_shift[kRows], row_inv[kRows], pos[3 * kCols];
    __shared__ int far;  // some row's inv is not 1
    const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
    const int lane = tid & 31, warp = tid >> 5;
    const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, kRows, blockIdx.x);
    const int rows = t.cloud == -2 ? 0 : (int)(t.n - t.first < kRows ? t.n - t.first : kRows);
    const int64_t row0 = t.start + t.first;
    if (t.cloud < 0) {
        for (int i = tid; i < rows * a.dim; i += kThreads) store1(dq + ((row0 + i / a.dim) * a.heads + h) * a.dim + i % a.dim, 0.0f);
        for (int r = tid; r < rows; r += kThreads) stats.put((int64_t)h * a.n_query + row0 + r, 0.0f, near_weight(neg_inf()));
        if (part)
            for (int b = tid; b < a.buckets; b += kThreads) part[((int64_t)blockIdx.x * a.heads + h) * a.buckets + b] = 0.0f;
        return;
    }
    const int64_t k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
    const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2), nk = k1 > k0 ? k1 - k0 : 0;
    const int64_t off = nk - t.n, ro = (int64_t)a.heads * a.dim;
    if (tid < 2) again[tid] = 0;
    if (tid == 0) far = 0;
    __syncthreads();
    load_rows<T, D>((const T *)a.q + row0 * a.q_row + (int64_t)h * a.q_head, a.q_row, rows, a.dim, Q, again);
    load_rows<T, D>(dout + row0 * ro + (int64_t)h * a.dim, ro, rows, a.dim, G, again);
    for (int r = warp; r < rows; r += kThreads / 32) {
        float s = 0.0f;
        for (int d = lane; d < a.dim; d += 32) {
            const int64_t at = (row0 + r) * ro + (int64_t)h * a.dim + d;
            s = fmaf(load1(out + at) + (rest ? load1(rest + at) : 0.0f), load1(dout + at), s);
        }
        s = warp_sum(s);
        const float ls = lse[(int64_t)h * a.n_query + row0 + r];
        const RowWeight w = far_lse(ls) ? far_weight<T>(a, h, t.start, t.n, k0, nk, t.first + r) : near_weight(ls);
        if (lane == 0) {
            row_delta[r] = s;
            row_shift[r] = w.shift;
            row_inv[r] = w.inv;
            if (w.inv != 1.0f) far = 1;
            stats.put((int64_t)h * a.n_query + row0 + r, s, w);
        }
    }
    if (a.bias) {
        for (int i = tid; i < a.buckets; i += kThreads) table[i] = bias2_at(a, (int64_t)h * a.buckets + i);
        if (part)
            for (int i = 0; i < a.buckets; ++i) hist[i * kThreads + tid] = 0.0f;
    }
    __syncthreads();
    int vis_lo[4], vis_hi[4];
    float sh[4], de[4], o[4][D / 8], px[4], py[4], pz[4];
    bool seen_bad[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i < rows ? ty * 4 + i : rows - 1;
        const KeyRange vis = visible_keys(a, t.first + r + off, nk);
        vis_lo[i] = (int)vis.lo;
        vis_hi[i] = ty * 4 + i < rows ? (int)vis.hi : 0;
        sh[i] = row_shift[r];
        de[i] = row_delta[r];
        seen_bad[i] = false;
        px[i] = py[i] = pz[i] = 0.0f;
        if (a.bias) {
            px[i] = a.pos_q[3 * (row0 + r)];
            py[i] = a.pos_q[3 * (row0 + r) + 1];
            pz[i] = a.pos_q[3 * (row0 + r) + 2];
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[i][d] = 0.0f;
    }
    const KeyRange first = visible_keys(a, t.first + off, nk), last = visible_keys(a, t.first + rows - 1 + off, nk);
    int64_t sinks = a.num_sinks < first.lo ? a.num_sinks : first.lo;
    if (sinks > last.hi) sinks = last.hi;
    const float scale2 = a.scale * kLog2e;
    Load<T, D> lk, lv;
    float lp = 0.0f;
    auto read = [&](const Span &s) {
        const int n = (int)(s.end - s.j < kCols ? s.end - s.j : kCols);
        lk.read((const T *)a.k + (k0 + s.j) * a.k_row + (int64_t)hk * a.k_head, a.k_row, n, a.dim);
        lv.read((const T *)a.v + (k0 + s.j) * a.v_row + (int64_t)hk * a.v_head, a.v_row, n, a.dim);
        if (a.bias) lp = read_point(a.pos_k + 3 * (k0 + s.j), n);
    };
    Span s(sinks, first.lo, last.hi);
    if (kAhead<D> && s.more()) read(s);
    for (Span ahead = s; s.more(); s = ahead) {
        const int n = (int)(s.end - s.j < kCols ? s.end - s.j : kCols);
        ahead.next();
        __syncthreads();
        if (tid == 0) bad = 0;
        __syncthreads();
        if (!kAhead<D>) read(s);
        lk.write(K, kColLd, Kr, &bad);
        lv.write(V, kColLd, nullptr, &bad);
        write_point(lp, pos);
        if (kAhead<D> && ahead.more()) read(ahead);
        __syncthreads();
        float x[4][4], g[4][4];
        product(Q, K, D, ty, tx, x);
        product(G, V, D, ty, tx, g);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = tx * 4 + j;
                const int key = (int)s.j + c;
                const bool see = c < n && key < vis_hi[i] && (key >= vis_lo[i] || key < a.num_sinks);
                const bool odd = see && (bad >> c & 1);
                seen_bad[i] |= odd;
                float v = x[i][j] * scale2;
                int b = 0;
                if (a.bias && see) {
                    b = distance_bucket(a, px[i], py[i], pz[i], pos[c], pos[kCols + c], pos[2 * kCols + c]);
                    v += table[b];
                }
                float e = v + sh[i], f = g[i][j] - de[i];
                if (far) {
                    e = row_inv[ty * 4 + i] != 1.0f ? not_above_0(e) : e;
                    f *= row_inv[ty * 4 + i];
                }
                x[i][j] = see ? ex2(e) * f : 0.0f;
                // For the bucket sums alone (dQ of the row is computed again): a key that is not finite leaves lse and delta
                // finite only with weight 0.
                if (odd) x[i][j] = sh[i] == neg_inf() ? 0.0f : (sh[i] - sh[i]) + (de[i] - de[i]);
                if (part) hist[b * kThreads + tid] += x[i][j];
            }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4 *>(P + (tx * 4 + j) * kRowLd + ty * 4) = make_float4(x[0][j], x[1][j], x[2][j], x[3][j]);
        __syncthreads();
        gather<D>(P, Kr, ty, tx, o);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        if (r >= rows) continue;
        T *op = dq + ((row0 + r) * a.heads + h) * a.dim;
#pragma unroll
        for (int g = 0; g < D / 32; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (tx * 4 + 32 * g + j < a.dim) store1(op + tx * 4 + 32 * g + j, o[i][4 * g + j] * a.scale);
        if (seen_bad[i]) atomicOr(again + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int r = warp; r < rows; r += kThreads / 32)
        if (again[r >> 5] >> (r & 31) & 1)
            attention_dq_row<T>(a, h, t.start, t.n, k0, nk, t.first + r, P + warp * 2 * kAttnMaxDim,
                                P + (warp * 2 + 1) * kAttnMaxDim, stats, dout, dq);
    if (part)
        for (int b = warp; b < a.buckets; b += kThreads / 32) {
            float s = 0.0f;
            for (int k = lane; k < kThreads; k += 32) s += hist[b * kThreads + k];
            s = warp_sum(s);
            if (lane == 0) part[((int64_t)blockIdx.x * a.heads + h) * a.buckets + b] = s;
        }
}

template <int D>
constexpr size_t dkv_smem(int nb) {
    return (size_t)(2 * D * kRowLd + 2 * D * kColLd + 2 * kCols * (D + 4) + 2 * kCols * kRowLd + nb + 6 * kCols) * 4;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads)
    attn_simt_dkv_kernel(const __grid_constant__ gdl_attention a, const RowStats stats, const T *__restrict__ dout,
                         T *__restrict__ dk, T *__restrict__ dv, const SinkPlan sp, int64_t main_ctas) {
    extern __shared__ __align__(16) float sm[];
    float *K = sm, *V = K + D * kRowLd, *Q = V + D * kRowLd, *G = Q + D * kColLd, *Qr = G + D * kColLd,
          *Gr = Qr + kCols * (D + 4), *P = Gr + kCols * (D + 4), *S = P + kCols * kRowLd, *cols = S + kCols * kRowLd,
          *table = cols + 6 * kCols;  // cols [6][kCols]: shift, delta, x, y, z, inv of a tile's queries
    __shared__ uint32_t bad;
    __shared__ uint32_t again[2];
    const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7, warp = tid >> 5;
    const SinkUnit u = sink_unit(a, sp, main_ctas, kRows);
    if (u.skip) return;
    const int group = a.heads / a.kv_heads, rows = u.rows, hk = u.hk;
    const int64_t ro = (int64_t)a.heads * a.dim, kr0 = u.k0 + u.j0;
    if (u.hi <= u.lo) {
        for (int i = tid; i < (rows - u.first_out) * a.dim; i += kThreads) {
            const int64_t at = ((kr0 + u.first_out + i / a.dim) * a.kv_heads + hk) * a.dim + i % a.dim;
            store1(dk + at, 0.0f);
            store1(dv + at, 0.0f);
        }
        for (int i = tid; i < u.first_out * 2 * a.dim; i += kThreads) u.partial[i] = 0.0f;
        return;
    }
    if (tid < 2) again[tid] = 0;
    __syncthreads();
    load_rows<T, D>((const T *)a.k + kr0 * a.k_row + (int64_t)hk * a.k_head, a.k_row, rows, a.dim, K, again);
    load_rows<T, D>((const T *)a.v + kr0 * a.v_row + (int64_t)hk * a.v_head, a.v_row, rows, a.dim, V, again);
    int vis_lo[4], vis_hi[4];
    float ok[4][D / 8], ov[4][D / 8], px[4], py[4], pz[4];
    bool seen_bad[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i < rows ? ty * 4 + i : rows - 1;
        const QueryRange vis = visible_queries(a, u.j0 + r, u.nq, u.nk);
        vis_lo[i] = (int)vis.lo;
        vis_hi[i] = ty * 4 + i >= rows ? 0 : (int)(vis.hi < u.hi ? vis.hi : u.hi);
        seen_bad[i] = false;
        px[i] = py[i] = pz[i] = 0.0f;
        if (a.bias) {
            px[i] = a.pos_k[3 * (kr0 + r)];
            py[i] = a.pos_k[3 * (kr0 + r) + 1];
            pz[i] = a.pos_k[3 * (kr0 + r) + 2];
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) ok[i][d] = ov[i][d] = 0.0f;
    }
    const float scale2 = a.scale * kLog2e;
    Load<T, D> lq, lg;
    float lc[6] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    auto read = [&](int h, int64_t c0) {
        const int n = (int)(u.hi - c0 < kCols ? u.hi - c0 : kCols);
        lq.read((const T *)a.q + (u.q0 + c0) * a.q_row + (int64_t)h * a.q_head, a.q_row, n, a.dim);
        lg.read(dout + (u.q0 + c0) * ro + (int64_t)h * a.dim, ro, n, a.dim);
        if (tid < kCols) {
            const int64_t q = u.q0 + c0 + (tid < n ? tid : 0), at = (int64_t)h * a.n_query + q;
            lc[0] = stats.shift(at);
            lc[1] = stats.delta(at);
            lc[5] = stats.inv(at);
            if (a.bias)
#pragma unroll
                for (int x = 0; x < 3; ++x) lc[2 + x] = a.pos_q[3 * q + x];
        }
    };
    if (kAhead<D>) read(hk * group, u.lo);
    for (int h = hk * group; h < (hk + 1) * group; ++h)
        for (int64_t c0 = u.lo; c0 < u.hi; c0 += kCols) {
            const int n = (int)(u.hi - c0 < kCols ? u.hi - c0 : kCols);
            __syncthreads();
            if (tid == 0) bad = 0;
            if (a.bias && c0 == u.lo)
                for (int i = tid; i < a.buckets; i += kThreads) table[i] = bias2_at(a, (int64_t)h * a.buckets + i);
            __syncthreads();
            if (!kAhead<D>) read(h, c0);
            lq.write(Q, kColLd, Qr, &bad);
            lg.write(G, kColLd, Gr, &bad);
            if (tid < kCols)
#pragma unroll
                for (int x = 0; x < 6; ++x) cols[x * kCols + tid] = lc[x];
            if (kAhead<D>) {
                const bool more = c0 + kCols < u.hi;
                if (more || h + 1 < (hk + 1) * group) read(more ? h : h + 1, more ? c0 + kCols : u.lo);
            }
            __syncthreads();
            float x[4][4], g[4][4];
            product(K, Q, D, ty, tx, x);
            product(V, G, D, ty, tx, g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = tx * 4 + j;
                    const int q = (int)c0 + c;
                    bool see = c < n && q >= vis_lo[i] && q < vis_hi[i];
                    if (see && (bad >> c & 1)) {
                        seen_bad[i] = true;
                        see = false;
                    }
                    float v = x[i][j] * scale2;
                    if (a.bias && see)
                        v += table[distance_bucket(a, px[i], py[i], pz[i], cols[2 * kCols + c], cols[3 * kCols + c], cols[4 * kCols + c])];
                    const float p = see ? weight(v, cols[c], cols[5 * kCols + c]) : 0.0f;
                    x[i][j] = p;
                    g[i][j] = see ? p * (g[i][j] - cols[kCols + c]) : 0.0f;
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                *reinterpret_cast<float4 *>(P + (tx * 4 + j) * kRowLd + ty * 4) = make_float4(x[0][j], x[1][j], x[2][j], x[3][j]);
                *reinterpret_cast<float4 *>(S + (tx * 4 + j) * kRowLd + ty * 4) = make_float4(g[0][j], g[1][j], g[2][j], g[3][j]);
            }
            __syncthreads();
            gather<D>(P, Gr, ty, tx, ov);
            gather<D>(S, Qr, ty, tx, ok);
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
        if (r >= rows) continue;
        const int64_t at = ((kr0 + r) * a.kv_heads + hk) * a.dim;
#pragma unroll
        for (int g = 0; g < D / 32; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = tx * 4 + 32 * g + j;
                if (d >= a.dim) continue;
                const float x = ok[i][4 * g + j] * a.scale, y = ov[i][4 * g + j];
                if (r < u.first_out) {
                    u.partial[(2 * r) * a.dim + d] = x;
                    u.partial[(2 * r + 1) * a.dim + d] = y;
                } else {
                    store1(dk + at + d, x);
                    store1(dv + at + d, y);
                }
            }
        if (seen_bad[i]) atomicOr(again + (r >> 5), 1u << (r & 31));
    }
    __syncthreads();
    for (int r = warp; r < rows; r += kThreads / 32)
        if (again[r >> 5] >> (r & 31) & 1)
            attention_dkv_row<T>(a, hk, u.q0, u.nq, u.k0, u.nk, u.j0 + r, u.lo, u.hi, P + warp * 2 * kAttnMaxDim,
                                 P + (warp * 2 + 1) * kAttnMaxDim, stats, dout,
                                 r < u.first_out ? u.partial + (int64_t)r * 2 * a.dim : nullptr, dk, dv);
}

template <typename F>
int by_dim(int dim, F f) {
    if (dim <= 32) return f(std::integral_constant<int, 32>{});
    if (dim <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

template <typename T>
int forward(const gdl_attention &a, T *out, float *lse, T *rest, cudaStream_t st) {
    return by_dim(a.dim, [&](auto d) -> int {
        constexpr int D = decltype(d)::value;
        const size_t smem = fwd_smem<D>(a.bias ? a.buckets : 0);
        GDL_CUDA_TRY(cudaFuncSetAttribute(attn_simt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        attn_simt_kernel<T, D><<<dim3((unsigned)ragged_slots(a.n_query, a.num_clouds, kRows), a.heads), kThreads, smem, st>>>(a, out, lse, rest);
        GDL_CUDA_TRY(cudaGetLastError());
        return GDL_OK;
    });
}

template <typename T>
int backward(const gdl_attention &a, const T *out, const float *lse, const T *rest, const T *dout, T *dq, T *dk, T *dv, const RowStats stats,
             float *part, float *sink_ws, int chunk, cudaStream_t st) {
    const SinkPlan sp = sink_plan(a, sink_ws, kRows, chunk);
    return by_dim(a.dim, [&](auto d) -> int {
        constexpr int D = decltype(d)::value;
        const int nb = a.bias ? a.buckets : 0;
        if (a.n_query > 0) {
            const size_t smem = dq_smem<D>(nb, part != nullptr);
            GDL_CUDA_TRY(cudaFuncSetAttribute(attn_simt_dq_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            attn_simt_dq_kernel<T, D><<<dim3((unsigned)ragged_slots(a.n_query, a.num_clouds, kRows), a.heads), kThreads, smem, st>>>(
                a, out, lse, rest, dout, dq, stats, part);
            GDL_CUDA_TRY(cudaGetLastError());
        }
        if (a.n_key > 0) {
            const size_t smem = dkv_smem<D>(nb);
            const int64_t main = ragged_slots(a.n_key, a.num_clouds, kRows) * a.kv_heads, all = main + sp.tiles * sp.slots * a.kv_heads;
            GDL_RETURN_IF(all > ((int64_t)1 << 31) - 1, GDL_ERR_OVERFLOW);
            GDL_CUDA_TRY(cudaFuncSetAttribute(attn_simt_dkv_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            attn_simt_dkv_kernel<T, D><<<(unsigned)all, kThreads, smem, st>>>(a, stats, dout, dk, dv, sp, main);
            GDL_CUDA_TRY(cudaGetLastError());
        }
        return join_sinks<T>(a, sp, kRows, dk, dv, st);
    });
}

}  // namespace

int attention_simt_rows() { return kRows; }

int attention_forward_simt(const gdl_attention &a, void *out, float *lse, void *rest, cudaStream_t st) {
    return a.dtype == GDL_DTYPE_F32 ? forward<float>(a, (float *)out, lse, nullptr, st)
                                    : forward<uint16_t>(a, (uint16_t *)out, lse, (uint16_t *)rest, st);
}

int attention_backward_simt(const gdl_attention &a, const void *out, const float *lse, const void *rest, const void *dout,
                            void *dq, void *dk, void *dv, const RowStats stats, float *part, float *sink_ws, int chunk,
                            cudaStream_t st) {
    if (a.dtype == GDL_DTYPE_F32)
        return backward<float>(a, (const float *)out, lse, (const float *)nullptr, (const float *)dout, (float *)dq, (float *)dk, (float *)dv, stats, part, sink_ws, chunk, st);
    return backward<uint16_t>(a, (const uint16_t *)out, lse, (const uint16_t *)rest, (const uint16_t *)dout, (uint16_t *)dq, (uint16_t *)dk, (uint16_t *)dv,
                              stats, part, sink_ws, chunk, st);
}

}  // namespace gdl
