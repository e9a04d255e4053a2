// attention.cuh -- what the windowed-attention kernels share: visible ranges, distance buckets, and the
// routines by which one warp computes one row (a query's output or gradient, a key's gradients) from
// nothing but the rows it sees.
#pragma once

#include "ragged.cuh"

namespace gdl {

constexpr int kAttnMaxDim = 128;
constexpr int kAttnMaxBuckets = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFloatMax = 3.4028234664e38f;

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

__device__ __forceinline__ float load1(const float *p) { return __ldg(p); }
__device__ __forceinline__ float load1(const uint16_t *p) { return bf16_bits_to_f32(__ldg(p)); }
__device__ __forceinline__ void store1(float *p, float v) { *p = v; }
__device__ __forceinline__ void store1(uint16_t *p, float v) { *p = f32_to_bf16_bits(v); }

// v to *p, and to *rest, if given, what that left over
template <typename T>
__device__ __forceinline__ void store_rest(T *p, T *rest, float v) {
    store1(p, v);
    if (sizeof(T) == 2 && rest) store1(rest, v - bf16_bits_to_f32(f32_to_bf16_bits(v)));
}

// keys that the query at place i of a cloud of nk keys sees: [0, sinks) and [lo, hi)
struct KeyRange {
    int64_t sinks, lo, hi;
};
__device__ __forceinline__ KeyRange visible_keys(const gdl_attention &a, int64_t i, int64_t nk) {
    KeyRange r;
    r.hi = a.right < 0 || i + a.right + 1 > nk ? nk : i + a.right + 1;
    if (r.hi < 0) r.hi = 0;
    r.lo = a.left < 0 || i - a.left < 0 ? 0 : i - a.left;
    r.sinks = a.num_sinks < r.lo ? a.num_sinks : r.lo;
    if (r.sinks > r.hi) r.sinks = r.hi;
    return r;
}

// queries (rows of the cloud's nq) that see key j: [lo, hi)
struct QueryRange {
    int64_t lo, hi;
};
__device__ __forceinline__ QueryRange visible_queries(const gdl_attention &a, int64_t j, int64_t nq, int64_t nk) {
    const int64_t off = nk - nq;
    QueryRange r;
    r.lo = a.right < 0 || j - a.right - off < 0 ? 0 : j - a.right - off;
    r.hi = a.left < 0 || j < a.num_sinks || j + a.left + 1 - off > nq ? nq : j + a.left + 1 - off;
    return r;
}

__device__ __forceinline__ int distance_bucket(const gdl_attention &a, float px, float py, float pz, float rx, float ry,
                                               float rz) {
    const float t = fmaf(dist2(px, py, pz, rx, ry, rz), a.inv_radius2, 1.0f);
    const unsigned u = (__float_as_uint(t) >> (23 - a.steps_log2)) - (127u << a.steps_log2);
    const unsigned top = (unsigned)(a.buckets - 1);
    return (int)(u < top ? u : top);
}

__device__ __forceinline__ float bias_at(const gdl_attention &a, int64_t i) {
    return a.bias_dtype == GDL_DTYPE_F32 ? __ldg((const float *)a.bias + i)
                                         : bf16_bits_to_f32(__ldg((const uint16_t *)a.bias + i));
}

// The same in powers of two. The type's lowest value (a mask) stays finite: a row of nothing else weighs all alike.
__device__ __forceinline__ float bias2_at(const gdl_attention &a, int64_t i) {
    const float b = bias_at(a, i), t = b * kLog2e;
    return fabsf(b) <= kFloatMax ? fminf(fmaxf(t, -kFloatMax), kFloatMax) : t;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <typename T>
__device__ __forceinline__ float row_dot(const float *s, const T *p, int dim) {
    float acc = 0.0f;
    for (int d = 0; d < dim; ++d) acc = fmaf(s[d], load1(p + d), acc);
    return acc;
}

// a row of `dim` values into a warp's shared-memory strip
template <typename T>
__device__ __forceinline__ void stage_row(float *s, const T *p, int dim) {
    for (int d = threadIdx.x & 31; d < dim; d += 32) s[d] = load1(p + d);
}

// The logit (in powers of two) of global query row qi and global key row kj, head h, from their product.
__device__ __forceinline__ float logit2_of(const gdl_attention &a, int h, float dot, int64_t qi, int64_t kj) {
    const float s = dot * (a.scale * kLog2e);
    if (!a.bias) return s;
    const float *p = a.pos_q + 3 * qi, *r = a.pos_k + 3 * kj;
    return s + bias2_at(a, (int64_t)h * a.buckets + distance_bucket(a, p[0], p[1], p[2], r[0], r[1], r[2]));
}
template <typename T>
__device__ __forceinline__ const T *key_row(const gdl_attention &a, int h, int64_t kj) {
    return (const T *)a.k + kj * a.k_row + (int64_t)(h / (a.heads / a.kv_heads)) * a.k_head;
}
template <typename T>
__device__ __forceinline__ float logit2(const gdl_attention &a, int h, const float *sq, int64_t qi, int64_t kj) {
    return logit2_of(a, h, row_dot(sq, key_row<T>(a, h, kj), a.dim), qi, kj);
}

// A row's weights in the gradients, from its logits x in powers of two: P = exp2(x + shift) inv. From the forward's
// lse, shift is -lse and inv 1 (-inf where every logit is -inf: P = 0). Beside a large lse (a finite mask over all that a
// row sees) 32 bits hold too little of the sum's logarithm: shift is then minus the largest logit and inv one over the sum,
// both found anew, and x + shift is kept from rising above 0 by a rounding.
struct RowWeight {
    float shift, inv;
};
constexpr float kFarLse = 2048.0f;  // (from here on lse alone would put P off by more than 3e-4)
__device__ __forceinline__ bool far_lse(float ls) { return fabsf(ls) > kFarLse && fabsf(ls) <= kFloatMax; }
__device__ __forceinline__ RowWeight near_weight(float ls) {
    return {ls == neg_inf() ? ls : ls * -kLog2e, 1.0f};
}
__device__ __forceinline__ float not_above_0(float x) { return x > 0.0f ? 0.0f : x; }  // (NaN stays)

// One warp: the weights of a row with a large lse.
template <typename T>
__device__ __noinline__ RowWeight far_weight(const gdl_attention &a, int h, int64_t q0, int64_t nq, int64_t k0,
                                             int64_t nk, int64_t row) {
    const int lane = threadIdx.x & 31;
    const int64_t qi = q0 + row;
    const T *qp = (const T *)a.q + qi * a.q_row + (int64_t)h * a.q_head;
    const KeyRange r = visible_keys(a, row + nk - nq, nk);
    float m = neg_inf(), l = 0.0f;
    for (int part = 0; part < 2; ++part)
        for (int64_t j = (part ? r.lo : 0) + lane; j < (part ? r.hi : r.sinks); j += 32) {
            const T *kp = key_row<T>(a, h, k0 + j);
            float dot = 0.0f;
            for (int d = 0; d < a.dim; ++d) dot = fmaf(load1(qp + d), load1(kp + d), dot);
            const float x = logit2_of(a, h, dot, qi, k0 + j), mn = fmaxf(m, x), base = mn == neg_inf() ? 0.0f : mn;
            l = fmaf(l, ex2(m - base), ex2(x - base));
            m = mn;
        }
    const float top = warp_max(m);
    const float sum = warp_sum(m == neg_inf() ? 0.0f : l * ex2(m - top));
    return {-top, 1.0f / sum};
}

// One warp: output row and lse (natural) of query row `row` of a cloud (starts q0, k0; sizes nq, nk).
// sq: kAttnMaxDim floats of the warp's own. rest (nullable): what rounding the output left over.
template <typename T>
__device__ __noinline__ void attention_row(const gdl_attention &a, int h, int64_t q0, int64_t nq, int64_t k0,
                                           int64_t nk, int64_t row, float *sq, T *out, float *lse, T *rest) {
    const int lane = threadIdx.x & 31;
    const int64_t qi = q0 + row;
    const int hk = h / (a.heads / a.kv_heads);
    __syncwarp();
    stage_row(sq, (const T *)a.q + qi * a.q_row + (int64_t)h * a.q_head, a.dim);
    __syncwarp();
    const KeyRange r = visible_keys(a, row + nk - nq, nk);
    float m = neg_inf(), l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int part = 0; part < 2; ++part) {
        const int64_t from = part ? r.lo : 0, to = part ? r.hi : r.sinks;
        // (one NaN makes the sum and every output NaN for good: after a step that diverged all rows come here)
        for (int64_t j0 = from; j0 < to && l == l; j0 += 32) {
            const int64_t j = j0 + lane;
            const float s = j < to ? logit2<T>(a, h, sq, qi, k0 + j) : neg_inf();
            const float mn = fmaxf(m, warp_max(s));
            const float base = mn == neg_inf() ? 0.0f : mn;
            const float c = ex2(m - base);
            const float p = j < to ? ex2(s - base) : 0.0f;
            l = fmaf(l, c, warp_sum(p));
            m = mn;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] *= c;
            const int cnt = to - j0 < 32 ? (int)(to - j0) : 32;
            for (int t = 0; t < cnt; ++t) {
                const float pt = __shfl_sync(0xffffffffu, p, t);
                const T *vp = (const T *)a.v + (k0 + j0 + t) * a.v_row + (int64_t)hk * a.v_head;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lane + 32 * e < a.dim) acc[e] = fmaf(pt, load1(vp + lane + 32 * e), acc[e]);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *op = out + (qi * a.heads + h) * a.dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.dim) store_rest(op + lane + 32 * e, rest ? rest + (op - out) + lane + 32 * e : nullptr, acc[e] * inv);
    if (lse && lane == 0) lse[(int64_t)h * a.n_query + qi] = l == 0.0f ? neg_inf() : (m + log2f(l)) * kLn2;
}

// What the dQ kernels find of each row, [3][heads][n_query]: delta, and the weights' shift and inv.
struct RowStats {
    float *at;
    int64_t each;  // heads * n_query
    __device__ __forceinline__ void put(int64_t i, float delta, RowWeight w) const {
        at[i] = delta;
        at[each + i] = w.shift;
        at[2 * each + i] = w.inv;
    }
    __device__ __forceinline__ float delta(int64_t i) const { return at[i]; }
    __device__ __forceinline__ float shift(int64_t i) const { return at[each + i]; }
    __device__ __forceinline__ float inv(int64_t i) const { return at[2 * each + i]; }
};
__device__ __forceinline__ float weight(float x, float shift, float inv) {
    const float e = x + shift;
    return ex2(inv != 1.0f ? not_above_0(e) : e) * inv;
}

// One warp: dq of a query row. sq, sd: strips of the warp's own.
template <typename T>
__device__ __noinline__ void attention_dq_row(const gdl_attention &a, int h, int64_t q0, int64_t nq, int64_t k0,
                                              int64_t nk, int64_t row, float *sq, float *sd,
                                              const RowStats stats, const T *dout, T *dq) {
    const int lane = threadIdx.x & 31;
    const int64_t qi = q0 + row;
    const int hk = h / (a.heads / a.kv_heads);
    const int64_t ro = (qi * a.heads + h) * a.dim;
    __syncwarp();
    stage_row(sq, (const T *)a.q + qi * a.q_row + (int64_t)h * a.q_head, a.dim);
    stage_row(sd, dout + ro, a.dim);
    __syncwarp();
    const int64_t at = (int64_t)h * a.n_query + qi;
    const float de = stats.delta(at), shift = stats.shift(at), inv = stats.inv(at);
    const KeyRange r = visible_keys(a, row + nk - nq, nk);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int part = 0; part < 2; ++part) {
        const int64_t from = part ? r.lo : 0, to = part ? r.hi : r.sinks;
        for (int64_t j0 = from; j0 < to; j0 += 32) {
            const int64_t j = j0 + lane;
            float ds = 0.0f;
            if (j < to) {
                const T *vp = (const T *)a.v + (k0 + j) * a.v_row + (int64_t)hk * a.v_head;
                ds = weight(logit2<T>(a, h, sq, qi, k0 + j), shift, inv) * (row_dot(sd, vp, a.dim) - de);
            }
            const int cnt = to - j0 < 32 ? (int)(to - j0) : 32;
            for (int t = 0; t < cnt; ++t) {
                const float dt = __shfl_sync(0xffffffffu, ds, t);
                const T *kp = (const T *)a.k + (k0 + j0 + t) * a.k_row + (int64_t)hk * a.k_head;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lane + 32 * e < a.dim) acc[e] = fmaf(dt, load1(kp + lane + 32 * e), acc[e]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.dim) store1(dq + ro + lane + 32 * e, acc[e] * a.scale);
}

// One warp: dk and dv of a key row, for one head of keys and values, over the cloud's queries lo .. hi - 1; as
// sums in f32 to `partial` (dk, then dv), if given.
template <typename T>
__device__ __noinline__ void attention_dkv_row(const gdl_attention &a, int hk, int64_t q0, int64_t nq, int64_t k0,
                                               int64_t nk, int64_t row, int64_t lo, int64_t hi, float *sk, float *sv,
                                               const RowStats stats, const T *dout, float *partial, T *dk, T *dv) {
    const int lane = threadIdx.x & 31;
    const int64_t kj = k0 + row;
    const int group = a.heads / a.kv_heads;
    __syncwarp();
    stage_row(sk, (const T *)a.k + kj * a.k_row + (int64_t)hk * a.k_head, a.dim);
    stage_row(sv, (const T *)a.v + kj * a.v_row + (int64_t)hk * a.v_head, a.dim);
    __syncwarp();
    QueryRange r = visible_queries(a, row, nq, nk);
    if (r.lo < lo) r.lo = lo;
    if (r.hi > hi) r.hi = hi;
    float ak[4] = {0.0f, 0.0f, 0.0f, 0.0f}, av[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
        for (int64_t i0 = r.lo; i0 < r.hi; i0 += 32) {
            const int64_t qi = q0 + i0 + lane;
            float p = 0.0f, ds = 0.0f;
            if (i0 + lane < r.hi) {
                const int64_t at = (int64_t)h * a.n_query + qi;
                const float dot = row_dot(sk, (const T *)a.q + qi * a.q_row + (int64_t)h * a.q_head, a.dim);
                p = weight(logit2_of(a, h, dot, qi, kj), stats.shift(at), stats.inv(at));
                ds = p * (row_dot(sv, dout + (qi * a.heads + h) * a.dim, a.dim) - stats.delta(at));
            }
            const int cnt = r.hi - i0 < 32 ? (int)(r.hi - i0) : 32;
            for (int t = 0; t < cnt; ++t) {
                const float pt = __shfl_sync(0xffffffffu, p, t), dt = __shfl_sync(0xffffffffu, ds, t);
                const int64_t q = q0 + i0 + t;
                const T *qp = (const T *)a.q + q * a.q_row + (int64_t)h * a.q_head;
                const T *dp = dout + (q * a.heads + h) * a.dim;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lane + 32 * e < a.dim) {
                        ak[e] = fmaf(dt, load1(qp + lane + 32 * e), ak[e]);
                        av[e] = fmaf(pt, load1(dp + lane + 32 * e), av[e]);
                    }
            }
        }
    }
    const int64_t ro = (kj * a.kv_heads + hk) * a.dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < a.dim) {
            const int d = lane + 32 * e;
            if (partial) {
                partial[d] = ak[e] * a.scale;
                partial[a.dim + d] = av[e];
            } else {
                store1(dk + ro + d, ak[e] * a.scale);
                store1(dv + ro + d, av[e]);
            }
        }
}

}  // namespace gdl
