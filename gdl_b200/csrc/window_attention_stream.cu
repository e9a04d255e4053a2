// window_attention_stream.cu -- windowed attention of few query rows (a stream's new rows against its cached
// keys), bf16 and f32 (sm_100a).
//
// One query row has nothing to tile: each key and value is read once for it and the heads that share them, so
// the call is a read of the window. A cluster of CTAs takes one row and up to 4 heads of one key head; its
// CTAs' warps share out the visible keys. In a warp, LPR lanes hold one row of K (16 bytes each), 32 / LPR
// keys at a time, 4 such steps in flight; every lane keeps its part of the outputs with a running maximum and
// sum per group of lanes. The groups, warps and CTAs (through distributed shared memory) are joined in a fixed
// order. Only visible keys are read. 8 rows over up to 1040 keys each, 8 heads of 64 over 2, 32 buckets, bf16:
// 10.5 us, where the bytes take 0.6: latency.
#include <cooperative_groups.h>

#include "attention_mma.cuh"

namespace gdl {
namespace {

namespace cg = cooperative_groups;

constexpr int kStreamWarps = 8;
constexpr int kSteps = 4;      // steps of keys in flight
constexpr int kMaxSplits = 4;  // CTAs of a cluster (one row over 1040 keys: 1, 2, 4, 8 take 19.0, 13.6, 10.8, 15.1 us)

template <typename T>
struct Lane16;  // 16 bytes of a row
template <>
struct Lane16<uint16_t> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void widen(const uint4 &v, float *f) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
template <>
struct Lane16<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void widen(const uint4 &v, float *f) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
};

// joins (m, l, o[]) of another part into this one
template <int N>
__device__ __forceinline__ void join(float &m, float &l, float *o, float m2, float l2, const float *o2) {
    const float mn = fmaxf(m, m2), base = mn == neg_inf() ? 0.0f : mn;
    const float f = ex2(m - base), f2 = ex2(m2 - base);
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * f + o2[i] * f2;
    m = mn;
}

template <typename T, int LPR, int HEADS>
__global__ void __launch_bounds__(32 * kStreamWarps)
    attn_stream_kernel(const __grid_constant__ gdl_attention a, int splits, T *__restrict__ out, float *__restrict__ lse,
                       T *__restrict__ rest) {
    constexpr int E = Lane16<T>::n, KEYS = 32 / LPR, ROW = LPR * E;
    __shared__ float part[kStreamWarps][HEADS][2 + ROW];  // m, l, o of each warp
    __shared__ float mine[HEADS][2 + ROW];                // of the CTA
    __shared__ float table[HEADS][kAttnMaxBuckets];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane % LPR, key = lane / LPR;
    const int group = a.heads / a.kv_heads, chunks = (group + HEADS - 1) / HEADS;
    const int hk = blockIdx.y / chunks, h0 = hk * group + blockIdx.y % chunks * HEADS;
    const int heads = (hk + 1) * group - h0 < HEADS ? (hk + 1) * group - h0 : HEADS;
    const int rank = (int)(blockIdx.x % splits);
    const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, 1, blockIdx.x / splits);
    if (t.cloud == -2) return;  // the whole cluster
    const int64_t qi = t.start + t.first;
    KeyRange vis = {0, 0, 0};
    int64_t k0 = 0;
    if (t.cloud >= 0) {
        k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
        const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2), nk = k1 > k0 ? k1 - k0 : 0;
        vis = visible_keys(a, t.first + nk - t.n, nk);
    }
    const bool on = sub * E < a.dim;  // dim is a multiple of E
    float q[HEADS][E], o[HEADS][E], m[HEADS], l[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
        m[h] = neg_inf();
        l[h] = 0.0f;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (on && h < heads)
            v = __ldg(reinterpret_cast<const uint4 *>((const T *)a.q + qi * a.q_row + (int64_t)(h0 + h) * a.q_head + sub * E));
        Lane16<T>::widen(v, q[h]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[h][e] *= a.scale * kLog2e;
            o[h][e] = 0.0f;
        }
    }
    float px = 0.0f, py = 0.0f, pz = 0.0f;
    if (a.bias) {
        for (int i = tid; i < heads * a.buckets; i += 32 * kStreamWarps)
            table[i / a.buckets][i % a.buckets] = bias2_at(a, (int64_t)h0 * a.buckets + i);
        px = a.pos_q[3 * qi];
        py = a.pos_q[3 * qi + 1];
        pz = a.pos_q[3 * qi + 2];
        __syncthreads();
    }
    // the visible keys in one count: the sinks, then the window; this CTA's warps take every splits * 8th step
    const int64_t total = vis.sinks + (vis.hi > vis.lo ? vis.hi - vis.lo : 0);
    const T *kb = (const T *)a.k + (int64_t)hk * a.k_head + sub * E, *vb = (const T *)a.v + (int64_t)hk * a.v_head + sub * E;
    for (int64_t c0 = ((int64_t)rank * kStreamWarps + warp) * (KEYS * kSteps); c0 < total;
         c0 += (int64_t)splits * kStreamWarps * (KEYS * kSteps)) {
        uint4 kr[kSteps], vr[kSteps];
        float rx[kSteps], ry[kSteps], rz[kSteps];
        bool see[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int64_t c = c0 + s * KEYS + key;
            see[s] = c < total;
            const int64_t kj = k0 + (c < vis.sinks ? c : vis.lo + c - vis.sinks);
            kr[s] = vr[s] = make_uint4(0, 0, 0, 0);
            if (see[s] && on) {
                kr[s] = __ldg(reinterpret_cast<const uint4 *>(kb + kj * a.k_row));
                vr[s] = __ldg(reinterpret_cast<const uint4 *>(vb + kj * a.v_row));
            }
            if (a.bias && see[s]) {
                const float *r = a.pos_k + 3 * kj;
                rx[s] = __ldg(r);
                ry[s] = __ldg(r + 1);
                rz[s] = __ldg(r + 2);
            }
        }
        float x[kSteps][HEADS];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float k[E];
            Lane16<T>::widen(kr[s], k);
            int bucket = 0;
            if (a.bias && see[s]) bucket = distance_bucket(a, px, py, pz, rx[s], ry[s], rz[s]);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) d = fmaf(q[h][e], k[e], d);
#pragma unroll
                for (int w = LPR / 2; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
                if (a.bias && h < heads) d += table[h][bucket];
                x[s][h] = see[s] ? d : neg_inf();
            }
        }
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float mn = m[h];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) mn = fmaxf(mn, x[s][h]);
            const float base = mn == neg_inf() ? 0.0f : mn, f = ex2(m[h] - base);
            m[h] = mn;
            l[h] *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[h][e] *= f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const float p = ex2(x[s][h] - base);
                x[s][h] = see[s] ? p : 0.0f;
                l[h] += x[s][h];
            }
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float v[E];
            Lane16<T>::widen(vr[s], v);
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
#pragma unroll
                for (int e = 0; e < E; ++e) o[h][e] = fmaf(x[s][h], v[e], o[h][e]);
        }
    }
    // the warp's groups of lanes, the CTA's warps, the cluster's CTAs
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
#pragma unroll
        for (int w = LPR; w < 32; w <<= 1) {
            float o2[E];
            const float m2 = __shfl_xor_sync(0xffffffffu, m[h], w), l2 = __shfl_xor_sync(0xffffffffu, l[h], w);
#pragma unroll
            for (int e = 0; e < E; ++e) o2[e] = __shfl_xor_sync(0xffffffffu, o[h][e], w);
            join<E>(m[h], l[h], o[h], m2, l2, o2);
        }
        if (key == 0) {
            if (sub == 0) {
                part[warp][h][0] = m[h];
                part[warp][h][1] = l[h];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) part[warp][h][2 + sub * E + e] = o[h][e];
        }
    }
    __syncthreads();
    for (int i = tid; i < HEADS * ROW; i += 32 * kStreamWarps) {
        const int h = i / ROW, d = i % ROW;
        float mm = neg_inf(), ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < kStreamWarps; ++w) join<1>(mm, ll, &oo, part[w][h][0], part[w][h][1], &part[w][h][2 + d]);
        mine[h][2 + d] = oo;
        if (d == 0) {
            mine[h][0] = mm;
            mine[h][1] = ll;
        }
    }
    if (splits > 1)
        cluster.sync();
    else
        __syncthreads();
    if (rank == 0) {
        for (int i = tid; i < heads * a.dim; i += 32 * kStreamWarps) {
            const int h = i / a.dim, d = i % a.dim;
            float mm = mine[h][0], ll = mine[h][1], oo = mine[h][2 + d];
            float rm[kMaxSplits], rl[kMaxSplits], rv[kMaxSplits];  // all remote reads at once: each takes a trip to another SM
#pragma unroll
            for (int r = 1; r < kMaxSplits; ++r)
                if (r < splits) {
                    const float *p = cluster.map_shared_rank(&mine[h][0], r);
                    rm[r] = p[0];
                    rl[r] = p[1];
                    rv[r] = p[2 + d];
                }
#pragma unroll
            for (int r = 1; r < kMaxSplits; ++r)
                if (r < splits) join<1>(mm, ll, &oo, rm[r], rl[r], &rv[r]);
            const int64_t at = (qi * a.heads + h0 + h) * a.dim + d;
            store_rest(out + at, rest ? rest + at : nullptr, ll == 0.0f ? 0.0f : oo / ll);
            if (lse && d == 0)
                lse[(int64_t)(h0 + h) * a.n_query + qi] = ll == 0.0f ? neg_inf() : (mm + log2f(ll)) * kLn2;
        }
    }
    if (splits > 1) cluster.sync();  // the others' shared memory stays until it has been read
}

template <typename T, int LPR, int HEADS>
int launch(const gdl_attention &a, int splits, T *out, float *lse, T *rest, cudaStream_t st) {
    const int group = a.heads / a.kv_heads, chunks = (group + HEADS - 1) / HEADS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ragged_slots(a.n_query, a.num_clouds, 1) * splits), (unsigned)(a.kv_heads * chunks));
    cfg.blockDim = dim3(32 * kStreamWarps);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    GDL_CUDA_TRY(cudaLaunchKernelEx(&cfg, attn_stream_kernel<T, LPR, HEADS>, a, splits, out, lse, rest));
    return GDL_OK;
}

template <typename T, int LPR>
int by_heads(const gdl_attention &a, int splits, T *out, float *lse, T *rest, cudaStream_t st) {
    const int group = a.heads / a.kv_heads;
    if (group == 1) return launch<T, LPR, 1>(a, splits, out, lse, rest, st);
    if (group == 2) return launch<T, LPR, 2>(a, splits, out, lse, rest, st);
    return launch<T, LPR, 4>(a, splits, out, lse, rest, st);
}

template <typename T>
int stream_forward(const gdl_attention &a, T *out, float *lse, T *rest, cudaStream_t st) {
    // CTAs to a row: enough for two to an SM over the call, while each still has a step of keys for its warps
    const int group = a.heads / a.kv_heads, chunks = group <= 2 ? 1 : (group + 3) / 4;
    const int64_t side = a.left < 0 || a.right < 0 ? a.n_key : a.left + a.right + 1 + a.num_sinks;
    const int64_t span = side < a.n_key ? side : a.n_key, ctas = a.n_query * a.kv_heads * chunks;
    int splits = 1;
    while (splits < kMaxSplits && ctas * splits * 2 <= 2 * kSmCount && span / (splits * 2) >= 64) splits *= 2;
    const int per = 16 / (int)sizeof(T);
    if (a.dim <= 2 * per) return by_heads<T, 2>(a, splits, out, lse, rest, st);
    if (a.dim <= 4 * per) return by_heads<T, 4>(a, splits, out, lse, rest, st);
    if (a.dim <= 8 * per) return by_heads<T, 8>(a, splits, out, lse, rest, st);
    if (a.dim <= 16 * per) return by_heads<T, 16>(a, splits, out, lse, rest, st);
    return by_heads<T, 32>(a, splits, out, lse, rest, st);
}

}  // namespace

// Few rows: up to 16 to a cloud on average. (Clouds of 4096 keys, window 1024, 8 heads of 64 over 2: the tile
// kernel reads as much for one row as for 128.) The host does not know how they are spread: one cloud of 3000 rows
// beside 200 of one row (2000 keys each, window 1024, 8 heads of 64 over 2) takes 648 us here, where the two
// alone take 40 us in tiles and 67 us here. Calls that mix prompts and single rows are better split.
bool takes_stream(const gdl_attention &a) {
    const int per = a.dtype == GDL_DTYPE_BF16 ? 8 : 4, bytes = 16 / per;
    const auto fits = [&](const void *p, int64_t head, int64_t row) {
        return ((uintptr_t)p & 15) == 0 && head * bytes % 16 == 0 && row * bytes % 16 == 0;
    };
    return a.n_query <= (int64_t)16 * a.num_clouds && a.n_query <= 65536 && a.dim % per == 0 && a.kv_heads * a.heads < 65536 &&
           fits(a.q, a.q_head, a.q_row) && fits(a.k, a.k_head, a.k_row) && fits(a.v, a.v_head, a.v_row);
}

int attention_forward_stream(const gdl_attention &a, void *out, float *lse, void *rest, cudaStream_t st) {
    return a.dtype == GDL_DTYPE_F32 ? stream_forward<float>(a, (float *)out, lse, nullptr, st)
                                    : stream_forward<uint16_t>(a, (uint16_t *)out, lse, (uint16_t *)rest, st);
}

}  // namespace gdl
