// attention_sinks.cuh -- how the dK, dV kernels of the windowed attention share out their work.
//
// A CTA takes a tile of keys and the queries whose windows reach it. Sinks are seen by every later query as
// well: the queries beyond their tile's windows are split into chunks, each a CTA of its own that leaves f32
// partial sums of the sinks' rows; a last kernel adds them in order.
#pragma once

#include "attention_mma.cuh"

namespace gdl {

// Partial sums lie in rows of [2][dim] floats (dK, dV), for each key head: a cloud's sinks take as many as it has, so
// that cloud b starts at min(b * sinks, its first key) and no two overlap; chunk i of a cloud's queries takes them
// (first query / size + i) * sinks rows further on.
struct SinkPlan {
    int tiles;       // key tiles with sinks in them
    int sinks, size; // sinks of a cloud at most; queries of a chunk
    int64_t slots;   // chunks (slots of a ragged tiling)
    int64_t main_rows, chunk_rows;  // of one key head
    float *main, *chunk;
};
__device__ __forceinline__ int64_t sink_base(const SinkPlan &sp, int64_t cloud, int64_t k0) {
    return cloud * sp.sinks < k0 ? cloud * sp.sinks : k0;
}

// queries of a cloud that the window alone lets see keys up to j1: the end of a tile's own range
__device__ __forceinline__ int64_t window_end(const gdl_attention &a, int64_t j1, int64_t nq, int64_t nk) {
    if (a.left < 0) return nq;
    const int64_t e = j1 + a.left + 1 - (nk - nq);
    return e < 0 ? 0 : e > nq ? nq : e;
}

// `chunk`: queries of a chunk where sinks are few. With many it grows, so that the chunks of all queries together have
// no more rows than there are keys (131072 rows, 4 key heads of 64, 2048 sinks: 0.27 GB in chunks of 2048).
inline SinkPlan sink_plan(const gdl_attention &a, float *ws, int tile_rows, int chunk) {
    SinkPlan sp = {};
    if (a.left < 0 || a.num_sinks == 0 || a.n_key == 0 || a.n_query == 0) return sp;
    sp.sinks = (int)(a.num_sinks < a.n_key ? a.num_sinks : a.n_key);
    sp.tiles = (sp.sinks + tile_rows - 1) / tile_rows;
    const int64_t least = (a.n_query * sp.sinks + a.n_key - 1) / a.n_key;
    const int64_t size = (least + chunk - 1) / chunk * chunk;
    sp.size = (int)(size < ((int64_t)1 << 30) ? size : (int64_t)1 << 30);
    sp.slots = ragged_slots(a.n_query, a.num_clouds, sp.size);
    const int64_t every = (int64_t)a.num_clouds * sp.sinks;
    sp.main_rows = every < a.n_key ? every : a.n_key;
    sp.chunk_rows = a.n_query / sp.size * sp.sinks + sp.main_rows;
    sp.main = ws;
    sp.chunk = ws ? ws + sp.main_rows * a.kv_heads * 2 * a.dim : nullptr;
    return sp;
}
inline size_t sink_bytes(const gdl_attention &a, int chunk) {
    const SinkPlan sp = sink_plan(a, nullptr, 1, chunk);
    return (size_t)(sp.main_rows + sp.chunk_rows) * a.kv_heads * 2 * a.dim * sizeof(float);
}

// What a CTA does: CTAs 0 .. main - 1 are the key tiles (slot * kv_heads + head), then the sinks' chunks.
struct SinkUnit {
    bool skip, chunk;
    int hk, rows;                    // keys j0 .. j0 + rows of the cloud
    int first_out;                   // rows below it go to the partial, the others are final
    int64_t q0, nq, k0, nk, j0;      // the cloud's queries and keys
    int64_t lo, hi;                  // queries of the cloud
    float *partial;                  // [rows][2][dim]
};
__device__ __forceinline__ SinkUnit sink_unit(const gdl_attention &a, const SinkPlan &sp, int64_t main_ctas, int tile_rows) {
    SinkUnit u = {};
    u.chunk = blockIdx.x >= main_ctas;
    const int64_t unit = u.chunk ? blockIdx.x - main_ctas : blockIdx.x;
    u.hk = (int)(unit % a.kv_heads);
    u.skip = true;
    if (u.chunk) {
        const int s = (int)(unit / a.kv_heads % sp.tiles);
        const Tile t = ragged_tile(a.ptr_q, a.num_clouds, a.n_query, sp.size, unit / a.kv_heads / sp.tiles);
        if (t.cloud < 0) return u;
        u.q0 = t.start;
        u.nq = t.n;
        u.k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 1);
        const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, t.cloud + 2);
        u.nk = k1 > u.k0 ? k1 - u.k0 : 0;
        u.j0 = (int64_t)s * tile_rows;
        const int64_t j1 = u.j0 + tile_rows < u.nk ? u.j0 + tile_rows : u.nk, js = j1 < a.num_sinks ? j1 : a.num_sinks;
        if (js <= u.j0) return u;
        u.rows = u.first_out = (int)(js - u.j0);
        const int64_t end = window_end(a, j1 - 1, u.nq, u.nk);
        u.lo = end > t.first ? end : t.first;
        u.hi = t.first + sp.size < u.nq ? t.first + sp.size : u.nq;
        if (u.hi <= u.lo) return u;  // the last kernel skips it by the same rule
        u.partial = sp.chunk + (u.hk * sp.chunk_rows + (u.q0 / sp.size + t.first / sp.size) * sp.sinks +
                                sink_base(sp, t.cloud, u.k0) + u.j0) * 2 * a.dim;
    } else {
        const Tile t = ragged_tile(a.ptr_k, a.num_clouds, a.n_key, tile_rows, unit / a.kv_heads);
        if (t.cloud == -2) return u;
        u.k0 = t.start;
        u.nk = t.n;
        u.j0 = t.first;
        u.rows = (int)(u.nk - u.j0 < tile_rows ? u.nk - u.j0 : tile_rows);
        if (t.cloud >= 0) {
            u.q0 = ragged_bound(a.ptr_q, a.num_clouds, a.n_query, t.cloud + 1);
            const int64_t q1 = ragged_bound(a.ptr_q, a.num_clouds, a.n_query, t.cloud + 2);
            u.nq = q1 > u.q0 ? q1 - u.q0 : 0;
            u.lo = visible_queries(a, u.j0, u.nq, u.nk).lo;
            u.hi = window_end(a, u.j0 + u.rows - 1, u.nq, u.nk);
            if (sp.tiles > 0 && u.j0 < a.num_sinks) {
                u.partial = sp.main + (u.hk * sp.main_rows + sink_base(sp, t.cloud, u.k0) + u.j0) * 2 * a.dim;
                u.first_out = (int)(a.num_sinks - u.j0 < u.rows ? a.num_sinks - u.j0 : u.rows);
            }
        }
    }
    u.skip = false;
    return u;
}

// dk, dv of the sinks: their own tile's sums and the chunks' in order; one CTA to a cloud's tile and head
template <typename T>
static __global__ void __launch_bounds__(256)
    attn_sink_join_kernel(const __grid_constant__ gdl_attention a, const SinkPlan sp, int tile_rows, T *__restrict__ dk,
                          T *__restrict__ dv) {
    const int hk = blockIdx.x % a.kv_heads, s = blockIdx.x / a.kv_heads % sp.tiles;
    const int b = blockIdx.x / a.kv_heads / sp.tiles;
    const int64_t q0 = ragged_bound(a.ptr_q, a.num_clouds, a.n_query, b + 1);
    const int64_t q1 = ragged_bound(a.ptr_q, a.num_clouds, a.n_query, b + 2);
    const int64_t k0 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, b + 1);
    const int64_t k1 = ragged_bound(a.ptr_k, a.num_clouds, a.n_key, b + 2);
    const int64_t nq = q1 > q0 ? q1 - q0 : 0, nk = k1 > k0 ? k1 - k0 : 0;
    const int64_t j0 = (int64_t)s * tile_rows, j1 = j0 + tile_rows < nk ? j0 + tile_rows : nk;
    const int64_t js = j1 < a.num_sinks ? j1 : a.num_sinks;
    if (js <= j0) return;
    const int64_t end = window_end(a, j1 - 1, nq, nk), at = sink_base(sp, b, k0) + j0;
    const float *main = sp.main + (hk * sp.main_rows + at) * 2 * a.dim;
    const int64_t first = end < nq ? end / sp.size : 0, last = end < nq ? (nq - 1) / sp.size + 1 : 0;
    const int64_t step = (int64_t)sp.sinks * 2 * a.dim;
    const float *chunk = sp.chunk + (hk * sp.chunk_rows + q0 / sp.size * sp.sinks + at) * 2 * a.dim;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < (int)(js - j0) * 2 * a.dim; i += gridDim.y * 256) {
        float sum = main[i];
#pragma unroll 8
        for (int64_t c = first; c < last; ++c) sum += chunk[c * step + i];
        const int r = i / (2 * a.dim), half = i / a.dim & 1, d = i % a.dim;
        store1((half ? dv : dk) + ((k0 + j0 + r) * a.kv_heads + hk) * a.dim + d, sum);
    }
}
template <typename T>
int join_sinks(const gdl_attention &a, const SinkPlan &sp, int tile_rows, T *dk, T *dv, cudaStream_t st) {
    if (sp.tiles == 0 || a.num_clouds == 0) return GDL_OK;
    const int64_t ctas = (int64_t)a.num_clouds * sp.tiles * a.kv_heads;
    GDL_RETURN_IF(ctas > ((int64_t)1 << 31) - 1, GDL_ERR_OVERFLOW);
    const int rows = sp.sinks < tile_rows ? sp.sinks : tile_rows, blocks = (rows * 2 * a.dim + 255) / 256;
    attn_sink_join_kernel<T><<<dim3((unsigned)ctas, blocks), 256, 0, st>>>(a, sp, tile_rows, dk, dv);
    GDL_CUDA_TRY(cudaGetLastError());
    return GDL_OK;
}

}  // namespace gdl
