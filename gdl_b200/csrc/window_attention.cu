// window_attention.cu -- attention over packed clouds with a sliding window, sinks and a distance bias:
// argument checks, the choice of the kernels, and the last sum of the bias gradient.
#include "attention_sinks.cuh"

namespace gdl {
namespace {

// dbias[h][b] = sum over the partials, in a fixed order; one CTA to an entry
template <typename TB>
__global__ void __launch_bounds__(256) attn_dbias_kernel(const float *__restrict__ part, int64_t parts, int heads,
                                                         int buckets, TB *__restrict__ dbias) {
    __shared__ float sums[8];
    const int64_t at = blockIdx.x;
    float s = 0.0f;
    for (int64_t k = threadIdx.x; k < parts; k += 256) s += part[k * heads * buckets + at];
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float total = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) total += sums[k];
        store1(dbias + at, total);
    }
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

int check(const gdl_attention *a) {
    GDL_RETURN_IF(!a, GDL_ERR_INVALID);
    GDL_RETURN_IF(a->dtype != GDL_DTYPE_F32 && a->dtype != GDL_DTYPE_BF16, GDL_ERR_INVALID);
    GDL_RETURN_IF(a->num_clouds < 0 || a->n_query < 0 || a->n_key < 0 || a->heads < 1 || a->kv_heads < 1 ||
                      a->heads % a->kv_heads != 0 || a->dim < 1 || a->num_sinks < 0 || a->left < -1 || a->right < -1,
                  GDL_ERR_INVALID);
    GDL_RETURN_IF(a->dim > kAttnMaxDim, GDL_ERR_UNSUPPORTED);
    GDL_RETURN_IF(!a->ptr_q || !a->ptr_k, GDL_ERR_INVALID);
    GDL_RETURN_IF(a->n_query > 0 && !a->q, GDL_ERR_INVALID);
    GDL_RETURN_IF(a->n_key > 0 && (!a->k || !a->v), GDL_ERR_INVALID);
    if (a->bias) {
        GDL_RETURN_IF(a->buckets < 1 || a->buckets > kAttnMaxBuckets || a->steps_log2 < 0 || a->steps_log2 > 4 ||
                          (a->bias_dtype != GDL_DTYPE_F32 && a->bias_dtype != GDL_DTYPE_BF16) ||
                          !(a->inv_radius2 >= 0.0f && a->inv_radius2 <= 3.4028234e38f),  // (t below 1 has no bucket)
                      GDL_ERR_INVALID);
        GDL_RETURN_IF((a->n_query > 0 && !a->pos_q) || (a->n_key > 0 && !a->pos_k), GDL_ERR_INVALID);
    }
    GDL_RETURN_IF(a->heads > 65535 || a->n_query > ((int64_t)1 << 31) - 1 || a->n_key > ((int64_t)1 << 31) - 1,
                  GDL_ERR_OVERFLOW);
    return GDL_OK;
}

// The same windows in numbers that leave room for sums of places: a side that reaches over all rows is open, and
// where every key is a sink (or the left side is open) there is nothing for sinks to do.
gdl_attention normal(const gdl_attention &given) {
    gdl_attention a = given;
    if (a.left >= a.n_key || a.num_sinks >= a.n_key) a.left = -1;
    if (a.right >= a.n_key + a.n_query) a.right = -1;
    if (a.left < 0) a.num_sinks = 0;
    return a;
}

// Which kernels take a call: few rows stream the window (window_attention_stream.cu), bf16 in layouts that TMA
// can read goes to the tensor cores (window_attention_mma*.cu), everything else (f32, head sizes that are no
// multiple of 8, unaligned views) to the FFMA tiles (window_attention_simt.cu).
bool takes_mma(const gdl_attention &a) {
    return a.dtype == GDL_DTYPE_BF16 && a.n_key > 0 && a.n_query > 0 &&
           mma_layout(a.q, a.q_head, a.q_row, a.heads, a.n_query, a.dim) &&
           mma_layout(a.k, a.k_head, a.k_row, a.kv_heads, a.n_key, a.dim) &&
           mma_layout(a.v, a.v_head, a.v_row, a.kv_heads, a.n_key, a.dim);
}

int reduce_bias(const gdl_attention &a, const float *part, int64_t parts, void *dbias, cudaStream_t st) {
    if (a.bias_dtype == GDL_DTYPE_F32)
        attn_dbias_kernel<float><<<a.heads * a.buckets, 256, 0, st>>>(part, parts, a.heads, a.buckets, (float *)dbias);
    else
        attn_dbias_kernel<uint16_t><<<a.heads * a.buckets, 256, 0, st>>>(part, parts, a.heads, a.buckets,
                                                                         (uint16_t *)dbias);
    GDL_CUDA_TRY(cudaGetLastError());
    return GDL_OK;
}

// Queries of a chunk of the sinks': 16 tiles on the tensor cores, 4 in the FFMA tiles (8: 131 instead of 101 us for dK,
// dV of 6 ragged clouds up to 1023 rows, 4 heads of 24 over 2). By the inputs alone, as the workspace is asked for.
int sink_chunk(const gdl_attention &a) { return takes_mma(a) ? 1024 : 128; }

// workspace: the rows' stats [3][heads][n_query], the bucket sums of each slot of query rows, the sinks' partial sums
size_t stats_bytes(const gdl_attention &a) { return align256((size_t)3 * a.heads * a.n_query * 4); }
size_t part_bytes(const gdl_attention &a) {
    return a.bias ? align256((size_t)ragged_slots(a.n_query, a.num_clouds, attention_simt_rows()) * a.heads * a.buckets * 4) : 0;
}

}  // namespace
}  // namespace gdl

using namespace gdl;

extern "C" int gdl_window_attention(const gdl_attention *given, void *out, float *lse, void *out_rest, void *stream) {
    const int rc = check(given);
    if (rc != GDL_OK) return rc;
    const gdl_attention a = normal(*given);
    if (a.n_query == 0) return GDL_OK;
    GDL_RETURN_IF(!out, GDL_ERR_INVALID);
    cudaStream_t st = (cudaStream_t)stream;
    GDL_RETURN_IF(out_rest && a.dtype != GDL_DTYPE_BF16, GDL_ERR_INVALID);
    const bool few = takes_stream(a);
    if (!few && takes_mma(a) && (((uintptr_t)out | (uintptr_t)out_rest) & 15) == 0)
        return attention_forward_mma(a, (uint16_t *)out, lse, (uint16_t *)out_rest, st);
    if (few) return attention_forward_stream(a, out, lse, out_rest, st);
    return attention_forward_simt(a, out, lse, out_rest, st);
}

extern "C" size_t gdl_window_attention_backward_workspace_size(const gdl_attention *given) {
    if (check(given) != GDL_OK) return 256;
    const gdl_attention a = normal(*given);
    return stats_bytes(a) + part_bytes(a) + sink_bytes(a, sink_chunk(a)) + 256;
}

extern "C" int gdl_window_attention_backward(const gdl_attention *given, const void *out, const float *lse,
                                             const void *out_rest, const void *grad_out, void *dq, void *dk, void *dv,
                                             void *dbias, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = check(given);
    if (rc != GDL_OK) return rc;
    const gdl_attention a = normal(*given);
    GDL_RETURN_IF(a.n_query > 0 && (!out || !lse || !grad_out || !dq), GDL_ERR_INVALID);
    GDL_RETURN_IF(a.n_key > 0 && (!dk || !dv), GDL_ERR_INVALID);
    GDL_RETURN_IF(dbias && !a.bias, GDL_ERR_INVALID);
    GDL_RETURN_IF(!workspace || workspace_bytes < gdl_window_attention_backward_workspace_size(given), GDL_ERR_WORKSPACE);
    cudaStream_t st = (cudaStream_t)stream;
    char *ws = (char *)workspace;
    const RowStats stats = {(float *)ws, (int64_t)a.heads * a.n_query};
    float *part = dbias ? (float *)(ws + stats_bytes(a)) : nullptr;
    float *sinks = (float *)(ws + stats_bytes(a) + part_bytes(a));
    const uintptr_t all = (uintptr_t)out | (uintptr_t)out_rest | (uintptr_t)grad_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv;
    const bool mma = takes_mma(a) && (all & 15) == 0;
    const int done = mma ? attention_backward_mma(a, (const uint16_t *)out, lse, (const uint16_t *)out_rest,
                                                  (const uint16_t *)grad_out, (uint16_t *)dq, (uint16_t *)dk,
                                                  (uint16_t *)dv, stats, part, sinks, sink_chunk(a), st)
                         : attention_backward_simt(a, out, lse, out_rest, grad_out, dq, dk, dv, stats, part, sinks, sink_chunk(a), st);
    if (done != GDL_OK || !dbias) return done;
    const int64_t parts = ragged_slots(a.n_query, a.num_clouds, mma ? kMmaRows : attention_simt_rows());
    return reduce_bias(a, part, a.n_query > 0 ? parts : 0, dbias, st);
}
