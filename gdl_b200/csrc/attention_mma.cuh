// attention_mma.cuh -- what the tensor-core kernels of the windowed attention share: the tiles of keys (or
// queries) that a CTA visits, their masks, the logits of a row, and the tensor maps.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "tc.cuh"

namespace gdl {

constexpr int kMmaRows = 128;  // rows of a CTA: the M of its products, one TMEM lane and thread each
constexpr int kMmaKeys = 64;   // columns of one S tile

// the lowest x bits (all 32 for x >= 32, none for x <= 0); shl gives 0 for 32 and more
__device__ __forceinline__ uint32_t bits_below(int x) {
    uint32_t r;
    asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(1u), "r"(x > 0 ? x : 0));
    return r - 1;
}

// One of the stages of a ring of buffers, and the parity of its barrier's phase.
template <int N>
struct Ring {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) {
            at = 0;
            parity ^= 1;
        }
    }
};

// Waits (bounded) until the last n loads before ring place `next` have landed.
template <int N>
__device__ void drain(uint32_t bar, Ring<N> next, int n) {
    for (; n > 0; --n) {
        if (next.at-- == 0) {
            next.at = N - 1;
            next.parity ^= 1;
        }
        tc::mbar_wait(bar + 8 * next.at, next.parity);
    }
}

// Tiles of keys for queries at places i0 .. i1 of a cloud: `sink` tiles over [0, sinks), then tiles over
// the span [lo, hi) of their windows. Each visible key lies in exactly one of them. Places within a cloud
// fit 32 bits (a cloud has fewer than 2^31 rows).
struct KeyTiles {
    int sinks, lo, hi;
    int every_lo, every_hi;  // keys that every query sees: [every_lo, every_hi), and the sinks below every_hi
    int sink, count;
};
// The tile that a loop over i = 0 .. count - 1 is at: keys [j, end), at most 64 of them.
struct KeyTile {
    int i, j, end;
    __device__ __forceinline__ explicit KeyTile(const KeyTiles &t)
        : i(0), j(t.sink ? 0 : t.lo), end(t.sink ? t.sinks : t.hi) {}
    __device__ __forceinline__ void next(const KeyTiles &t) {
        j += kMmaKeys;
        if (++i == t.sink) {
            j = t.lo;
            end = t.hi;
        }
    }
    // every query sees every key of it
    __device__ __forceinline__ bool full(const KeyTiles &t, int num_sinks) const {
        const int e = j + kMmaKeys;
        return e <= end && e <= t.every_hi && (j >= t.every_lo || e <= num_sinks);
    }
    // columns off .. off + 31 that a row sees whose window is [lo, hi)
    __device__ __forceinline__ uint32_t mask(int off, int lo, int hi, int num_sinks) const {
        const int at = j + off;
        return bits_below((end < hi ? end : hi) - at) & (~bits_below(lo - at) | bits_below(num_sinks - at));
    }
};

__device__ __forceinline__ KeyTiles key_tiles(const gdl_attention &a, int64_t i0, int64_t i1, int64_t nk) {
    KeyTiles t;
    const KeyRange first = visible_keys(a, i0, nk), last = visible_keys(a, i1, nk);
    t.lo = (int)first.lo;
    t.every_hi = (int)first.hi;
    t.every_lo = (int)last.lo;
    t.hi = (int)last.hi;
    t.sinks = a.num_sinks < t.lo ? a.num_sinks : t.lo;
    if (t.sinks > t.hi) t.sinks = t.hi;
    t.sink = (t.sinks + kMmaKeys - 1) / kMmaKeys;
    t.count = t.sink + (t.hi > t.lo ? (t.hi - t.lo + kMmaKeys - 1) / kMmaKeys : 0);
    return t;
}

// Reads of the bias table: pure, so that they move freely between the loads and stores around them (the table
// is written before the products whose results an address is made of).
__device__ __forceinline__ float lds(uint32_t addr) {
    float v;
    asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint32_t mad(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("mad.lo.u32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }

// dist2() of two pairs of points, for the negated coordinates of one of them: a sum where dist2_x2 has a
// difference (its square is the same), since packed operands have no free sign.
__device__ __forceinline__ uint64_t dist2_neg(uint64_t nx, uint64_t ny, uint64_t nz, uint64_t x, uint64_t y,
                                              uint64_t z) {
    const uint64_t dx = add2(nx, x), dy = add2(ny, y), dz = add2(nz, z);
    uint64_t r;
    asm("mul.rn.ftz.f32x2 %0, %1, %1;" : "=l"(r) : "l"(dy));
    asm("fma.rn.ftz.f32x2 %0, %1, %1, %2;" : "=l"(r) : "l"(dx), "l"(r));
    asm("fma.rn.ftz.f32x2 %0, %1, %1, %2;" : "=l"(r) : "l"(dz), "l"(r));
    return r;
}

// The bias of one row: its negated position in packed pairs, and the bucket arithmetic. The table lies in
// shared memory as [buckets][32], a copy for each lane (any lane's bucket is free of bank conflicts).
struct RowBias {
    uint64_t nx, ny, nz, inv2;
    unsigned shift, top, low;  // bucket = min(bits(t) >> shift, top) - low
    uint32_t tab;              // address of this lane's copy, less low rows
};
__device__ __forceinline__ RowBias row_bias(const gdl_attention &a, const float *p, const float *table) {
    RowBias b;
    b.nx = pack2(-p[0], -p[0]);
    b.ny = pack2(-p[1], -p[1]);
    b.nz = pack2(-p[2], -p[2]);
    b.inv2 = pack2(a.inv_radius2, a.inv_radius2);
    b.shift = 23 - a.steps_log2;
    b.low = 127u << a.steps_log2;
    b.top = b.low + a.buckets - 1;
    b.tab = tc::smem_addr(table) + (threadIdx.x & 31) * 4 - b.low * 128;
    return b;
}
// buckets (plus b.low) of columns c .. c + 3; pos [3][64] in shared memory
__device__ __forceinline__ void buckets4(const RowBias &b, const float *pos, int c, unsigned (&u)[4]) {
    const uint64_t one2 = pack2(1.0f, 1.0f);
    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(pos + c);
    const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(pos + kMmaKeys + c);
    const ulonglong2 z = *reinterpret_cast<const ulonglong2 *>(pos + 2 * kMmaKeys + c);
    float t[4];
    unpack2(fma2(dist2_neg(b.nx, b.ny, b.nz, x.x, y.x, z.x), b.inv2, one2), t[0], t[1]);
    unpack2(fma2(dist2_neg(b.nx, b.ny, b.nz, x.y, y.y, z.y), b.inv2, one2), t[2], t[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned v = __float_as_uint(t[e]) >> b.shift;
        u[e] = min(v, b.top);
    }
}
// Products of columns c .. c + 3 to two pairs of logits in powers of two: s * scale2 (+ bias)
template <bool BIAS>
__device__ __forceinline__ void logits4(const uint32_t *s, uint64_t scale2, const RowBias &b, const unsigned (&u)[4],
                                        uint64_t &x01, uint64_t &x23) {
    if (BIAS) {
        x01 = fma2(pair(s[0], s[1]), scale2, pack2(lds(mad(u[0], 128, b.tab)), lds(mad(u[1], 128, b.tab))));
        x23 = fma2(pair(s[2], s[3]), scale2, pack2(lds(mad(u[2], 128, b.tab)), lds(mad(u[3], 128, b.tab))));
    } else {
        x01 = mul2(pair(s[0], s[1]), scale2);
        x23 = mul2(pair(s[2], s[3]), scale2);
    }
}

// What a warp's 32 rows see of a tile, by chunks of 16 columns: none of them anything (nothing is computed),
// all of them everything (no mask), or a part. Windows are diagonal bands, so few chunks are the latter.
constexpr int kChunk = 16;
struct ChunkSets {
    unsigned any, all;  // bit k: chunk k
};
// chunks 2 w, 2 w + 1 from the mask of columns 32 w .. 32 w + 31
__device__ __forceinline__ ChunkSets chunk_sets(uint32_t mask, int w = 0) {
    const bool a0 = (mask & 0xffffu) != 0, a1 = mask > 0xffffu, f0 = (mask & 0xffffu) == 0xffffu,
               f1 = mask >= 0xffff0000u;
    ChunkSets s;
    s.any = ((__any_sync(0xffffffffu, a0) ? 1u : 0u) | (__any_sync(0xffffffffu, a1) ? 2u : 0u)) << (2 * w);
    s.all = ((__all_sync(0xffffffffu, f0) ? 1u : 0u) | (__all_sync(0xffffffffu, f1) ? 2u : 0u)) << (2 * w);
    return s;
}

// Replaces what is not finite in a tile of 64 rows (panels of 64 bf16, rows of 128 bytes) by 0, and returns
// the rows that had any; called by the softmax threads (r; 128 of them work) for tiles i = 0, 1, ... in turn, with `words`
// three times two words of shared memory, 0 at first (tile i clears those of tile i + 2: its readers of tile
// i - 1 are past the barrier). The writes reach the products that are issued after this thread's next
// arrival on an mbarrier. ok = false: a wait gave up.
template <int PANELS>
__device__ __noinline__ uint2 zero_nonfinite(uint32_t tile, uint32_t *words, uint32_t bar, int i, int r, bool &ok) {
    uint32_t *mine = words + i % 3 * 2;
    bool any = false;
    for (int p = 0; p < PANELS && r < 128; ++p)
        for (int c = 0; c < 16; ++c) {  // half a row: 16 words
            const uint32_t at = tile + p * kMmaKeys * 128 + (r >> 1) * 128 + (r & 1) * 64 + c * 4;
            uint32_t w, v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
            v = (w & 0x7f80u) == 0x7f80u ? w & 0xffff0000u : w;
            v = (v & 0x7f800000u) == 0x7f800000u ? v & 0xffffu : v;
            if (v != w) {
                any = true;
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(v));
            }
        }
    if (any) atomicOr(mine + (r >> 6), 1u << ((r >> 1) & 31));
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc::mbar_arrive(bar);
    ok = ok && tc::mbar_wait(bar, i & 1);
    if (r < 2) words[(i + 2) % 3 * 2 + r] = 0;
    volatile uint32_t *w = mine;
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void zero_rows(uint16_t *p, int64_t stride, int rows, int dim) {
    for (int i = threadIdx.x; i < rows * dim; i += blockDim.x) p[(int64_t)(i / dim) * stride + i % dim] = 0;
}

// Tensor map of [rows][heads][dim] bf16 with boxes of 64 columns of one head x `box` rows, 128-byte
// swizzle; columns beyond dim read as 0. false: the driver refused it.
bool head_map(CUtensorMap *map, const void *base, int dim, int heads, int64_t rows, int64_t head_stride,
              int64_t row_stride, int box);

// whether the tensor-core kernels can read these inputs: bf16, dim a multiple of 8, 16-byte aligned rows
// and heads
bool mma_layout(const void *p, int64_t head_stride, int64_t row_stride, int heads, int64_t rows, int dim);

int attention_forward_mma(const gdl_attention &a, uint16_t *out, float *lse, uint16_t *rest, cudaStream_t st);
bool takes_stream(const gdl_attention &a);
int attention_forward_stream(const gdl_attention &a, void *out, float *lse, void *rest, cudaStream_t st);
int attention_simt_rows();
int attention_forward_simt(const gdl_attention &a, void *out, float *lse, void *rest, cudaStream_t st);
int attention_backward_simt(const gdl_attention &a, const void *out, const float *lse, const void *rest, const void *dout, void *dq, void *dk,
                            void *dv, const RowStats stats, float *part, float *sink_ws, int chunk, cudaStream_t st);
int attention_backward_mma(const gdl_attention &a, const uint16_t *out, const float *lse, const uint16_t *rest, const uint16_t *dout,
                           uint16_t *dq, uint16_t *dk, uint16_t *dv, const RowStats stats, float *part, float *sink_ws,
                           int chunk, cudaStream_t st);

}  // namespace gdl
