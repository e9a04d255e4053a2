// gated_scan.cu -- gated linear recurrence along packed clouds, forward and backward (sm_100a).
//
//     log a_t = -softplus(decay_c) sigmoid(gate_t),  b_t = sqrt(1 - a_t^2),  h_t = a_t h_{t-1} + b_t x_t
// backward, for dh, with c_t = a_t g_t the gradient that row t hands to the row before it:
//     g_t = dh_t + c_{t+1},  dx_t = b_t g_t,
//     dl_t = a_t g_t (h_{t-1} - x_t a_t / b_t)                 (the derivative by log a_t),
//     dgate_t = dl_t log a_t (1 - sigmoid(gate_t)),  ddecay_c = -sigmoid(decay_c) sum_t dl_t sigmoid(gate_t)
//
// A row is an affine map h -> a h + u, and maps compose: a block of rows is (A, H) with h_out = A h_in + H.
// So the scan runs in three launches, each wide over rows and channels: (1) every warp folds a segment of 32
// or 64 rows (lanes: channels) and every CTA its 8 segments; (2) per cloud and channel, the CTAs' maps are chained to
// the state before each; (3) every warp goes over its segment again from its state and writes. The rows are
// read twice, 5 transfers instead of 3 (7 instead of 5 backward). The backward is the same in the other
// direction, with h recomputed from the f32 states that the forward kept (one to 16 rows): h itself is not
// read back, and its rounding to bf16 does not reach the gradients. All orders of summation are fixed.
//
// 8 x 131072 rows of 64 channels, bf16: fold 77 us, chain 5, write 92; backwards 68, 7, 188. By their bytes the
// four large ones would take 42, 65, 42 and 107 us at the measured copy rate.
#include "attention_mma.cuh"

namespace gdl {
namespace {

constexpr int kBlock = 16;     // rows that a warp has in registers at once, and to a kept state
constexpr int kWarps = 8;      // segments of a CTA; a segment is NB blocks
constexpr int scan_rows(int nb) { return kBlock * nb * kWarps; }
constexpr int kScanThreads = 32 * kWarps;
constexpr int kChainWarps = 32;
// Calls of so few rows run in one launch, a thread to a channel of a cloud: 3 launches take longer than a few
// rows in turn (64 clouds of one row, 256 channels: 2.4 us).
constexpr int64_t kSerialRows = 256;
constexpr int kSerialClouds = 65533;  // (with the rows of no cloud, the y of a grid)
bool takes_serial(int64_t n_rows, int32_t clouds) { return n_rows <= kSerialRows && clouds <= kSerialClouds; }

__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rsqrt_approx(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// Two channels of one row: what comes of the gate.
struct Gate {
    uint64_t sig, l, a, b;
};

// sigmoid(gate), l = log a, a and b of two elements; nrate = -softplus(decay). 1 - a is what a long memory is
// made of (an error e of a grows to e / (1 - a) in h), so it comes from a series and a from it: with y = -l / 4,
// q = 1 - exp(-y) = y (1 - y/2 + ... + y^6/5040) (under 2e-8 of it for y < 0.35), and twice 1 - exp(-2y) =
// q (2 - q). b = sqrt((1 - a)(1 + a)) has no cancellation either way. WIDE: some channel of the warp can have
// l < -1.4, where exp(l) is taken directly. 3 special-function instructions (4 if wide).
template <bool NEED_B, bool WIDE>
__device__ __forceinline__ Gate scan_gate(uint64_t gate, uint64_t nrate) {
    Gate g;
    const uint64_t one = both(1.0f), z = mul2(gate, both(-kLog2e));
    const uint64_t d = add2(pack2(ex2(lo(z)), ex2(hi(z))), one);
    g.sig = pack2(rcp(lo(d)), rcp(hi(d)));
    g.l = mul2(nrate, g.sig);
    const uint64_t y = mul2(g.l, both(-0.25f));
    uint64_t s = fma2(y, both(1.0f / 5040.0f), both(-1.0f / 720.0f));
    s = fma2(y, s, both(1.0f / 120.0f));
    s = fma2(y, s, both(-1.0f / 24.0f));
    s = fma2(y, s, both(1.0f / 6.0f));
    s = fma2(y, s, both(-0.5f));
    s = fma2(y, s, one);
    uint64_t q = mul2(y, s);
    const uint64_t two = both(2.0f), minus = both(-1.0f);
    q = mul2(q, fma2(q, minus, two));
    uint64_t e = mul2(q, fma2(q, minus, two));  // 1 - a
    g.a = fma2(e, minus, one);
    if (WIDE) {
        const float f0 = ex2(kLog2e * lo(g.l)), f1 = ex2(kLog2e * hi(g.l));
        const bool w0 = lo(g.l) < -1.4f, w1 = hi(g.l) < -1.4f;
        g.a = pack2(w0 ? f0 : lo(g.a), w1 ? f1 : hi(g.a));
        e = pack2(w0 ? 1.0f - f0 : lo(e), w1 ? 1.0f - f1 : hi(e));
    }
    if (NEED_B) {
        const uint64_t v = mul2(e, add2(g.a, one)), w = add2(v, both(1e-30f));  // 0 stays 0
        g.b = mul2(v, pack2(rsqrt_approx(lo(w)), rsqrt_approx(hi(w))));
    }
    return g;
}

__device__ __forceinline__ float softplus(float d) { return d > 20.0f ? d : log1pf(expf(d)); }

// VEC = 2: a lane has channels c, c + 1 (an even number of channels, so that pairs stay aligned); 1: channel c
// alone, and 0 beside it.
// A segment's rows are loaded as they are, all at once, and widened where they are used.
template <typename T, int VEC>
struct Raw;
template <>
struct Raw<float, 2> {
    uint64_t v = 0;
    __device__ __forceinline__ void load(const float *p) { v = __ldg(reinterpret_cast<const unsigned long long *>(p)); }
    __device__ __forceinline__ uint64_t wide() const { return v; }
};
template <>
struct Raw<float, 1> {
    float v = 0.0f;
    __device__ __forceinline__ void load(const float *p) { v = __ldg(p); }
    __device__ __forceinline__ uint64_t wide() const { return pack2(v, 0.0f); }
};
template <>
struct Raw<uint16_t, 2> {
    uint32_t v = 0;
    __device__ __forceinline__ void load(const uint16_t *p) { v = __ldg(reinterpret_cast<const uint32_t *>(p)); }
    __device__ __forceinline__ uint64_t wide() const { return pair(v << 16, v & 0xffff0000u); }
};
template <>
struct Raw<uint16_t, 1> {
    uint32_t v = 0;
    __device__ __forceinline__ void load(const uint16_t *p) { v = (uint32_t)__ldg(p) << 16; }
    __device__ __forceinline__ uint64_t wide() const { return pair(v, 0); }
};
template <int VEC>
__device__ __forceinline__ void store2(float *p, uint64_t v) {
    if (VEC == 2)
        *reinterpret_cast<float2 *>(p) = make_float2(lo(v), hi(v));
    else
        *p = lo(v);
}
template <int VEC>
__device__ __forceinline__ void store2(uint16_t *p, uint64_t v) {
    if (VEC == 2)
        *reinterpret_cast<uint32_t *>(p) = tc::pack_bf16(lo(v), hi(v));
    else
        *p = f32_to_bf16_bits(lo(v));
}

// One warp's segment: its cloud, its rows in the direction of the recurrence, its channels.
struct Segment {
    Tile t;
    int64_t first;  // step of the segment's first row within the cloud
    int n;          // rows, 0 .. kBlock * NB
    int c;          // first channel of the lane
    bool on;        // the lane has a channel
};
template <int VEC, int NB>
__device__ __forceinline__ Segment segment(const int64_t *__restrict__ ptr, int B, int64_t n_rows, int C) {
    Segment s;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    s.t = ragged_tile(ptr, B, n_rows, scan_rows(NB), blockIdx.x);
    s.first = s.t.first + warp * (kBlock * NB);
    const int64_t left = s.t.cloud == -2 ? 0 : s.t.n - s.first;
    s.n = left <= 0 ? 0 : left < kBlock * NB ? (int)left : kBlock * NB;
    s.c = (blockIdx.y * 32 + lane) * VEC;
    s.on = s.c < C;
    return s;
}
// element offset of the segment's first row at the lane's channel, and the step to the next row
__device__ __forceinline__ int64_t first_at(const Segment &s, int C, int reverse) {
    return (reverse ? s.t.start + s.t.n - 1 - s.first : s.t.start + s.first) * C + s.c;
}

// A lane's two decays: -softplus, and whether the warp has a wide one.
template <int VEC>
__device__ __forceinline__ uint64_t rates(const float *__restrict__ decay, const Segment &s, bool &wide) {
    const float r0 = s.on ? softplus(decay[s.c]) : 0.0f, r1 = s.on && VEC == 2 ? softplus(decay[s.c + 1]) : 0.0f;
    wide = __any_sync(0xffffffffu, fmaxf(r0, r1) > 1.4f);
    return pack2(-r0, -r1);
}

// f(full, wide) with both as types, for a block with n rows left: a whole one runs without a branch between its rows, so that the chains of
// special functions of different rows overlap (with a test of each row's number, (3) took 222 us instead of 174 at
// 8 x 131072 x 64 bf16).
template <typename F>
__device__ __forceinline__ void by_length(int n, bool wide, F f) {
    if (n >= kBlock) {
        if (wide)
            f(std::true_type{}, std::true_type{});
        else
            f(std::true_type{}, std::false_type{});
    } else if (n > 0) {
        f(std::false_type{}, std::true_type{});
    }
}

// maps [slots][kWarps + 1][C] of (A, H): the segments', then the CTA's; slot and channel-block outermost
struct Maps {
    float2 *at;
    int C;
    __device__ __forceinline__ float2 *of(int64_t slot, int w, int c) const {
        return at + (slot * (kWarps + 1) + w) * C + c;
    }
};

template <int VEC>
__device__ __forceinline__ void put_map(float2 *p, uint64_t A, uint64_t H) {
    if (VEC == 2)
        *reinterpret_cast<float4 *>(p) = make_float4(lo(A), lo(H), hi(A), hi(H));
    else
        *p = make_float2(lo(A), lo(H));
}
template <int VEC>
__device__ __forceinline__ void get_map(const float2 *p, uint64_t &A, uint64_t &H) {
    if (VEC == 2) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        A = pack2(v.x, v.z);
        H = pack2(v.y, v.w);
    } else {
        A = pack2(p->x, 1.0f);
        H = pack2(p->y, 0.0f);
    }
}

// (1) BACK = false: (A, H) of each segment and CTA, h_out = A h_in + H. BACK = true: the same for c, which runs
// against the rows: c_out = a (dh + c_in). `in` is x, or dh (nullable: 0).
template <typename T, int VEC, bool BACK, int NB>
__global__ void __launch_bounds__(kScanThreads, sizeof(T) == 2 ? 4 : 2)
    scan_fold_kernel(const T *__restrict__ in, const T *__restrict__ gate, const float *__restrict__ decay,
                     const int64_t *__restrict__ ptr, int B, int64_t n_rows, int C, int reverse, Maps maps) {
    __shared__ float4 part[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Segment s = segment<VEC, NB>(ptr, B, n_rows, C);
    if (s.t.cloud < 0) return;
    bool wide;
    const uint64_t nrate = rates<VEC>(decay, s, wide);
    const int64_t at0 = first_at(s, C, reverse);
    const int step = reverse ? -C : C;
    const T *gp = gate + at0, *vp = in + at0;
    uint64_t A = both(1.0f), H = 0;
#pragma unroll 1
    for (int k = 0; k < NB; ++k) {
        const int r0 = (BACK ? NB - 1 - k : k) * kBlock;
        by_length(s.n - r0, wide, [&](auto full, auto is_wide) {
            Raw<T, VEC> gs[kBlock], vs[kBlock];
            const T *g0 = gp + r0 * step, *v0 = vp + r0 * step;
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
                if (s.on && (full.value || r0 + i < s.n)) {
                    gs[i].load(g0 + i * step);
                    if (!BACK || in) vs[i].load(v0 + i * step);
                }
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                const int i = BACK ? kBlock - 1 - j : j;
                if (!full.value && r0 + i >= s.n) continue;
                const Gate g = scan_gate<!BACK, is_wide.value>(gs[i].wide(), nrate);
                H = BACK ? mul2(g.a, add2(H, vs[i].wide())) : fma2(g.a, H, mul2(g.b, vs[i].wide()));
                A = mul2(A, g.a);
            }
        });
    }
    if (s.on) put_map<VEC>(maps.of(blockIdx.x, warp, s.c), A, H);
    if (s.t.n <= scan_rows(NB)) return;  // (a cloud of one CTA is not chained)
    part[warp][lane] = make_float4(lo(A), hi(A), lo(H), hi(H));
    __syncthreads();
    if (warp == 0 && s.on) {
        A = both(1.0f);
        H = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float4 p = part[BACK ? kWarps - 1 - k : k][lane];
            H = fma2(pack2(p.x, p.y), H, pack2(p.z, p.w));
            A = mul2(pack2(p.x, p.y), A);
        }
        put_map<VEC>(maps.of(blockIdx.x, kWarps, s.c), A, H);
    }
}

// (2) Per cloud and channel: the state before (BACK: the gradient c after) each CTA's rows, carry[slot][C].
// A warp folds a run of CTAs, the runs are chained, and each warp goes over its run again.
template <bool BACK, int NB>
__global__ void __launch_bounds__(32 * kChainWarps)
    scan_chain_kernel(const int64_t *__restrict__ ptr, int B, int64_t n_rows, int C, const float *__restrict__ init,
                      Maps maps, float *__restrict__ carry, float *__restrict__ empty_out) {
    __shared__ float2 run[kChainWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x, c = blockIdx.y * 32 + lane;
    const int64_t start = ragged_bound(ptr, B, n_rows, b + 1), end = ragged_bound(ptr, B, n_rows, b + 2);
    const int64_t n = end > start ? end - start : 0;
    const bool on = c < C;
    const float h0 = on && init ? init[(int64_t)b * C + c] : 0.0f;
    if (n == 0) {
        if (on && warp == 0 && empty_out) empty_out[(int64_t)b * C + c] = h0;
        return;
    }
    const int64_t slot0 = start / scan_rows(NB) + b + 1, slots = (n + scan_rows(NB) - 1) / scan_rows(NB);
    const int64_t per = (slots + kChainWarps - 1) / kChainWarps;
    const int64_t k0 = warp * per, k1 = k0 + per < slots ? k0 + per : slots;
    float A = 1.0f, H = 0.0f;
    if (slots > 1 && on) {
#pragma unroll 8
        for (int64_t k = k0; k < k1; ++k) {
            const float2 m = *maps.of(slot0 + (BACK ? slots - 1 - k : k), kWarps, c);
            H = fmaf(m.x, H, m.y);
            A *= m.x;
        }
    }
    run[warp][lane] = make_float2(A, H);
    __syncthreads();
    if (!on) return;
    float h = h0;
    for (int w = 0; w < warp; ++w) h = fmaf(run[w][lane].x, h, run[w][lane].y);
#pragma unroll 8
    for (int64_t k = k0; k < k1; ++k) {
        const int64_t slot = slot0 + (BACK ? slots - 1 - k : k);
        carry[slot * C + c] = h;
        if (k + 1 < k1) {
            const float2 m = *maps.of(slot, kWarps, c);
            h = fmaf(m.x, h, m.y);
        }
    }
}

// The state at this warp's segment from the CTA's: over the segments before it (BACK: behind it)
template <int VEC, bool BACK>
__device__ __forceinline__ uint64_t segment_carry(const Segment &s, Maps maps, const float *__restrict__ carry, int C,
                                                  int own) {
    const int warp = threadIdx.x >> 5;
    const float *p = carry + (int64_t)blockIdx.x * C + s.c;
    uint64_t h = VEC == 2 ? pack2(p[0], p[1]) : pack2(p[0], 0.0f);
    for (int w = BACK ? own - 1 : 0; BACK ? w > warp : w < warp; w += BACK ? -1 : 1) {
        uint64_t A, H;
        get_map<VEC>(maps.of(blockIdx.x, w, s.c), A, H);
        h = fma2(A, h, H);
    }
    return h;
}

// (3) h from each segment's state
template <typename T, int VEC, int NB>
__global__ void __launch_bounds__(kScanThreads, sizeof(T) == 2 ? 4 : 2)
    scan_write_kernel(const T *__restrict__ x, const T *__restrict__ gate, const float *__restrict__ decay,
                      const int64_t *__restrict__ ptr, int B, int64_t n_rows, int C, int reverse, Maps maps,
                      const float *__restrict__ carry, T *__restrict__ h, float *__restrict__ last,
                      float *__restrict__ states) {
    const int warp = threadIdx.x >> 5;
    const Segment s = segment<VEC, NB>(ptr, B, n_rows, C);
    if (s.t.cloud == -2) return;
    if (s.t.cloud == -1) {
        for (int i = 0; i < s.n && s.on; ++i) store2<VEC>(h + (s.t.start + s.first + i) * C + s.c, 0);
        return;
    }
    bool wide;
    const uint64_t nrate = rates<VEC>(decay, s, wide);
    const int64_t at0 = first_at(s, C, reverse);
    const int step = reverse ? -C : C;
    const T *gp = gate + at0, *xp = x + at0;
    T *out = h + at0;
    if (!s.on || s.n == 0) return;
    uint64_t v = segment_carry<VEC, false>(s, maps, carry, C, kWarps);
#pragma unroll 1
    for (int r0 = 0; r0 < s.n; r0 += kBlock) {
        if (states) store2<VEC>(states + (((int64_t)blockIdx.x * kWarps + warp) * NB + r0 / kBlock) * C + s.c, v);
        by_length(s.n - r0, wide, [&](auto full, auto is_wide) {
            Raw<T, VEC> gs[kBlock], xs[kBlock];
            const T *g0 = gp + r0 * step, *x0 = xp + r0 * step;
            T *o0 = out + r0 * step;
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
                if (full.value || r0 + i < s.n) {
                    gs[i].load(g0 + i * step);
                    xs[i].load(x0 + i * step);
                }
#pragma unroll
            for (int i = 0; i < kBlock; ++i) {
                if (!full.value && r0 + i >= s.n) continue;
                const Gate g = scan_gate<true, is_wide.value>(gs[i].wide(), nrate);
                v = fma2(g.a, v, mul2(g.b, xs[i].wide()));
                store2<VEC>(o0 + i * step, v);
            }
        });
    }
    if (last && s.first + s.n == s.t.n) store2<VEC>(last + (int64_t)s.t.cloud * C + s.c, v);
}

// (3) backward: h from the segment's state forwards, c from its carry backwards. part [slots * kWarps][C]: the
// segment's sum of dl sigmoid.
template <typename T, int VEC, int NB>
__global__ void __launch_bounds__(kScanThreads, sizeof(T) == 2 ? 2 : 1)
    scan_write_back_kernel(const T *__restrict__ x, const T *__restrict__ gate, const float *__restrict__ decay,
                           const int64_t *__restrict__ ptr, int B, int64_t n_rows, int C, int reverse, Maps maps,
                           const float *__restrict__ carry, const float *__restrict__ states,
                           const T *__restrict__ dh, T *__restrict__ dx, T *__restrict__ dgate,
                           float *__restrict__ dh0, float *__restrict__ sums) {
    __shared__ float4 part[kWarps][32];
    extern __shared__ uint64_t kept[];  // [3][kBlock][kScanThreads]: each thread's sigmoids, b and states before its rows
    const int warp = threadIdx.x >> 5;
    const Segment s = segment<VEC, NB>(ptr, B, n_rows, C);
    uint64_t *sig = kept + threadIdx.x, *hp = sig + kBlock * kScanThreads,
             *bs = hp + kBlock * kScanThreads;
    float *sum_at = sums + (int64_t)blockIdx.x * C + s.c;
    if (s.t.cloud < 0) {
        if (s.on && warp == 0) store2<VEC>(sum_at, 0);
        if (s.t.cloud == -1)
            for (int i = 0; i < s.n && s.on; ++i) {
                store2<VEC>(dx + (s.t.start + s.first + i) * C + s.c, 0);
                store2<VEC>(dgate + (s.t.start + s.first + i) * C + s.c, 0);
            }
        return;
    }
    bool wide;
    const uint64_t nrate = rates<VEC>(decay, s, wide);
    const int64_t at0 = first_at(s, C, reverse);
    const int step = reverse ? -C : C;
    const T *gp = gate + at0, *xp = x + at0, *dp = dh + at0;
    T *ox = dx + at0, *og = dgate + at0;
    uint64_t c = 0, sum = 0;
    if (s.on && s.n > 0) {
        const int own = (int)((s.t.n - s.t.first + kBlock * NB - 1) / (kBlock * NB));
        c = segment_carry<VEC, true>(s, maps, carry, C, own < kWarps ? own : kWarps);
    }
#pragma unroll 1
    for (int r0 = (s.n - 1) / kBlock * kBlock; r0 >= 0 && s.n > 0; r0 -= kBlock) {
        uint64_t v = 0;
        if (s.on) {
            const float *p = states + (((int64_t)blockIdx.x * kWarps + warp) * NB + r0 / kBlock) * C + s.c;
            v = VEC == 2 ? pack2(p[0], p[1]) : pack2(p[0], 0.0f);
        }
        Raw<T, VEC> xs[kBlock], ds[kBlock];
        uint64_t a[kBlock];
        by_length(s.n - r0, wide, [&](auto full, auto is_wide) {
            Raw<T, VEC> gs[kBlock];
            const T *g0 = gp + r0 * step, *x0 = xp + r0 * step, *d0 = dp + r0 * step;
#pragma unroll
            for (int i = 0; i < kBlock; ++i)
                if (s.on && (full.value || r0 + i < s.n)) {
                    gs[i].load(g0 + i * step);
                    xs[i].load(x0 + i * step);
                    if (dh) ds[i].load(d0 + i * step);
                }
#pragma unroll
            for (int i = 0; i < kBlock; ++i) {
                if (!full.value && r0 + i >= s.n) continue;
                const Gate g = scan_gate<true, is_wide.value>(gs[i].wide(), nrate);
                sig[i * kScanThreads] = g.sig;
                a[i] = g.a;
                bs[i * kScanThreads] = g.b;
                hp[i * kScanThreads] = v;
                v = fma2(g.a, v, mul2(g.b, xs[i].wide()));
            }
        });
        by_length(s.n - r0, false, [&](auto full, auto) {
            T *oxi = ox + (r0 + kBlock - 1) * step, *ogi = og + (r0 + kBlock - 1) * step;
#pragma unroll
            for (int k = 0; k < kBlock; ++k, oxi -= step, ogi -= step) {
                const int i = kBlock - 1 - k;
                if (!full.value && r0 + i >= s.n) continue;
                const uint64_t g = add2(ds[i].wide(), c);
                c = mul2(a[i], g);
                // x a / b: 0 where the gate is so far shut that b = 0
                const uint64_t b = bs[i * kScanThreads];
                const float b0 = lo(b) > 0.0f ? rcp(lo(b)) : 0.0f, b1 = hi(b) > 0.0f ? rcp(hi(b)) : 0.0f;
                const uint64_t t = mul2(xs[i].wide(), mul2(a[i], pack2(-b0, -b1)));
                const uint64_t dl = mul2(c, add2(hp[i * kScanThreads], t)), sg = sig[i * kScanThreads];
                const uint64_t ds1 = mul2(dl, sg);
                sum = add2(sum, ds1);
                // dl l (1 - sig), with l = nrate sig
                if (s.on) {
                    store2<VEC>(oxi, mul2(b, g));
                    store2<VEC>(ogi, mul2(mul2(ds1, nrate), fma2(sg, both(-1.0f), both(1.0f))));
                }
            }
        });
    }
    if (dh0 && s.on && s.first == 0 && s.n > 0) store2<VEC>(dh0 + (int64_t)s.t.cloud * C + s.c, c);
    part[warp][threadIdx.x & 31] = make_float4(lo(sum), hi(sum), 0.0f, 0.0f);
    __syncthreads();
    if (warp == 0 && s.on) {
        sum = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum = add2(sum, pack2(part[w][threadIdx.x].x, part[w][threadIdx.x].y));
        store2<VEC>(sum_at, sum);
    }
}

// ddecay[c] from the slots' sums, in two launches of a fixed order: runs of slots, then the runs
constexpr int kDecayRuns = 64;
__global__ void __launch_bounds__(256) scan_decay_runs_kernel(const float *__restrict__ sums, int64_t slots, int C,
                                                              float *__restrict__ runs) {
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.y * 32 + lane;
    const int64_t per = (slots + kDecayRuns - 1) / kDecayRuns;
    const int64_t k0 = blockIdx.x * per, k1 = k0 + per < slots ? k0 + per : slots;
    float s = 0.0f;
    if (c < C)
#pragma unroll 4
        for (int64_t k = k0 + warp; k < k1; k += 8) s += sums[k * C + c];
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < C) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += part[w][lane];
        runs[(int64_t)blockIdx.x * C + c] = s;
    }
}
__global__ void __launch_bounds__(256) scan_decay_kernel(const float *__restrict__ part, const float *__restrict__ decay,
                                                         int64_t rows, int C, float *__restrict__ ddecay) {
    __shared__ float sums[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < C)
#pragma unroll 8
        for (int64_t r = warp; r < rows; r += 8) s += part[r * C + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < C) {
        s = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += sums[w][lane];
        ddecay[c] = -s * rcp(1.0f + expf(-decay[c]));
    }
}

// ---------------------------------------------------------------------------------------- few rows
template <typename T>
__global__ void scan_serial_kernel(const T *__restrict__ x, const T *__restrict__ gate,
                                   const float *__restrict__ decay, const int64_t *__restrict__ ptr, int B,
                                   int64_t n_rows, int C, const float *__restrict__ h0, int reverse, T *__restrict__ h,
                                   float *__restrict__ last, float *__restrict__ states) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    const int b = (int)blockIdx.y - 1;  // -1 and B: the rows of no cloud
    if (c >= C) return;
    const int64_t start = ragged_bound(ptr, B, n_rows, b + 1), end = ragged_bound(ptr, B, n_rows, b + 2);
    const int64_t n = end > start ? end - start : 0;
    if (b < 0 || b >= B) {
        for (int64_t t = 0; t < n; ++t) store1(h + (start + t) * C + c, 0.0f);
        return;
    }
    const float rate = softplus(decay[c]);
    float s = h0 ? h0[(int64_t)b * C + c] : 0.0f;
    constexpr int rows = scan_rows(2);  // (few rows: always the smaller segments)
    const int64_t slot0 = start / rows + b + 1;
    for (int64_t t = 0; t < n; ++t) {
        if (states && t % kBlock == 0)
            states[((slot0 + t / rows) * (rows / kBlock) + t % rows / kBlock) * C + c] = s;
        const int64_t at = (reverse ? end - 1 - t : start + t) * C + c;
        const Gate g = scan_gate<true, true>(pack2(load1(gate + at), 0.0f), pack2(-rate, 0.0f));
        s = fmaf(lo(g.a), s, lo(g.b) * load1(x + at));
        store1(h + at, s);
    }
    if (last) last[(int64_t)b * C + c] = s;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Blocks to a warp's segment: 4 where that still makes two waves of CTAs (8 x 131072 x 64: 446 instead of 488 us,
// less of each warp's fixed work), else 2 (16 x 2048 x 64 f32: 38 instead of 52 us, more CTAs).
int scan_blocks(int64_t n_rows, int32_t C) {
    return n_rows / scan_rows(4) * ((C + 63) / 64) >= 2 * 4 * kSmCount ? 4 : 2;
}

// workspace: the maps, the carries, the sums of the decay's gradient and its runs
struct ScanSpace {
    size_t maps, carry, sums, runs, total;
};
ScanSpace scan_space(int64_t n_rows, int32_t B, int32_t C, bool back) {
    const size_t slots = (size_t)ragged_slots(n_rows, B, scan_rows(scan_blocks(n_rows, C)));
    ScanSpace s;
    s.maps = 0;
    s.carry = align256(slots * (kWarps + 1) * C * sizeof(float2));
    s.sums = s.carry + align256(slots * C * 4);
    s.runs = s.sums + (back ? align256(slots * C * 4) : 0);
    s.total = s.runs + (back ? align256((size_t)kDecayRuns * C * 4) : 0) + 256;
    return s;
}

template <typename T, int VEC, int NB>
int forward_in(const T *x, const T *gate, const float *decay, const int64_t *ptr, int B, int64_t n_rows, int C,
                 const float *h0, int reverse, T *h, float *last, float *states, char *ws, cudaStream_t st) {
    const ScanSpace sp = scan_space(n_rows, B, C, false);
    const Maps maps = {(float2 *)(ws + sp.maps), C};
    float *carry = (float *)(ws + sp.carry);
    const dim3 grid((unsigned)ragged_slots(n_rows, B, scan_rows(NB)), (C + 32 * VEC - 1) / (32 * VEC));
    scan_fold_kernel<T, VEC, false, NB><<<grid, kScanThreads, 0, st>>>(x, gate, decay, ptr, B, n_rows, C, reverse, maps);
    if (B > 0)
        scan_chain_kernel<false, NB><<<dim3(B, (C + 31) / 32), 32 * kChainWarps, 0, st>>>(ptr, B, n_rows, C, h0, maps, carry,
                                                                                    last);
    scan_write_kernel<T, VEC, NB><<<grid, kScanThreads, 0, st>>>(x, gate, decay, ptr, B, n_rows, C, reverse, maps, carry, h,
                                                             last, states);
    GDL_CUDA_TRY(cudaGetLastError());
    return GDL_OK;
}

template <typename T, int VEC, int NB>
int backward_in(const T *x, const T *gate, const float *decay, const int64_t *ptr, int B, int64_t n_rows, int C,
                  const float *states, int reverse, const T *dh, const float *dlast, T *dx, T *dgate, float *ddecay,
                  float *dh0, char *ws, cudaStream_t st) {
    const ScanSpace sp = scan_space(n_rows, B, C, true);
    const Maps maps = {(float2 *)(ws + sp.maps), C};
    float *carry = (float *)(ws + sp.carry), *sums = (float *)(ws + sp.sums), *runs = (float *)(ws + sp.runs);
    const int64_t slots = ragged_slots(n_rows, B, scan_rows(NB));
    const dim3 grid((unsigned)slots, (C + 32 * VEC - 1) / (32 * VEC));
    scan_fold_kernel<T, VEC, true, NB><<<grid, kScanThreads, 0, st>>>(dh, gate, decay, ptr, B, n_rows, C, reverse, maps);
    if (B > 0)
        scan_chain_kernel<true, NB><<<dim3(B, (C + 31) / 32), 32 * kChainWarps, 0, st>>>(ptr, B, n_rows, C, dlast, maps,
                                                                                   carry, dh0);
    const int kept = 3 * kBlock * kScanThreads * (int)sizeof(uint64_t);
    GDL_CUDA_TRY(cudaFuncSetAttribute(scan_write_back_kernel<T, VEC, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kept));
    scan_write_back_kernel<T, VEC, NB><<<grid, kScanThreads, kept, st>>>(x, gate, decay, ptr, B, n_rows, C, reverse, maps, carry,
                                                                  states, dh, dx, dgate, dh0, sums);
    if (slots > 8 * kDecayRuns) {
        scan_decay_runs_kernel<<<dim3(kDecayRuns, (C + 31) / 32), 256, 0, st>>>(sums, slots, C, runs);
        scan_decay_kernel<<<(C + 31) / 32, 256, 0, st>>>(runs, decay, kDecayRuns, C, ddecay);
    } else {
        scan_decay_kernel<<<(C + 31) / 32, 256, 0, st>>>(sums, decay, slots, C, ddecay);
    }
    GDL_CUDA_TRY(cudaGetLastError());
    return GDL_OK;
}

template <typename T, int VEC, typename... A>
int scan_forward(const T *x, const T *gate, const float *decay, const int64_t *ptr, int B, int64_t n_rows, int C, A... rest) {
    return scan_blocks(n_rows, C) == 4 ? forward_in<T, VEC, 4>(x, gate, decay, ptr, B, n_rows, C, rest...)
                                       : forward_in<T, VEC, 2>(x, gate, decay, ptr, B, n_rows, C, rest...);
}
template <typename T, int VEC, typename... A>
int scan_backward(const T *x, const T *gate, const float *decay, const int64_t *ptr, int B, int64_t n_rows, int C, A... rest) {
    return scan_blocks(n_rows, C) == 4 ? backward_in<T, VEC, 4>(x, gate, decay, ptr, B, n_rows, C, rest...)
                                       : backward_in<T, VEC, 2>(x, gate, decay, ptr, B, n_rows, C, rest...);
}

int scan_check(int32_t dtype, const float *decay, const int64_t *ptr, int32_t B, int64_t n_rows, int32_t C) {
    GDL_RETURN_IF(B < 0 || n_rows < 0 || C < 0, GDL_ERR_INVALID);
    GDL_RETURN_IF(dtype != GDL_DTYPE_F32 && dtype != GDL_DTYPE_BF16, GDL_ERR_INVALID);
    if (C == 0) return GDL_OK;
    GDL_RETURN_IF(!decay || !ptr, GDL_ERR_INVALID);
    GDL_RETURN_IF(ragged_slots(n_rows, B, scan_rows(2)) > ((int64_t)1 << 31) - 1 || C > 32 * 65535, GDL_ERR_OVERFLOW);
    return GDL_OK;
}

// pairs of channels can be read at once: an even number of them, and aligned tensors
bool in_pairs(int32_t C, int32_t dtype, uintptr_t all) { return C % 2 == 0 && all % (dtype == GDL_DTYPE_F32 ? 8 : 4) == 0; }

}  // namespace
}  // namespace gdl

using namespace gdl;

extern "C" size_t gdl_gated_scan_states_size(int64_t n_rows, int32_t num_clouds, int32_t channels) {
    if (n_rows < 0 || num_clouds < 0 || channels < 0) return 0;
    const int rows = scan_rows(scan_blocks(n_rows, channels));
    return (size_t)ragged_slots(n_rows, num_clouds, rows) * (rows / kBlock) * channels;
}

extern "C" size_t gdl_gated_scan_workspace_size(int64_t n_rows, int32_t num_clouds, int32_t channels) {
    if (n_rows < 0 || num_clouds < 0 || channels < 0 || takes_serial(n_rows, num_clouds)) return 256;
    return scan_space(n_rows, num_clouds, channels, false).total;
}

extern "C" size_t gdl_gated_scan_backward_workspace_size(int64_t n_rows, int32_t num_clouds, int32_t channels) {
    if (n_rows < 0 || num_clouds < 0 || channels < 0) return 256;
    return scan_space(n_rows, num_clouds, channels, true).total;
}

extern "C" int gdl_gated_scan(const void *x, const void *gate, int32_t dtype, const float *decay, const int64_t *ptr,
                              int32_t num_clouds, int64_t n_rows, int32_t channels, const float *h0, int32_t reverse,
                              void *h, float *last, float *states, void *workspace, size_t workspace_bytes,
                              void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    const int rc = scan_check(dtype, decay, ptr, num_clouds, n_rows, channels);
    if (rc != GDL_OK || channels == 0) return rc;
    GDL_RETURN_IF(n_rows > 0 && (!x || !gate || !h), GDL_ERR_INVALID);
    const int C = channels, B = num_clouds;
    if (takes_serial(n_rows, B)) {
        const dim3 grid((C + kScanThreads - 1) / kScanThreads, B + 2);
        if (dtype == GDL_DTYPE_F32)
            scan_serial_kernel<float><<<grid, kScanThreads, 0, st>>>((const float *)x, (const float *)gate, decay, ptr, B,
                                                                     n_rows, C, h0, reverse, (float *)h, last, states);
        else
            scan_serial_kernel<uint16_t><<<grid, kScanThreads, 0, st>>>((const uint16_t *)x, (const uint16_t *)gate,
                                                                        decay, ptr, B, n_rows, C, h0, reverse,
                                                                        (uint16_t *)h, last, states);
        GDL_CUDA_TRY(cudaGetLastError());
        return GDL_OK;
    }
    GDL_RETURN_IF(!workspace || workspace_bytes < scan_space(n_rows, B, C, false).total, GDL_ERR_WORKSPACE);
    char *ws = (char *)workspace;
    const bool two = in_pairs(C, dtype, (uintptr_t)x | (uintptr_t)gate | (uintptr_t)h) &&
                     in_pairs(C, GDL_DTYPE_F32, (uintptr_t)last | (uintptr_t)states);
    if (dtype == GDL_DTYPE_F32) {
        const float *xf = (const float *)x, *gf = (const float *)gate;
        return two ? scan_forward<float, 2>(xf, gf, decay, ptr, B, n_rows, C, h0, reverse, (float *)h, last, states, ws, st)
                   : scan_forward<float, 1>(xf, gf, decay, ptr, B, n_rows, C, h0, reverse, (float *)h, last, states, ws, st);
    }
    const uint16_t *xb = (const uint16_t *)x, *gb = (const uint16_t *)gate;
    return two ? scan_forward<uint16_t, 2>(xb, gb, decay, ptr, B, n_rows, C, h0, reverse, (uint16_t *)h, last, states, ws, st)
               : scan_forward<uint16_t, 1>(xb, gb, decay, ptr, B, n_rows, C, h0, reverse, (uint16_t *)h, last, states, ws, st);
}

extern "C" int gdl_gated_scan_backward(const void *x, const void *gate, int32_t dtype, const float *decay,
                                       const int64_t *ptr, int32_t num_clouds, int64_t n_rows, int32_t channels,
                                       const float *states, int32_t reverse, const void *grad_h,
                                       const float *grad_last, void *dx, void *dgate, float *ddecay, float *dh0,
                                       void *workspace, size_t workspace_bytes, void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    const int rc = scan_check(dtype, decay, ptr, num_clouds, n_rows, channels);
    if (rc != GDL_OK || channels == 0) return rc;
    GDL_RETURN_IF(!ddecay, GDL_ERR_INVALID);
    GDL_RETURN_IF(n_rows > 0 && (!x || !gate || !states || !dx || !dgate), GDL_ERR_INVALID);
    const int C = channels, B = num_clouds;
    GDL_RETURN_IF(!workspace || workspace_bytes < scan_space(n_rows, B, C, true).total, GDL_ERR_WORKSPACE);
    char *ws = (char *)workspace;
    const bool two = in_pairs(C, dtype, (uintptr_t)x | (uintptr_t)gate | (uintptr_t)grad_h | (uintptr_t)dx | (uintptr_t)dgate) &&
                     in_pairs(C, GDL_DTYPE_F32, (uintptr_t)dh0 | (uintptr_t)states);
    if (dtype == GDL_DTYPE_F32) {
        const float *xf = (const float *)x, *gf = (const float *)gate, *df = (const float *)grad_h;
        float *ox = (float *)dx, *og = (float *)dgate;
        return two ? scan_backward<float, 2>(xf, gf, decay, ptr, B, n_rows, C, states, reverse, df, grad_last, ox, og, ddecay, dh0, ws, st)
                   : scan_backward<float, 1>(xf, gf, decay, ptr, B, n_rows, C, states, reverse, df, grad_last, ox, og, ddecay, dh0, ws, st);
    }
    const uint16_t *xb = (const uint16_t *)x, *gb = (const uint16_t *)gate, *db = (const uint16_t *)grad_h;
    uint16_t *ox = (uint16_t *)dx, *og = (uint16_t *)dgate;
    return two ? scan_backward<uint16_t, 2>(xb, gb, decay, ptr, B, n_rows, C, states, reverse, db, grad_last, ox, og, ddecay, dh0, ws, st)
               : scan_backward<uint16_t, 1>(xb, gb, decay, ptr, B, n_rows, C, states, reverse, db, grad_last, ox, og, ddecay, dh0, ws, st);
}
