// gdn_norm.cu -- the root-mean-square norms on either side of a recurrent
// layer, with an e4m3 output for an 8-bit product behind them.
//
//   add_norm:   r = x + residual,  y = r / sqrt(mean(r^2) + eps) * weight      (over a row)
//   gated_norm: y = x / sqrt(mean(x^2) + eps) * weight * z sigmoid(z)          (over a head)
// With n = r / rms and u = dy * weight (* gate):
//   dr = u / rms - n mean(u n) / rms (+ d_new_residual),  dweight = sum dy n (* gate),
//   dz = dy n weight (sig + z sig (1 - sig)).
// e4m3: scale = max(amax |y|, 1e-12) / 448 over a row, or over 128 channels;
// the code is e4m3 of the fp32 quotient y / scale by the stored scale.  The norm is of
// the fp32 sum; new_residual is that sum rounded to the inputs' type.
//
// All of it is one pass over the data: a row (or head) stays in registers
// between its statistics and its output.  8 elements per thread and load
// (one 16-byte vector of a 16-bit type), arithmetic on packed fp32 pairs.
// HBM-bound.  Into outputs kept between calls, 65536 x 4096 bf16 with a residual
// takes 311 us (6.9 TB/s; the rate of a copy is 6.6), to e4m3 by rows 299 us (6.3;
// 316 to 330 into outputs that each call allocates), by groups 312 us (6.0);
// backward 323 us (6.6); 32768 tokens of 32 heads of 128 gated 128 us (6.3), to
// e4m3 135 us (5.0), backward 222 us (6.0).
#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

namespace gdn {

constexpr float kFp8Max = 448.0f;
constexpr float kAmaxMin = 1e-12f;  // an all-zero row keeps a finite scale
constexpr int kQuantGroup = 128;    // channels per scale in group mode: 16 threads of 8
constexpr int kNormStages = 3;  // rows in flight per CTA (backward)
constexpr int kNormThreads = 512, kNormWarps = 32;  // up to 1024 threads in the backward kernel's narrow form

struct NormParams {
    const void* x;
    const void* residual;  // NULL: y is the norm of x
    int64_t x_stride, residual_stride;
    const void* weight;
    bool weight_f32;
    int mode;   // kApart, kVec or kShift
    int quant;  // 0 none, 1 a scale per row, 2 a scale per 128 channels
    int64_t rows;
    int width;
    float eps;
    void* out;
    void* new_residual;
    float* scale;
    int stages;  // backward: rows in flight in shared memory
};

struct NormGradParams {
    const void* dy;
    const void* dr;  // NULL: zero
    int64_t dy_stride, dr_stride;
    void* dx;
    float* part;  // [CTAs, width] partial dweight
};

struct GatedNormParams {
    const void* x;
    const void* z;
    int64_t x_stride, z_stride;  // elements between tokens; the heads of one token are contiguous
    const void* weight;
    bool weight_f32;
    bool vec;
    bool quant;
    unsigned items;  // tokens * heads
    unsigned heads;
    float eps;
    void* out;
    float* scale;
};

struct GatedNormGradParams {
    const void* dy;
    int64_t dy_stride;
    void* dx;
    void* dz;
    float* part;
};

// 8 consecutive elements as they are stored.
template <typename T>
struct Raw8 {
    uint4 v[sizeof(T) / 2];
};
// How a row's elements are dealt to the threads, 8 at a time.
constexpr int kApart = 0;  // any alignment: blockDim.x apart, so that a warp's accesses touch neighbours
constexpr int kVec = 1;    // rows are whole 8-element vectors on 16-byte boundaries
// Rows of 16 elements or more whose width is not a multiple of 8, contiguous or
// apart by a multiple of 8 elements more: the vectors of the whole tensor, of
// which a row's first and last are only partly its own (16384 x 5333 bf16: 147
// to 154 us forward, 181 backward; dealt apart 301 and 378).
constexpr int kShift = 2;
struct Cols {
    int first, step, width;
    __device__ __forceinline__ bool in(int i) const {
        return static_cast<unsigned>(first + i * step) < static_cast<unsigned>(width);
    }
    __device__ __forceinline__ bool whole() const { return first >= 0 && first + 8 <= width; }  // step 1
    __device__ __forceinline__ bool any() const { return first < width && first + 7 * step >= 0; }
};
// A thread's j-th; `m` elements lie between the boundary and the row's start (kShift).
template <int MODE>
__device__ __forceinline__ Cols row_cols(int j, int width, bool groups, int m) {
    const int t = threadIdx.x, n = blockDim.x;
    return MODE == kShift           ? Cols{(t + j * n) * 8 - m, 1, width}
           : MODE == kVec || groups ? Cols{(t + j * n) * 8, 1, width}
                                    : Cols{j * 8 * n + t, n, width};
}

template <typename T>
__device__ __forceinline__ Raw8<T> load_vec8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
// A shifted row's first and last vectors come with their neighbours' elements,
// for own8 to drop, but for the end of the tensor's `last` row.
template <typename T, int MODE>
__device__ __forceinline__ Raw8<T> load8(const T* row, Cols c, bool last = true) {
    Raw8<T> r = {};
    if constexpr (MODE == kVec) {
        if (c.in(0)) r = load_vec8(row + c.first);
        return r;
    }
    if (MODE == kShift && !c.any()) return r;
    if (MODE == kShift && (!last || c.first + 8 <= c.width)) return load_vec8(row + c.first);
    // all loads first, from the row's start where the column is outside:
    // `row` is a row of the tensor even where none of the columns counts
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = row[c.in(i) ? c.first + i * c.step : 0];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c.in(i) ? e[i] : from_f32<T>(0.0f);
    memcpy(&r, e, sizeof(r));
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, F2 (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = load_pair<T>(reinterpret_cast<const T*>(&r) + 2 * i);
}

template <int MODE>
__device__ __forceinline__ void own8(F2 (&f)[4], Cols c) {
    if (MODE == kShift && !c.whole()) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = unpack2(f[i]);
            f[i] = pack2(c.in(2 * i) ? v.x : 0.0f, c.in(2 * i + 1) ? v.y : 0.0f);
        }
    }
}

template <typename T, int MODE>
__device__ __forceinline__ void store8(T* row, Cols c, const F2 (&f)[4]) {
    Raw8<T> r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2(f[i]);
        e[2 * i] = from_f32<T>(v.x);
        e[2 * i + 1] = from_f32<T>(v.y);
    }
    if (MODE == kVec ? c.in(0) : MODE == kShift && c.whole()) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(row + c.first)[i] = r.v[i];
    } else if (MODE != kVec) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c.in(i)) row[c.first + i * c.step] = e[i];
    }
}

// The scale of values up to amax, and its reciprocal in two words: y over the
// scale is y (inv + rest), the fp32 quotient, where y inv alone is off by a
// unit or two and at a tie of two codes gives the other one.  (One multiply more:
// 65536 x 4096 bf16 to e4m3 by rows 299 us, 294 without.)  An infinite amax has no
// second word: finite values over it are 0, infinite ones NaN.
struct Scale {
    float scale, inv, rest;
    __device__ __forceinline__ explicit Scale(float amax) : scale(amax / kFp8Max), inv(kFp8Max / amax) {
        rest = amax <= 3.402823466e38f ? fmaf(-inv, scale, 1.0f) * inv : 0.0f;
    }
    __device__ __forceinline__ F2 quotient(F2 y) const { return fma2(y, splat2(inv), mul2(y, splat2(rest))); }
};
template <int MODE>
__device__ __forceinline__ void store8_e4m3(uint8_t* row, Cols c, const F2 (&f)[4], Scale by) {
    uint2 u;
    uint16_t* h = reinterpret_cast<uint16_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(unpack2(by.quotient(f[i])), __NV_SATFINITE, __NV_E4M3);
    if (MODE == kVec ? c.in(0) : MODE == kShift && c.whole()) {
        *reinterpret_cast<uint2*>(row + c.first) = u;
    } else if (MODE != kVec) {
        const uint8_t* e = reinterpret_cast<const uint8_t*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c.in(i)) row[c.first + i * c.step] = e[i];
    }
}

// Weights of a shifted row are off the boundary: an inner vector's come from two
// neighbouring vectors of w, moved by the row's m (element by element, 16384 x
// 5333 takes 10 us longer forward).
template <typename W>
__device__ __forceinline__ bool load_shifted8(const W* w, Cols c, F2 (&f)[4]) {
    const int m = -c.first & 7, at = c.first + m;  // elements at - m .. at - m + 7
    if (at < 8 || at + 8 > c.width || (reinterpret_cast<uintptr_t>(w) & 15) != 0) return false;
    F2 lo[4], hi[4];
    unpack8(load_vec8(w + at - 8), lo);
    unpack8(load_vec8(w + at), hi);
    float e[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2(lo[i]), b = unpack2(hi[i]);
        e[2 * i] = a.x, e[2 * i + 1] = a.y;
        e[8 + 2 * i] = b.x, e[9 + 2 * i] = b.y;
    }
    const int by = 8 - m;  // the result is e[by .. by + 7]
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {
#pragma unroll
        for (int i = 0; i < 16 - k; ++i)
            if (i < 7 + k) e[i] = by & k ? e[i + k] : e[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pack2(e[2 * i], e[2 * i + 1]);
    return true;
}
template <typename T, int MODE>
__device__ __forceinline__ void load_weight8(const void* w, bool f32, Cols c, F2 (&f)[4]) {
    if (MODE == kShift && (f32 ? load_shifted8(static_cast<const float*>(w), c, f) : load_shifted8(static_cast<const T*>(w), c, f)))
        return;
    if (f32)
        unpack8(load8<float, MODE == kVec ? kVec : kApart>(static_cast<const float*>(w), c), f);
    else
        unpack8(load8<T, MODE == kVec ? kVec : kApart>(static_cast<const T*>(w), c), f);
}

// Maxima keep a NaN (fmaxf drops it): a row that holds one gets a NaN scale.
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = max_keep_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float abs_max8(const F2 (&y)[4], float m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2(y[i]);
        m = max_keep_nan(m, max_keep_nan(fabsf(v.x), fabsf(v.y)));
    }
    return m;
}
__device__ __forceinline__ float sum2(F2 v) {
    const float2 f = unpack2(v);
    return f.x + f.y;
}

// Sum (or maximum) over a row's blockDim.x threads, in the same order on every
// run: lanes by xor-shuffle, then the row's warps in order.  Every thread of
// the CTA calls it; `red` is used by one call only.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
    v = MAX ? lanes_max<32>(v) : lanes_sum<32>(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    float* r = red + threadIdx.y * warps;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = r[0];
#pragma unroll 4
    for (int w = 1; w < warps; ++w) v = MAX ? max_keep_nan(v, r[w]) : v + r[w];
    return v;
}
// Sums of a and b over a warp, in five shuffles: the halves take one sum each.
// Lanes 0 and 16 hold them.
__device__ __forceinline__ float lanes_sum_pair(float a, float b) {
    const bool upper = threadIdx.x & 16;
    float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// blockDim = (threads per row, rows per CTA), 8 VPT elements of a row per thread.
template <typename T, int VPT, int MODE>
__global__ void __launch_bounds__(kNormThreads) gdn_add_norm_kernel(const NormParams p) {
    __shared__ float red_sum[kNormWarps], red_max[kNormWarps];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool live = row < p.rows;
    const int width = live ? p.width : 0;
    const T* x = static_cast<const T*>(p.x) + (live ? row * p.x_stride : 0);
    const T* res = static_cast<const T*>(p.residual) + (live && p.residual ? row * p.residual_stride : 0);
    const int64_t out = row * p.width;
    const bool groups = p.quant == 2;
    const int m = MODE == kShift ? static_cast<int>(out & 7) : 0;
    Raw8<T> rx[VPT], rr[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        rx[j] = load8<T, MODE>(x, row_cols<MODE>(j, width, groups, m), row >= p.rows - 1);
        if (p.residual) rr[j] = load8<T, MODE>(res, row_cols<MODE>(j, width, groups, m), row >= p.rows - 1);
    }
    F2 r[VPT][4], ss = splat2(0.0f);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        unpack8(rx[j], r[j]);
        if (p.residual) {
            F2 f[4];
            unpack8(rr[j], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) r[j][i] = add2(r[j][i], f[i]);
        }
        own8<MODE>(r[j], row_cols<MODE>(j, width, groups, m));
        if (p.residual) {
            store8<T, MODE>(static_cast<T*>(p.new_residual) + out, row_cols<MODE>(j, width, groups, m), r[j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fma2(r[j][i], r[j][i], ss);
    }
    const float rstd = rsqrtf(row_reduce<false>(sum2(ss), red_sum) / static_cast<float>(p.width) + p.eps);
    float amax8 = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const Cols c = row_cols<MODE>(j, width, groups, m);
        F2 w[4];
        load_weight8<T, MODE>(p.weight, p.weight_f32, c, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[j][i] = mul2(mul2(r[j][i], splat2(rstd)), w[i]);
        if (p.quant == 0) {
            store8<T, MODE>(static_cast<T*>(p.out) + out, c, r[j]);
        } else if (groups) {  // 16 threads hold a group's 128 channels
            const Scale by(lanes_max<16>(c.in(0) ? abs_max8(r[j], kAmaxMin) : kAmaxMin));
            store8_e4m3<MODE>(static_cast<uint8_t*>(p.out) + out, c, r[j], by);
            if (c.in(0) && (threadIdx.x & 15) == 0)
                p.scale[row * (p.width / kQuantGroup) + c.first / kQuantGroup] = by.scale;
        } else if (c.any()) {
            amax8 = abs_max8(r[j], amax8);
        }
    }
    if (p.quant == 1) {
        const Scale by(max_keep_nan(row_reduce<true>(amax8, red_max), kAmaxMin));
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            store8_e4m3<MODE>(static_cast<uint8_t*>(p.out) + out, row_cols<MODE>(j, width, false, m), r[j], by);
        if (width > 0 && threadIdx.x == 0) p.scale[row] = by.scale;
    }
}

// blockDim = (threads per row, 1); CTA k takes rows k, k + gridDim.x, ... and
// keeps its share of dweight in registers.  With p.stages > 0 the rows of x, dy
// and dr arrive in shared memory by bulk copies, p.stages rows ahead of use
// (without them a row's loads would wait for the row before it).
template <typename T, int VPT, int MODE>
__global__ void __launch_bounds__(VPT == 1 ? 1024 : kNormThreads) gdn_add_norm_backward_kernel(const NormParams p, const NormGradParams d) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float red[2][2][kNormWarps];
    __shared__ __align__(8) uint64_t s_bar[kNormStages];
    // kShift: gridDim.x is a multiple of 8 where a CTA has several rows
    const int m = MODE == kShift ? static_cast<int>(static_cast<int64_t>(blockIdx.x) * p.width & 7) : 0;
    F2 dw[VPT][4], w[VPT][4];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        load_weight8<T, MODE>(p.weight, p.weight_f32, row_cols<MODE>(j, p.width, false, m), w[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[j][i] = splat2(0.0f);
    }
    // A shifted row is copied with what its first and last vectors hold of its
    // neighbours, which the last row has only on one side: its end is read directly.
    const int slot = (m + p.width + 7) / 8 * 8, slot_max = (MODE == kShift ? p.width + 14 : p.width) / 8 * 8;
    const uint32_t bar = tc05::smem_u32(s_bar);
    auto fetch = [&](int64_t row, int stage) {  // by one thread
        if (row >= p.rows) return;
        const uint32_t to = tc05::smem_u32(smem) + stage * 3 * slot_max * sizeof(T), next = slot_max * sizeof(T);
        const uint32_t bytes = (MODE == kShift && row == p.rows - 1 ? (m + p.width) / 8 * 8 : slot) * sizeof(T);
        tc05::mbar_expect_tx(bar + 8 * stage, bytes * (d.dr ? 3 : 2));
        tc05::bulk_g2s(to, static_cast<const T*>(p.x) + row * p.x_stride - m, bytes, bar + 8 * stage);
        tc05::bulk_g2s(to + next, static_cast<const T*>(d.dy) + row * d.dy_stride - m, bytes, bar + 8 * stage);
        if (d.dr) tc05::bulk_g2s(to + 2 * next, static_cast<const T*>(d.dr) + row * d.dr_stride - m, bytes, bar + 8 * stage);
    };
    if (p.stages > 0 && threadIdx.x == 0) {
        for (int i = 0; i < p.stages; ++i) tc05::mbar_init(bar + 8 * i, 1);
        tc05::fence_mbar_init();
        for (int i = 0; i < p.stages; ++i) fetch(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, i);
    }
    if (p.stages > 0) __syncthreads();
    const float inv_width = 1.0f / static_cast<float>(p.width);
    int turn = 0, stage = 0, phase = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
        const T* dy = static_cast<const T*>(d.dy) + row * d.dy_stride;
        const T* dr = static_cast<const T*>(d.dr) + (d.dr ? row * d.dr_stride : 0);
        const T *ex = x, *edy = dy, *edr = dr;  // for the end of the last row
        if (MODE != kApart && p.stages > 0) {
            if (!tc05::mbar_wait(bar + 8 * stage, phase)) {
                // the copies under way land (bounded again) before the shared memory goes
                for (int i = 0; i < p.stages && row + static_cast<int64_t>(i) * gridDim.x < p.rows; ++i) {
                    const int at = (stage + i) % p.stages;
                    tc05::mbar_wait(bar + 8 * at, phase ^ (at < stage));
                }
                return record_status(32 /* GDN_ERR_DEVICE_TIMEOUT */);
            }
            x = reinterpret_cast<const T*>(smem) + stage * 3 * slot_max + m;
            dy = x + slot_max;
            dr = dy + slot_max;
        }
        F2 r[VPT][4], g[VPT][4], o[VPT][4], ss2 = splat2(0.0f), dot2 = splat2(0.0f);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const Cols c = row_cols<MODE>(j, p.width, false, m);
            const bool last = row == p.rows - 1, end = MODE == kShift && last && c.first + 8 > p.width;
            unpack8(load8<T, MODE>(end ? ex : x, c, last), r[j]);
            unpack8(load8<T, MODE>(end ? edy : dy, c, last), g[j]);
            own8<MODE>(r[j], c);
            own8<MODE>(g[j], c);
            if (d.dr) {
                unpack8(load8<T, MODE>(end ? edr : dr, c, last), o[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][i] = splat2(0.0f);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ss2 = fma2(r[j][i], r[j][i], ss2);
                dot2 = fma2(mul2(g[j][i], w[j][i]), r[j][i], dot2);
            }
        }
        // both sums in one exchange; the buffers alternate, so a fast warp's
        // next row cannot overwrite what a slow warp still reads
        const float both = lanes_sum_pair(sum2(ss2), sum2(dot2));
        const int warps = blockDim.x >> 5;
        if ((threadIdx.x & 15) == 0) red[turn][threadIdx.x >> 4 & 1][threadIdx.x >> 5] = both;
        __syncthreads();
        if (MODE != kApart && p.stages > 0) {  // every thread has its part of the row: the stage takes another
            if (threadIdx.x == 0) fetch(row + static_cast<int64_t>(p.stages) * gridDim.x, stage);
            stage = stage + 1 == p.stages ? 0 : stage + 1;
            phase ^= stage == 0;
        }
        float ss = 0.0f, dot = 0.0f;
        for (int k = 0; k < warps; k += 16) {  // 16 warps' sums of each kind, added by the two halves of a warp
            const int i = k + (threadIdx.x & 15);
            float v = i < warps ? red[turn][threadIdx.x >> 4 & 1][i] : 0.0f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            ss += __shfl_sync(0xffffffffu, v, 0);
            dot += __shfl_sync(0xffffffffu, v, 16);
        }
        const float rstd = rsqrtf(ss * inv_width + p.eps);
        const F2 rstd2 = splat2(rstd), back = splat2(-dot * rstd * rstd * rstd * inv_width);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dw[j][i] = fma2(g[j][i], mul2(r[j][i], rstd2), dw[j][i]);
                o[j][i] = add2(o[j][i], fma2(mul2(g[j][i], w[j][i]), rstd2, mul2(r[j][i], back)));
            }
            store8<T, MODE>(static_cast<T*>(d.dx) + row * p.width, row_cols<MODE>(j, p.width, false, m), o[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j)
        store8<float, MODE == kVec ? kVec : kApart>(d.part + static_cast<int64_t>(blockIdx.x) * p.width, row_cols<MODE>(j, p.width, false, m), dw[j]);
}

// out[c] = sum of part[.][c], in a fixed order.  blockDim = (32, 32).
__global__ void __launch_bounds__(1024) gdn_sum_columns_kernel(const float* part, int rows, int width, float* out) {
    __shared__ float red[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (int i = threadIdx.y; i < rows; i += 32) s += part[static_cast<int64_t>(i) * width + c];
    }
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = lanes_sum<32>(red[threadIdx.x][threadIdx.y]);
    if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < width) out[blockIdx.x * 32 + threadIdx.y] = s;
}

// LANES = head dim / 8 threads per head; item = (token, head), kGatedItems of
// them per thread.
constexpr int kGatedItems = 2;
template <typename T, int LANES, int MODE>
__global__ void __launch_bounds__(256) gdn_gated_norm_kernel(const GatedNormParams p) {
    constexpr int kHeadDim = LANES * 8, kGroups = 256 / LANES;
    const int col = (threadIdx.x % LANES) * 8;
    Raw8<T> rx[kGatedItems], rz[kGatedItems];
    unsigned items[kGatedItems];
#pragma unroll
    for (int n = 0; n < kGatedItems; ++n) {
        items[n] = (blockIdx.x * kGatedItems + n) * kGroups + threadIdx.x / LANES;
        const unsigned item = items[n] < p.items ? items[n] : 0;
        const unsigned token = item / p.heads, head = item - token * p.heads;
        const int64_t in = static_cast<int64_t>(head) * kHeadDim + col;
        rx[n] = load8<T, MODE>(static_cast<const T*>(p.x) + token * p.x_stride + in, {0, 1, items[n] < p.items ? 8 : 0});
        rz[n] = load8<T, MODE>(static_cast<const T*>(p.z) + token * p.z_stride + in, {0, 1, items[n] < p.items ? 8 : 0});
    }
    F2 w[4];
    load_weight8<T, MODE>(p.weight, p.weight_f32, {col, 1, kHeadDim}, w);
#pragma unroll
    for (int n = 0; n < kGatedItems; ++n) {
        const unsigned item = items[n];
        const Cols all = {0, 1, item < p.items ? 8 : 0};
        const int64_t o = static_cast<int64_t>(item) * kHeadDim + col;
        F2 x[4], z[4], ss = splat2(0.0f);
        unpack8(rx[n], x);
        unpack8(rz[n], z);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fma2(x[i], x[i], ss);
        const F2 rstd = splat2(rsqrtf(lanes_sum<LANES>(sum2(ss)) * (1.0f / kHeadDim) + p.eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(mul2(x[i], rstd), w[i]), mul2(z[i], sigmoid2(z[i])));
        if (!p.quant) {
            store8<T, MODE>(static_cast<T*>(p.out) + o, all, x);
        } else {
            const Scale by(lanes_max<LANES>(abs_max8(x, kAmaxMin)));
            store8_e4m3<MODE>(static_cast<uint8_t*>(p.out) + o, all, x, by);
            if (col == 0 && item < p.items) p.scale[item] = by.scale;
        }
    }
}

// Every thread keeps the same 8 columns for all its items: dweight stays in
// registers, and the CTA's groups are added in order at the end.  The next
// item is on its way while one is worked on.
template <typename T, int LANES, int MODE>
__global__ void __launch_bounds__(256) gdn_gated_norm_backward_kernel(const GatedNormParams p,
                                                                       const GatedNormGradParams d) {
    constexpr int kHeadDim = LANES * 8, kGroups = 256 / LANES;
    __shared__ float red[kGroups][kHeadDim];
    const int group = threadIdx.x / LANES, col = (threadIdx.x % LANES) * 8;
    F2 w[4], dw[4];
    load_weight8<T, MODE>(p.weight, p.weight_f32, {col, 1, kHeadDim}, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[i] = splat2(0.0f);
    Raw8<T> rx, rz, ry;
    auto fetch = [&](int64_t first) {
        const bool live = first + group < p.items;
        const Cols all = {0, 1, live ? 8 : 0};
        const unsigned item = live ? static_cast<unsigned>(first + group) : 0;
        const unsigned token = item / p.heads, head = item - token * p.heads;
        const int64_t in = static_cast<int64_t>(head) * kHeadDim + col;
        rx = load8<T, MODE>(static_cast<const T*>(p.x) + token * p.x_stride + in, all);
        rz = load8<T, MODE>(static_cast<const T*>(p.z) + token * p.z_stride + in, all);
        ry = load8<T, MODE>(static_cast<const T*>(d.dy) + token * d.dy_stride + in, all);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
    int64_t first = static_cast<int64_t>(blockIdx.x) * kGroups;
    fetch(first);
    for (; first < p.items; first += step) {
        const int64_t item = first + group;
        F2 x[4], z[4], dy[4], sig[4], ss2 = splat2(0.0f), dot2 = splat2(0.0f);
        unpack8(rx, x);
        unpack8(rz, z);
        unpack8(ry, dy);
        fetch(first + step);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sig[i] = sigmoid2(z[i]);
            ss2 = fma2(x[i], x[i], ss2);
            dot2 = fma2(mul2(mul2(dy[i], w[i]), mul2(z[i], sig[i])), x[i], dot2);
        }
        const float ss = lanes_sum<LANES>(sum2(ss2)), dot = lanes_sum<LANES>(sum2(dot2));
        const float rstd = rsqrtf(ss * (1.0f / kHeadDim) + p.eps);
        const F2 rstd2 = splat2(rstd), back = splat2(-dot * rstd * rstd * rstd * (1.0f / kHeadDim));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const F2 gate = mul2(z[i], sig[i]), dyn = mul2(dy[i], mul2(x[i], rstd2));
            if (item < p.items) dw[i] = fma2(dyn, gate, dw[i]);
            x[i] = fma2(mul2(mul2(dy[i], w[i]), gate), rstd2, mul2(x[i], back));
            z[i] = mul2(mul2(dyn, w[i]), fma2(gate, fma2(sig[i], splat2(-1.0f), splat2(1.0f)), sig[i]));
        }
        const Cols all = {0, 1, item < p.items ? 8 : 0};
        store8<T, MODE>(static_cast<T*>(d.dx) + item * kHeadDim + col, all, x);
        store8<T, MODE>(static_cast<T*>(d.dz) + item * kHeadDim + col, all, z);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = unpack2(dw[i]);
        red[group][col + 2 * i] = v.x;
        red[group][col + 2 * i + 1] = v.y;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < kHeadDim; c += 256) {
        float s = 0.0f;
        for (int g = 0; g < kGroups; ++g) s += red[g][c];
        d.part[static_cast<int64_t>(blockIdx.x) * kHeadDim + c] = s;
    }
}

// Threads per row (a multiple of 32) and vectors of 8 elements per thread.
struct RowShape {
    int threads, vpt;
};
static RowShape row_shape(int vecs, int vpt) { return {((vecs + vpt - 1) / vpt + 31) / 32 * 32, vpt}; }
// Forward.  Two vectors per thread halve the warps that a row's sum waits for
// (32768 x 2048 bf16: 82.7 us, 93.0 with one); four where a scale per row adds
// a second wait (65536 x 1024: 78.3 us, 84.6 with two); but fp32 takes two up to
// 1024 vectors, for its occupancy (16384 x 4096 with a scale per row: 133 us, 150
// with four; 16384 x 6144: 204 and 206; shifted 16384 x 4097: 183 and 236).  Rows
// dealt apart hold twice the registers per vector, so fewer (16384 x 5333: 301 us
// with two, 483 with four).  Eight spill up to 250 bytes a thread in fp32 and
// apart (4096 x 32768 bf16: 208 us, 5.2 TB/s).
static int row_vecs(int width, int mode) { return (width + (mode == kShift ? 14 : 7)) / 8; }
static RowShape row_shape_forward(const NormParams& p, size_t elem) {
    const int vecs = row_vecs(p.width, p.mode);
    if (p.mode == kApart) return row_shape(vecs, vecs <= 512 ? 1 : vecs <= 1024 ? 2 : vecs <= 2048 ? 4 : 8);
    if (p.quant == 1 && elem == 2 && p.mode == kVec && vecs >= 128 && vecs <= 2048) return row_shape(vecs, 4);
    return row_shape(vecs, vecs <= 32 ? 1 : vecs <= (elem == 4 ? 1024 : 512) ? 2 : vecs <= 2048 ? 4 : 8);
}
constexpr int kNormMaxWidth = kNormThreads * 8 * 8;

// Calls f with the vectors per thread and whether rows are whole vectors, as constants.
template <int V>
using Int = std::integral_constant<int, V>;
template <typename F>
static void with_row_shape(int vpt, int mode, F f) {
    const auto go = [&](auto n) { mode == kVec ? f(n, Int<kVec>{}) : mode == kShift ? f(n, Int<kShift>{}) : f(n, Int<kApart>{}); };
    vpt == 1 ? go(Int<1>{}) : vpt == 2 ? go(Int<2>{}) : vpt == 4 ? go(Int<4>{}) : go(Int<8>{});
}
template <typename F>
static void with_head_shape(int head_dim, bool vec, F f) {
    const auto go = [&](auto n) { vec ? f(n, Int<kVec>{}) : f(n, Int<kApart>{}); };
    head_dim == 64 ? go(Int<8>{}) : head_dim == 128 ? go(Int<16>{}) : go(Int<32>{});
}

template <typename T>
static cudaError_t launch_add_norm(const NormParams& p, cudaStream_t s) {
    const RowShape r = row_shape_forward(p, sizeof(T));
    const int per_cta = r.threads >= 256 ? 1 : 256 / r.threads;
    const dim3 block(r.threads, per_cta);
    const unsigned grid = static_cast<unsigned>((p.rows + per_cta - 1) / per_cta);
    with_row_shape(r.vpt, p.mode, [&](auto vpt, auto mode) { gdn_add_norm_kernel<T, vpt(), mode()><<<grid, block, 0, s>>>(p); });
    return cudaGetLastError();
}

// Backward: the weight and its gradient's share are held too, so two vectors at
// most while they fit (65536 x 4096 bf16: 323 us, 407 with one on twice the
// threads, whose sums wait for twice the warps).  A vector holds 40 floats (w, dw,
// r, g, o), so the wider rows spill, with four about 1 KB a thread and with eight
// 3 to 5 KB: 16384 x 12288 bf16 578 us, where the copy rate is 245; 8192 x 16384
// 312 and 164; 4096 x 32768 1190 and 164.
static RowShape row_shape_backward(int width, int mode) {
    const int vecs = row_vecs(width, mode);
    if (mode == kApart) return row_shape(vecs, vecs <= 1024 ? 1 : vecs <= 2048 ? 4 : 8);
    return row_shape(vecs, vecs <= 32 ? 1 : vecs <= 1024 ? 2 : vecs <= 2048 ? 4 : 8);
}

static int norm_backward_ctas(int64_t rows, int width, int mode) {
    const RowShape r = row_shape_backward(width, mode);
    const int per_sm = (r.vpt == 1 ? 1024 : 512) / r.threads;  // by registers
    int64_t most = static_cast<int64_t>(kSmCount) * (per_sm < 1 ? 1 : per_sm > 8 ? 8 : per_sm);
    if (mode == kShift) most = most / 8 * 8;  // a CTA's rows all start at the same place in a vector
    return static_cast<int>(rows < most ? (rows > 0 ? rows : 1) : most);
}

static cudaError_t launch_sum_columns(const float* part, int rows, int width, float* out, cudaStream_t s) {
    gdn_sum_columns_kernel<<<(width + 31) / 32, dim3(32, 32), 0, s>>>(part, rows, width, out);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_add_norm_backward(NormParams p, const NormGradParams& d, float* dweight, cudaStream_t s) {
    const RowShape r = row_shape_backward(p.width, p.mode);
    const int grid = norm_backward_ctas(p.rows, p.width, p.mode);
    // Rows in flight for about 200 KB of an SM's shared memory over its CTAs;
    // fewer than two would not run ahead, and rows at any alignment cannot be
    // copied in bulk (65536 x 4096: 407 us, 536 without).
    constexpr int kBudget = 200 << 10;
    const int per_sm = (grid + kSmCount - 1) / kSmCount;
    const size_t stage = 3 * 8 * static_cast<size_t>(row_vecs(p.width, p.mode)) * sizeof(T);
    const int fit = static_cast<int>(kBudget / per_sm / stage);
    p.stages = p.mode == kApart || fit < 2 ? 0 : fit < kNormStages ? fit : kNormStages;
    const int smem = static_cast<int>(p.stages * stage);
    cudaError_t e = cudaSuccess;
    with_row_shape(r.vpt, p.mode, [&](auto vpt, auto mode) {
        const auto kernel = gdn_add_norm_backward_kernel<T, vpt(), mode()>;
        // The limit belongs to the kernel, not to the call: one value for all
        // widths, or another thread's call could lower it before this launch.
        if (smem > (40 << 10)) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget);
        if (e == cudaSuccess) kernel<<<grid, r.threads, smem, s>>>(p, d);
    });
    if (e == cudaSuccess) e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_sum_columns(d.part, grid, p.width, dweight, s);
}

template <typename T>
static cudaError_t launch_gated_norm(const GatedNormParams& p, int head_dim, cudaStream_t s) {
    const unsigned per_cta = kGatedItems * 256 / (head_dim / 8), grid = (p.items + per_cta - 1) / per_cta;
    with_head_shape(head_dim, p.vec, [&](auto lanes, auto vec) {
        gdn_gated_norm_kernel<T, lanes(), vec()><<<grid, 256, 0, s>>>(p);
    });
    return cudaGetLastError();
}

static int gated_norm_backward_ctas(int64_t items, int head_dim) {
    const int64_t per_cta = 256 / (head_dim / 8), want = (items + per_cta - 1) / per_cta, most = kSmCount * 8;
    return static_cast<int>(want < most ? (want > 0 ? want : 1) : most);
}

template <typename T>
static cudaError_t launch_gated_norm_backward(const GatedNormParams& p, const GatedNormGradParams& d, int head_dim,
                                              float* dweight, cudaStream_t s) {
    const int grid = gated_norm_backward_ctas(p.items, head_dim);
    with_head_shape(head_dim, p.vec, [&](auto lanes, auto vec) {
        gdn_gated_norm_backward_kernel<T, lanes(), vec()><<<grid, 256, 0, s>>>(p, d);
    });
    if (cudaError_t e = cudaGetLastError()) return e;
    return launch_sum_columns(d.part, grid, head_dim, dweight, s);
}

// Row starts on 16-byte boundaries (8 for e4m3 codes), so whole vectors can be moved.
static bool rows_vec(const void* p, int64_t stride_bytes, uintptr_t bytes = 16) {
    return p == nullptr || (aligned(p, bytes) && stride_bytes % static_cast<int64_t>(bytes) == 0);
}

// How rows of `width` elements that are `stride` apart can be read, all tensors
// alike (absent ones NULL).
struct RowsOf {
    const void* p;
    int64_t stride;
};
static int row_mode(int64_t width, uintptr_t es, std::initializer_list<RowsOf> tensors) {
    const bool shift = width >= 16 && row_vecs(static_cast<int>(width), kShift) <= kNormThreads * 8;
    int mode = width % 8 == 0 ? kVec : shift ? kShift : kApart;
    for (const RowsOf& t : tensors) {
        if (t.p == nullptr) continue;
        const bool vec = rows_vec(t.p, t.stride * static_cast<int64_t>(es)), alike = aligned(t.p, 16) && (t.stride - width) % 8 == 0;
        if (mode == kVec ? !vec : !alike) mode = kApart;
    }
    return mode;
}

static int add_norm_setup(const GdnAddNormArgs* a, NormParams& p) {
    if (a == nullptr) return GDN_ERR_NULL_POINTER;
    if (!dtype_ok(a->dtype) || (a->weight_dtype != GDN_DTYPE_F32 && a->weight_dtype != a->dtype)) return GDN_ERR_BAD_DTYPE;
    if (a->rows < 0 || a->rows > 0x7fff0000LL || a->width < 1 || a->width > kNormMaxWidth ||
        a->quant < GDN_QUANT_NONE || a->quant > GDN_QUANT_GROUP ||
        (a->quant == GDN_QUANT_GROUP && a->width % kQuantGroup != 0) || !(a->eps >= 0.0f))
        return GDN_ERR_BAD_SIZE;
    if (a->rows > 1 && (a->x_stride < a->width || (a->residual && a->residual_stride < a->width)))
        return GDN_ERR_BAD_SIZE;
    if (!a->weight || (a->rows > 0 && !a->x)) return GDN_ERR_NULL_POINTER;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(a->x, es) || !aligned(a->residual, es) || !aligned(a->new_residual, es) ||
        !aligned(a->output, a->quant ? 1 : es) || !aligned(a->weight, dtype_bytes(a->weight_dtype)) ||
        !aligned(a->scale, 4))
        return GDN_ERR_MISALIGNED;
    p.x = a->x;
    p.residual = a->residual;
    p.x_stride = a->x_stride;
    p.residual_stride = a->residual_stride;
    p.weight = a->weight;
    p.weight_f32 = a->weight_dtype == GDN_DTYPE_F32;
    p.mode = row_mode(a->width, es, {{a->x, a->x_stride}, {a->residual, a->residual_stride}, {a->new_residual, a->width}});
    if (a->quant ? !aligned(a->output, 8) : !aligned(a->output, 16)) p.mode = kApart;
    if (p.mode == kVec && !aligned(a->weight, 16)) p.mode = kApart;
    p.quant = a->quant;
    p.rows = a->rows;
    p.width = static_cast<int>(a->width);
    p.eps = a->eps;
    p.out = a->output;
    p.new_residual = a->new_residual;
    p.scale = a->scale;
    p.stages = 0;
    return GDN_OK;
}

static int gated_norm_setup(const GdnGatedNormArgs* a, GatedNormParams& p) {
    if (a == nullptr) return GDN_ERR_NULL_POINTER;
    if (!dtype_ok(a->dtype) || (a->weight_dtype != GDN_DTYPE_F32 && a->weight_dtype != a->dtype)) return GDN_ERR_BAD_DTYPE;
    if (a->tokens < 0 || a->heads < 1 || a->heads > 4096 || (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) ||
        a->tokens > 0x7fff0000LL / a->heads || (a->quant != GDN_QUANT_NONE && a->quant != GDN_QUANT_GROUP) ||
        !(a->eps >= 0.0f))
        return GDN_ERR_BAD_SIZE;
    const int64_t width = static_cast<int64_t>(a->heads) * a->head_dim;
    if (a->tokens > 1 && (a->x_stride < width || a->z_stride < width)) return GDN_ERR_BAD_SIZE;
    if (!a->weight || (a->tokens > 0 && (!a->x || !a->z))) return GDN_ERR_NULL_POINTER;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(a->x, es) || !aligned(a->z, es) || !aligned(a->output, a->quant ? 1 : es) ||
        !aligned(a->weight, dtype_bytes(a->weight_dtype)) || !aligned(a->scale, 4))
        return GDN_ERR_MISALIGNED;
    p.x = a->x;
    p.z = a->z;
    p.x_stride = a->x_stride;
    p.z_stride = a->z_stride;
    p.weight = a->weight;
    p.weight_f32 = a->weight_dtype == GDN_DTYPE_F32;
    p.vec = rows_vec(a->x, a->x_stride * es) && rows_vec(a->z, a->z_stride * es) && aligned(a->weight, 16) &&
            aligned(a->output, a->quant ? 8 : 16);
    p.quant = a->quant != GDN_QUANT_NONE;
    p.items = static_cast<unsigned>(a->tokens * a->heads);
    p.heads = static_cast<unsigned>(a->heads);
    p.eps = a->eps;
    p.out = a->output;
    p.scale = a->scale;
    return GDN_OK;
}

// What the entry points of the two norms read.
static Operands add_norm_inputs(const GdnAddNormArgs* a) {
    const int64_t es = static_cast<int64_t>(dtype_bytes(a->dtype)), row = a->width * es;
    Operands o;
    o.read(a->x, a->rows, a->x_stride * es, row);
    o.read(a->residual, a->rows, a->residual_stride * es, row);
    o.read(a->weight, 1, 0, a->width * static_cast<int64_t>(dtype_bytes(a->weight_dtype)));
    return o;
}
static Operands gated_norm_inputs(const GdnGatedNormArgs* a) {
    const int64_t es = static_cast<int64_t>(dtype_bytes(a->dtype)), row = static_cast<int64_t>(a->heads) * a->head_dim * es;
    Operands o;
    o.read(a->x, a->tokens, a->x_stride * es, row);
    o.read(a->z, a->tokens, a->z_stride * es, row);
    o.read(a->weight, 1, 0, a->head_dim * static_cast<int64_t>(dtype_bytes(a->weight_dtype)));
    return o;
}
// All that is checked of the forward call's arguments.
static int gated_norm_checked(const GdnGatedNormArgs* a, GatedNormParams& p) {
    if (int rc = gated_norm_setup(a, p)) return rc;
    if (a->tokens > 0 && (!a->output || (a->quant && !a->scale))) return GDN_ERR_NULL_POINTER;
    Operands o = gated_norm_inputs(a);
    const int64_t n = static_cast<int64_t>(a->heads) * a->head_dim, row = n * static_cast<int64_t>(dtype_bytes(a->dtype));
    if (a->quant) {
        o.write(a->output, a->tokens, n, n);
        o.write(a->scale, 1, 0, a->tokens * a->heads * 4);
    } else {
        o.write(a->output, a->tokens, row, row, true);
    }
    return o.apart() ? GDN_OK : GDN_ERR_OVERLAP;
}
}  // namespace gdn

extern "C" int gdn_add_norm_launch(const GdnAddNormArgs* a, void* stream) {
    NormParams p;
    if (int rc = add_norm_setup(a, p)) return rc;
    if (a->rows > 0 && (!a->output || (a->residual && !a->new_residual) || (a->quant && !a->scale)))
        return GDN_ERR_NULL_POINTER;
    Operands o = add_norm_inputs(a);
    const int64_t row = a->width * static_cast<int64_t>(dtype_bytes(a->dtype));
    if (a->quant) {
        o.write(a->output, a->rows, a->width, a->width);
        o.write(a->scale, 1, 0, a->rows * (a->quant == GDN_QUANT_ROW ? 1 : a->width / kQuantGroup) * 4);
    } else {
        o.write(a->output, a->rows, row, row, true);
    }
    if (a->residual) o.write(a->new_residual, a->rows, row, row, true);
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    if (a->rows == 0) return GDN_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_add_norm<float>(p, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_add_norm<__half>(p, s)
                                                      : launch_add_norm<__nv_bfloat16>(p, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" size_t gdn_add_norm_backward_workspace_size(int64_t rows, int64_t width) {
    if (rows < 0 || width < 1 || width > kNormMaxWidth) return 0;
    int most = 0;
    for (int mode : {kApart, kVec, kShift}) {
        const int n = norm_backward_ctas(rows, static_cast<int>(width), mode);
        most = n > most ? n : most;
    }
    return static_cast<size_t>(most) * width * sizeof(float);
}

extern "C" int gdn_add_norm_backward_launch(const GdnAddNormArgs* a, const GdnNormGradArgs* g, void* workspace,
                                            size_t workspace_bytes, void* stream) {
    if (g == nullptr) return GDN_ERR_NULL_POINTER;
    NormParams p;
    if (int rc = add_norm_setup(a, p)) return rc;
    if (a->quant != GDN_QUANT_NONE) return GDN_ERR_BAD_SIZE;
    if (!g->d_weight || (a->rows > 0 && (!g->d_output || !g->dx))) return GDN_ERR_NULL_POINTER;
    if (a->rows > 1 && (g->d_output_stride < a->width || (g->d_new_residual && g->d_new_residual_stride < a->width)))
        return GDN_ERR_BAD_SIZE;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(g->d_output, es) || !aligned(g->d_new_residual, es) || !aligned(g->dx, es) || !aligned(g->d_weight, 4))
        return GDN_ERR_MISALIGNED;
    if (workspace == nullptr || workspace_bytes < gdn_add_norm_backward_workspace_size(a->rows, a->width) ||
        !aligned(workspace, 16))
        return GDN_ERR_WORKSPACE;
    Operands o = add_norm_inputs(a);
    const int64_t size = static_cast<int64_t>(es), row = a->width * size;
    o.read(g->d_output, a->rows, g->d_output_stride * size, row);
    o.read(g->d_new_residual, a->rows, g->d_new_residual_stride * size, row);
    o.write(g->dx, a->rows, row, row, true);
    o.write(g->d_weight, 1, 0, a->width * 4);
    o.write(workspace, 1, 0, static_cast<int64_t>(workspace_bytes));
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    const int mode = row_mode(a->width, es, {{g->d_output, g->d_output_stride}, {g->d_new_residual, g->d_new_residual_stride},
                                             {g->dx, a->width}});
    if (mode != p.mode) p.mode = kApart;
    NormGradParams d;
    d.dy = g->d_output;
    d.dr = g->d_new_residual;
    d.dy_stride = g->d_output_stride;
    d.dr_stride = g->d_new_residual_stride;
    d.dx = g->dx;
    d.part = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_add_norm_backward<float>(p, d, g->d_weight, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_add_norm_backward<__half>(p, d, g->d_weight, s)
                                                      : launch_add_norm_backward<__nv_bfloat16>(p, d, g->d_weight, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" int gdn_gated_norm_check(const GdnGatedNormArgs* a) {
    GatedNormParams p;
    return gated_norm_checked(a, p);
}

extern "C" int gdn_gated_norm_launch(const GdnGatedNormArgs* a, void* stream) {
    GatedNormParams p;
    if (int rc = gated_norm_checked(a, p)) return rc;
    if (int rc = check_device()) return rc;
    if (a->tokens == 0) return GDN_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_gated_norm<float>(p, a->head_dim, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_gated_norm<__half>(p, a->head_dim, s)
                                                      : launch_gated_norm<__nv_bfloat16>(p, a->head_dim, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" size_t gdn_gated_norm_backward_workspace_size(int64_t tokens, int32_t heads, int32_t head_dim) {
    if (tokens < 0 || heads < 1 || head_dim < 64 || head_dim > 256) return 0;
    return static_cast<size_t>(gated_norm_backward_ctas(tokens * heads, head_dim)) * head_dim * sizeof(float);
}

extern "C" int gdn_gated_norm_backward_launch(const GdnGatedNormArgs* a, const GdnNormGradArgs* g, void* workspace,
                                              size_t workspace_bytes, void* stream) {
    if (g == nullptr) return GDN_ERR_NULL_POINTER;
    GatedNormParams p;
    if (int rc = gated_norm_setup(a, p)) return rc;
    if (a->quant != GDN_QUANT_NONE) return GDN_ERR_BAD_SIZE;
    if (!g->d_weight || (a->tokens > 0 && (!g->d_output || !g->dx || !g->dz))) return GDN_ERR_NULL_POINTER;
    const int64_t width = static_cast<int64_t>(a->heads) * a->head_dim;
    if (a->tokens > 1 && g->d_output_stride < width) return GDN_ERR_BAD_SIZE;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(g->d_output, es) || !aligned(g->dx, es) || !aligned(g->dz, es) || !aligned(g->d_weight, 4))
        return GDN_ERR_MISALIGNED;
    if (workspace == nullptr || workspace_bytes < gdn_gated_norm_backward_workspace_size(a->tokens, a->heads, a->head_dim) ||
        !aligned(workspace, 16))
        return GDN_ERR_WORKSPACE;
    Operands o = gated_norm_inputs(a);
    const int64_t size = static_cast<int64_t>(es), row = width * size;
    o.read(g->d_output, a->tokens, g->d_output_stride * size, row);
    o.write(g->dx, a->tokens, row, row, true);
    o.write(g->dz, a->tokens, row, row, true);
    o.write(g->d_weight, 1, 0, a->head_dim * 4);
    o.write(workspace, 1, 0, static_cast<int64_t>(workspace_bytes));
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->tokens == 0)  // no head to read, not even one that does not count
        return cudaMemsetAsync(g->d_weight, 0, a->head_dim * sizeof(float), s) == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
    p.vec = p.vec && rows_vec(g->d_output, g->d_output_stride * es) && aligned(g->dx, 16) && aligned(g->dz, 16);
    GatedNormGradParams d;
    d.dy = g->d_output;
    d.dy_stride = g->d_output_stride;
    d.dx = g->dx;
    d.dz = g->dz;
    d.part = static_cast<float*>(workspace);
    const cudaError_t e =
        a->dtype == GDN_DTYPE_F32   ? launch_gated_norm_backward<float>(p, d, a->head_dim, g->d_weight, s)
        : a->dtype == GDN_DTYPE_F16 ? launch_gated_norm_backward<__half>(p, d, a->head_dim, g->d_weight, s)
                                    : launch_gated_norm_backward<__nv_bfloat16>(p, d, a->head_dim, g->d_weight, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}
