// gdn_norm.cu -- the root-mean-square norms on either side of a recurrent
// layer, with an e4m3 output for an 8-bit product behind them.
//
//   add_norm:   r = x + residual,  y = r / sqrt(mean(r^2) + eps) * weight      (over a row)
//   gated_norm: y = x / sqrt(mean(x^2) + eps) * weight * z sigmoid(z)          (over a head)
// With n = r / rms and u = dy * weight (* gate):
//   dr = u / rms - n mean(u n) / rms (+ d_new_residual),  dweight = sum dy n (* gate),
//   dz = dy n weight (sig + z sig (1 - sig)).
// e4m3: scale = max(amax |y|, 1e-12) / 448 over a row, or over 128 channels;
// the code is e4m3(y / scale), rounded once from the fp32 y.  The norm is of
// the fp32 sum; new_residual is that sum rounded to the inputs' type.
//
// All of it is one pass over the data: a row (or head) stays in registers
// between its statistics and its output.  8 elements per thread and load
// (one 16-byte vector of a 16-bit type).
#include <cuda_fp8.h>

namespace gdn {

constexpr float kFp8Max = 448.0f;
constexpr float kAmaxMin = 1e-12f;  // an all-zero row keeps a finite scale
constexpr int kQuantGroup = 128;    // channels per scale in group mode: 16 threads of 8

struct NormParams {
    const void* x;
    const void* residual;  // NULL: y is the norm of x
    int64_t x_stride, residual_stride;
    const void* weight;
    bool weight_f32;
    bool vec;  // every row starts on a 16-byte boundary and is whole vectors
    int quant;  // 0 none, 1 a scale per row, 2 a scale per 128 channels
    int64_t rows;
    int width;
    float eps;
    void* out;
    void* new_residual;
    float* scale;
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

// 8 consecutive elements as floats; `left` elements are inside the row.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int left, float (&f)[8]) {
    if (vec && left >= 8) {
        if constexpr (sizeof(T) == 2) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
        } else {
            const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
            f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = v.x, f[5] = v.y, f[6] = v.z, f[7] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? to_f32(p[i]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int left, const float (&f)[8]) {
    if (vec && left >= 8) {
        if constexpr (sizeof(T) == 2) {
            uint4 u;
            T* e = reinterpret_cast<T*>(&u);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
            *reinterpret_cast<uint4*>(p) = u;
        } else {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = from_f32<T>(f[i]);
    }
}

__device__ __forceinline__ void store8_e4m3(uint8_t* p, bool vec, int left, const float (&f)[8], float inv) {
    uint2 u;
    uint16_t* h = reinterpret_cast<uint16_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] * inv, f[2 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    if (vec && left >= 8) {
        *reinterpret_cast<uint2*>(p) = u;
    } else {
        const uint8_t* e = reinterpret_cast<const uint8_t*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = e[i];
    }
}

template <typename T>
__device__ __forceinline__ void load_weight8(const void* w, bool f32, int col, bool vec, int left, float (&f)[8]) {
    if (f32)
        load8(static_cast<const float*>(w) + col, vec, left, f);
    else
        load8(static_cast<const T*>(w) + col, vec, left, f);
}

// A maximum that keeps a NaN (fmaxf drops it): a row that holds one gets a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }

template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
    float m = fabsf(y[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(y[i]));
    return m;
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
    for (int w = 1; w < warps; ++w) v = MAX ? max_nan(v, r[w]) : v + r[w];
    return v;
}

// blockDim = (threads per row, rows per CTA); thread i holds the row's
// vectors i, i + blockDim.x, ...
template <typename T, int VPT>
__global__ void __launch_bounds__(1024) gdn_add_norm_kernel(const NormParams p) {
    __shared__ float red_sum[32], red_max[32];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool live = row < p.rows;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* res = static_cast<const T*>(p.residual) + row * p.residual_stride;
    float r[VPT][8];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int col = (threadIdx.x + j * blockDim.x) * 8;
        const int left = live ? p.width - col : 0;
        load8(x + col, p.vec, left, r[j]);
    }
    if (p.residual) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int col = (threadIdx.x + j * blockDim.x) * 8;
            const int left = live ? p.width - col : 0;
            float f[8];
            load8(res + col, p.vec, left, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] += f[i];
            store8(static_cast<T*>(p.new_residual) + row * p.width + col, p.vec, left, r[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(r[j][i], r[j][i], ss);
    ss = row_reduce<false>(ss, red_sum);
    const float rstd = rsqrtf(ss / static_cast<float>(p.width) + p.eps);
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int col = (threadIdx.x + j * blockDim.x) * 8;
        const int left = live ? p.width - col : 0;
        float w[8];
        load_weight8<T>(p.weight, p.weight_f32, col, p.vec, left, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[j][i] *= rstd * w[i];
        if (p.quant == 0) {
            store8(static_cast<T*>(p.out) + row * p.width + col, p.vec, left, r[j]);
        } else if (p.quant == 2) {  // 16 threads hold a group's 128 channels
            const float amax = max_nan(lanes_max<16>(left > 0 ? abs_max8(r[j]) : 0.0f), kAmaxMin);
            if (left > 0) {
                store8_e4m3(static_cast<uint8_t*>(p.out) + row * p.width + col, p.vec, left, r[j], kFp8Max / amax);
                if ((threadIdx.x & 15) == 0) p.scale[row * (p.width / kQuantGroup) + col / kQuantGroup] = amax / kFp8Max;
            }
        } else if (left > 0) {
            m = max_nan(m, abs_max8(r[j]));
        }
    }
    if (p.quant == 1) {
        const float amax = max_nan(row_reduce<true>(m, red_max), kAmaxMin);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int col = (threadIdx.x + j * blockDim.x) * 8;
            const int left = live ? p.width - col : 0;
            store8_e4m3(static_cast<uint8_t*>(p.out) + row * p.width + col, p.vec, left, r[j], kFp8Max / amax);
        }
        if (live && threadIdx.x == 0) p.scale[row] = amax / kFp8Max;
    }
}

// blockDim = (threads per row, 1); CTA k takes rows k, k + gridDim.x, ... and
// keeps its share of dweight in registers.
template <typename T, int VPT>
__global__ void __launch_bounds__(1024) gdn_add_norm_backward_kernel(const NormParams p, const NormGradParams d) {
    __shared__ float red[2][2][32];
    float dw[VPT][8], w[VPT][8];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int col = (threadIdx.x + j * blockDim.x) * 8;
        load_weight8<T>(p.weight, p.weight_f32, col, p.vec, p.width - col, w[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] = 0.0f;
    }
    const float inv_width = 1.0f / static_cast<float>(p.width);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
        const T* dy = static_cast<const T*>(d.dy) + row * d.dy_stride;
        float r[VPT][8], g[VPT][8];
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int col = (threadIdx.x + j * blockDim.x) * 8;
            load8(x + col, p.vec, p.width - col, r[j]);
            load8(dy + col, p.vec, p.width - col, g[j]);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ss = fmaf(r[j][i], r[j][i], ss);
                dot = fmaf(g[j][i] * w[j][i], r[j][i], dot);
            }
        // both sums in one exchange; the buffers alternate, so a fast warp's
        // next row cannot overwrite what a slow warp still reads
        ss = lanes_sum<32>(ss);
        dot = lanes_sum<32>(dot);
        const int warps = blockDim.x >> 5;
        if (warps > 1) {
            if ((threadIdx.x & 31) == 0) red[turn][0][threadIdx.x >> 5] = ss, red[turn][1][threadIdx.x >> 5] = dot;
            __syncthreads();
            ss = dot = 0.0f;
            for (int k = 0; k < warps; ++k) ss += red[turn][0][k], dot += red[turn][1][k];
        }
        const float rstd = rsqrtf(ss * inv_width + p.eps);
        const float back = dot * rstd * rstd * rstd * inv_width;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int col = (threadIdx.x + j * blockDim.x) * 8;
            const int left = p.width - col;
            float o[8];
            if (d.dr) {
                load8(static_cast<const T*>(d.dr) + row * d.dr_stride + col, p.vec, left, o);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dw[j][i] = fmaf(g[j][i], r[j][i] * rstd, dw[j][i]);
                o[i] += fmaf(g[j][i] * w[j][i], rstd, -r[j][i] * back);
            }
            store8(static_cast<T*>(d.dx) + row * p.width + col, p.vec, left, o);
        }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int col = (threadIdx.x + j * blockDim.x) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < p.width) d.part[static_cast<int64_t>(blockIdx.x) * p.width + col + i] = dw[j][i];
    }
}

// out[c] = sum of part[.][c], in a fixed order.  blockDim = (32, 32).
__global__ void __launch_bounds__(1024) gdn_sum_columns_kernel(const float* part, int rows, int width, float* out) {
    __shared__ float red[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < width)
        for (int i = threadIdx.y; i < rows; i += 32) s += part[static_cast<int64_t>(i) * width + c];
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = lanes_sum<32>(red[threadIdx.x][threadIdx.y]);
    if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < width) out[blockIdx.x * 32 + threadIdx.y] = s;
}

__device__ __forceinline__ float sigmoid_f(float z) { return 1.0f / (1.0f + __expf(-z)); }

// LANES = head dim / 8 threads per head; item = (token, head).
template <typename T, int LANES>
__global__ void __launch_bounds__(256) gdn_gated_norm_kernel(const GatedNormParams p) {
    constexpr int kHeadDim = LANES * 8;
    const unsigned item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const int col = (threadIdx.x % LANES) * 8;
    const int left = item < p.items ? 8 : 0;
    const unsigned token = item / p.heads, head = item - token * p.heads;
    const int64_t in = static_cast<int64_t>(head) * kHeadDim + col, o = static_cast<int64_t>(item) * kHeadDim + col;
    float x[8], z[8], w[8];
    load8(static_cast<const T*>(p.x) + token * p.x_stride + in, p.vec, left, x);
    load8(static_cast<const T*>(p.z) + token * p.z_stride + in, p.vec, left, z);
    load_weight8<T>(p.weight, p.weight_f32, col, p.vec, 8, w);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    const float rstd = rsqrtf(lanes_sum<LANES>(ss) * (1.0f / kHeadDim) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * rstd * w[i] * (z[i] * sigmoid_f(z[i]));
    if (!p.quant) {
        store8(static_cast<T*>(p.out) + o, p.vec, left, x);
        return;
    }
    const float amax = max_nan(lanes_max<LANES>(abs_max8(x)), kAmaxMin);
    store8_e4m3(static_cast<uint8_t*>(p.out) + o, p.vec, left, x, kFp8Max / amax);
    if (col == 0 && left) p.scale[item] = amax / kFp8Max;
}

// Every thread keeps the same 8 columns for all its items: dweight stays in
// registers, and the CTA's groups are added in order at the end.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) gdn_gated_norm_backward_kernel(const GatedNormParams p,
                                                                       const GatedNormGradParams d) {
    constexpr int kHeadDim = LANES * 8, kGroups = 256 / LANES;
    __shared__ float red[kGroups][kHeadDim];
    const int group = threadIdx.x / LANES, col = (threadIdx.x % LANES) * 8;
    float w[8], dw[8] = {};
    load_weight8<T>(p.weight, p.weight_f32, col, p.vec, 8, w);
    for (unsigned first = blockIdx.x * kGroups; first < p.items; first += gridDim.x * kGroups) {
        const unsigned item = first + group;
        const int left = item < p.items ? 8 : 0;
        const unsigned token = item / p.heads, head = item - token * p.heads;
        const int64_t in = static_cast<int64_t>(head) * kHeadDim + col, o = static_cast<int64_t>(item) * kHeadDim + col;
        float x[8], z[8], dy[8];
        load8(static_cast<const T*>(p.x) + token * p.x_stride + in, p.vec, left, x);
        load8(static_cast<const T*>(p.z) + token * p.z_stride + in, p.vec, left, z);
        load8(static_cast<const T*>(d.dy) + token * d.dy_stride + in, p.vec, left, dy);
        float ss = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ss = fmaf(x[i], x[i], ss);
            const float sig = sigmoid_f(z[i]);
            dot = fmaf(dy[i] * w[i] * (z[i] * sig), x[i], dot);
        }
        ss = lanes_sum<LANES>(ss);
        dot = lanes_sum<LANES>(dot);
        const float rstd = rsqrtf(ss * (1.0f / kHeadDim) + p.eps);
        const float back = dot * rstd * rstd * rstd * (1.0f / kHeadDim);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sig = sigmoid_f(z[i]), gate = z[i] * sig, n = x[i] * rstd, dyn = dy[i] * n;
            if (left) dw[i] = fmaf(dyn, gate, dw[i]);
            x[i] = fmaf(dy[i] * w[i] * gate, rstd, -x[i] * back);
            z[i] = dyn * w[i] * (sig + gate * (1.0f - sig));
        }
        store8(static_cast<T*>(d.dx) + o, p.vec, left, x);
        store8(static_cast<T*>(d.dz) + o, p.vec, left, z);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) red[group][col + i] = dw[i];
    __syncthreads();
    for (int c = threadIdx.x; c < kHeadDim; c += 256) {
        float s = 0.0f;
        for (int g = 0; g < kGroups; ++g) s += red[g][c];
        d.part[static_cast<int64_t>(blockIdx.x) * kHeadDim + c] = s;
    }
}

// Threads per row (a multiple of 32) and vectors per thread for a width.
struct RowShape {
    int threads, vpt;
};
static RowShape row_shape(int width) {
    const int vecs = (width + 7) / 8;
    int vpt = 1;
    while ((vecs + vpt - 1) / vpt > (vpt == 4 ? 1024 : 256) && vpt < 4) vpt *= 2;
    int threads = (vecs + vpt - 1) / vpt;
    threads = (threads + 31) / 32 * 32;
    return {threads, vpt};
}
constexpr int kNormMaxWidth = 1024 * 8 * 4;

template <typename T>
static cudaError_t launch_add_norm(const NormParams& p, cudaStream_t s) {
    const RowShape r = row_shape(p.width);
    const int per_cta = r.threads >= 256 ? 1 : 256 / r.threads;
    const dim3 block(r.threads, per_cta);
    const unsigned grid = static_cast<unsigned>((p.rows + per_cta - 1) / per_cta);
    if (r.vpt == 1)
        gdn_add_norm_kernel<T, 1><<<grid, block, 0, s>>>(p);
    else if (r.vpt == 2)
        gdn_add_norm_kernel<T, 2><<<grid, block, 0, s>>>(p);
    else
        gdn_add_norm_kernel<T, 4><<<grid, block, 0, s>>>(p);
    return cudaGetLastError();
}

static int norm_backward_ctas(int64_t rows, int width) {
    const RowShape r = row_shape(width);
    const int per_sm = 1024 / r.threads < 1 ? 1 : 1024 / r.threads > 8 ? 8 : 1024 / r.threads;
    const int64_t most = static_cast<int64_t>(kSmCount) * per_sm;
    return static_cast<int>(rows < most ? (rows > 0 ? rows : 1) : most);
}

static cudaError_t launch_sum_columns(const float* part, int rows, int width, float* out, cudaStream_t s) {
    gdn_sum_columns_kernel<<<(width + 31) / 32, dim3(32, 32), 0, s>>>(part, rows, width, out);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_add_norm_backward(const NormParams& p, const NormGradParams& d, float* dweight, cudaStream_t s) {
    const RowShape r = row_shape(p.width);
    const int grid = norm_backward_ctas(p.rows, p.width);
    if (r.vpt == 1)
        gdn_add_norm_backward_kernel<T, 1><<<grid, r.threads, 0, s>>>(p, d);
    else if (r.vpt == 2)
        gdn_add_norm_backward_kernel<T, 2><<<grid, r.threads, 0, s>>>(p, d);
    else
        gdn_add_norm_backward_kernel<T, 4><<<grid, r.threads, 0, s>>>(p, d);
    if (cudaError_t e = cudaGetLastError()) return e;
    return launch_sum_columns(d.part, grid, p.width, dweight, s);
}

template <typename T>
static cudaError_t launch_gated_norm(const GatedNormParams& p, int head_dim, cudaStream_t s) {
    const unsigned per_cta = 256 / (head_dim / 8), grid = (p.items + per_cta - 1) / per_cta;
    if (head_dim == 64)
        gdn_gated_norm_kernel<T, 8><<<grid, 256, 0, s>>>(p);
    else if (head_dim == 128)
        gdn_gated_norm_kernel<T, 16><<<grid, 256, 0, s>>>(p);
    else
        gdn_gated_norm_kernel<T, 32><<<grid, 256, 0, s>>>(p);
    return cudaGetLastError();
}

static int gated_norm_backward_ctas(int64_t items, int head_dim) {
    const int64_t per_cta = 256 / (head_dim / 8), want = (items + per_cta - 1) / per_cta, most = kSmCount * 4;
    return static_cast<int>(want < most ? (want > 0 ? want : 1) : most);
}

template <typename T>
static cudaError_t launch_gated_norm_backward(const GatedNormParams& p, const GatedNormGradParams& d, int head_dim,
                                              float* dweight, cudaStream_t s) {
    const int grid = gated_norm_backward_ctas(p.items, head_dim);
    if (head_dim == 64)
        gdn_gated_norm_backward_kernel<T, 8><<<grid, 256, 0, s>>>(p, d);
    else if (head_dim == 128)
        gdn_gated_norm_backward_kernel<T, 16><<<grid, 256, 0, s>>>(p, d);
    else
        gdn_gated_norm_backward_kernel<T, 32><<<grid, 256, 0, s>>>(p, d);
    if (cudaError_t e = cudaGetLastError()) return e;
    return launch_sum_columns(d.part, grid, head_dim, dweight, s);
}

// Row starts on 16-byte boundaries (8 for e4m3 codes), so whole vectors can be moved.
static bool rows_vec(const void* p, int64_t stride_bytes, uintptr_t bytes = 16) {
    return p == nullptr || (aligned(p, bytes) && stride_bytes % static_cast<int64_t>(bytes) == 0);
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
    const int64_t row = a->width * static_cast<int64_t>(es);
    p.x = a->x;
    p.residual = a->residual;
    p.x_stride = a->x_stride;
    p.residual_stride = a->residual_stride;
    p.weight = a->weight;
    p.weight_f32 = a->weight_dtype == GDN_DTYPE_F32;
    p.vec = a->width % 8 == 0 && rows_vec(a->x, a->x_stride * es) && rows_vec(a->residual, a->residual_stride * es) &&
            rows_vec(a->new_residual, row) && aligned(a->weight, 16) &&
            (a->quant ? aligned(a->output, 8) : rows_vec(a->output, row));
    p.quant = a->quant;
    p.rows = a->rows;
    p.width = static_cast<int>(a->width);
    p.eps = a->eps;
    p.out = a->output;
    p.new_residual = a->new_residual;
    p.scale = a->scale;
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
}  // namespace gdn

extern "C" int gdn_add_norm_launch(const GdnAddNormArgs* a, void* stream) {
    NormParams p;
    if (int rc = add_norm_setup(a, p)) return rc;
    if (a->rows > 0 && (!a->output || (a->residual && !a->new_residual) || (a->quant && !a->scale)))
        return GDN_ERR_NULL_POINTER;
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
    return static_cast<size_t>(norm_backward_ctas(rows, static_cast<int>(width))) * width * sizeof(float);
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
    if (int rc = check_device()) return rc;
    p.vec = p.vec && rows_vec(g->d_output, g->d_output_stride * es) &&
            rows_vec(g->d_new_residual, g->d_new_residual_stride * es) && rows_vec(g->dx, a->width * es);
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

extern "C" int gdn_gated_norm_launch(const GdnGatedNormArgs* a, void* stream) {
    GatedNormParams p;
    if (int rc = gated_norm_setup(a, p)) return rc;
    if (a->tokens > 0 && (!a->output || (a->quant && !a->scale))) return GDN_ERR_NULL_POINTER;
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
    if (int rc = check_device()) return rc;
    p.vec = p.vec && rows_vec(g->d_output, g->d_output_stride * es) && aligned(g->dx, 16) && aligned(g->dz, 16);
    GatedNormGradParams d;
    d.dy = g->d_output;
    d.dy_stride = g->d_output_stride;
    d.dx = g->dx;
    d.dz = g->dz;
    d.part = static_cast<float*>(workspace);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e =
        a->dtype == GDN_DTYPE_F32   ? launch_gated_norm_backward<float>(p, d, a->head_dim, g->d_weight, s)
        : a->dtype == GDN_DTYPE_F16 ? launch_gated_norm_backward<__half>(p, d, a->head_dim, g->d_weight, s)
                                    : launch_gated_norm_backward<__nv_bfloat16>(p, d, a->head_dim, g->d_weight, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}
