// gdn_recurrence.cu -- the per-channel gated linear recurrence: packed scan,
// its backward pass, and the decode step.
//
// Per channel c, with the gates of the delta-rule kernels:
//   z_t = a_t + dt_bias,  g_t = exp(-exp(A_log) softplus(z_t)),  beta_t = sigmoid(b_t)
//   h_t = g_t h_{t-1} + beta_t x_t,   y_t = h_t,   h before a sequence = its state row
// Backward, with e_t the gradient that reaches h_{t-1}:
//   G_t = dy_t + e_{t+1}  (e past a sequence's end = d_new_state),  e_t = g_t G_t
//   dx = G beta,  db = G x beta (1 - beta),  dl_t = G_t g_t h_{t-1}  (l = log g)
//   da = -dl exp(A_log) sigmoid(z),  dA_log = sum dl l,  d_dt_bias = sum da,
//   d_state = e at the sequence's first token.
// State, gates, sums and gradients are held in fp32; y and dx, da, db are
// rounded once, when they are stored.
#include <cuda_fp16.h>

#include "gdn_common.cuh"

namespace gdn {

// --------------------------------------------------- element type helpers --
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The carry into every kScanCkpt-th packed token is kept for the backward
// pass, which recomputes the states between two of them.
constexpr int kScanCkpt = 128;

struct ScanParams {
    const void* x;
    const void* a;
    const void* b;
    int64_t x_stride, a_stride, b_stride, out_stride;  // elements between tokens
    const float* A_log;
    const float* dt_bias;
    const float* state;  // NULL: zero
    const void* cu;
    bool cu_is_int64;
    int64_t tokens, seqs;
    int channels;
    void* out;
    float* new_state;
    float* ckpt;  // NULL: not wanted
};

struct ScanGradParams {
    const void* dy;
    int64_t dy_stride, dx_stride, da_stride, db_stride;
    const float* d_new_state;  // NULL: zero
    void* dx;
    void* da;
    void* db;
    float* d_state;  // NULL: not wanted
    float* dA_part;  // per-sequence partial sums [seqs, channels], then dA_log, ddt_bias
    float* dt_part;
    float* dA_log;
    float* ddt_bias;
};

__device__ __forceinline__ int64_t scan_cu(const ScanParams& p, int64_t n) {
    return p.cu_is_int64 ? static_cast<const int64_t*>(p.cu)[n] : static_cast<const int32_t*>(p.cu)[n];
}

__device__ __forceinline__ bool scan_bounds(const ScanParams& p, int64_t n, int64_t& t0, int64_t& t1) {
    t0 = scan_cu(p, n);
    t1 = scan_cu(p, n + 1);
    if (t0 < 0 || t1 < t0 || t1 > p.tokens) {
        record_status(16 /* GDN_ERR_DEVICE_BAD_SEQLENS */);
        t0 = t1 = 0;
        return false;
    }
    return true;
}

struct Gates {
    float l, g, beta, z;
};
__device__ __forceinline__ Gates scan_gates(float rate, float dt_bias, float a, float b) {
    Gates r;
    r.z = a + dt_bias;
    r.l = -rate * (fmaxf(r.z, 0.0f) + log1pf(expf(-fabsf(r.z))));
    r.g = expf(r.l);
    r.beta = 1.0f / (1.0f + expf(-b));
    return r;
}

// Simple form: one thread per (sequence, channel), token by token.
template <typename T>
__global__ void __launch_bounds__(128) gdn_scan_kernel(const ScanParams p) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.channels) return;
    const float rate = expf(p.A_log[c]), dtb = p.dt_bias[c];
    for (int64_t n = blockIdx.y; n < p.seqs; n += gridDim.y) {
        int64_t t0, t1;
        scan_bounds(p, n, t0, t1);
        float h = p.state ? p.state[n * p.channels + c] : 0.0f;
        for (int64_t t = t0; t < t1; ++t) {
            if (p.ckpt && t % kScanCkpt == 0) p.ckpt[t / kScanCkpt * p.channels + c] = h;
            const Gates q = scan_gates(rate, dtb, to_f32(static_cast<const T*>(p.a)[t * p.a_stride + c]),
                                       to_f32(static_cast<const T*>(p.b)[t * p.b_stride + c]));
            h = q.g * h + q.beta * to_f32(static_cast<const T*>(p.x)[t * p.x_stride + c]);
            static_cast<T*>(p.out)[t * p.out_stride + c] = from_f32<T>(h);
        }
        p.new_state[n * p.channels + c] = h;
    }
}

template <typename T>
__global__ void __launch_bounds__(128) gdn_scan_backward_kernel(const ScanParams p, const ScanGradParams d) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.channels) return;
    const float rate = expf(p.A_log[c]), dtb = p.dt_bias[c];
    for (int64_t n = blockIdx.y; n < p.seqs; n += gridDim.y) {
        int64_t t0, t1;
        scan_bounds(p, n, t0, t1);
        float e = d.d_new_state ? d.d_new_state[n * p.channels + c] : 0.0f;
        float sA = 0.0f, sdt = 0.0f;
        float before[kScanCkpt];
        int64_t end = t1;
        while (end > t0) {
            int64_t begin = (end - 1) / kScanCkpt * kScanCkpt;
            float h;
            if (begin <= t0) {
                begin = t0;
                h = p.state ? p.state[n * p.channels + c] : 0.0f;
            } else {
                h = p.ckpt[begin / kScanCkpt * p.channels + c];
            }
            for (int64_t t = begin; t < end; ++t) {
                before[t - begin] = h;
                const Gates q = scan_gates(rate, dtb, to_f32(static_cast<const T*>(p.a)[t * p.a_stride + c]),
                                           to_f32(static_cast<const T*>(p.b)[t * p.b_stride + c]));
                h = q.g * h + q.beta * to_f32(static_cast<const T*>(p.x)[t * p.x_stride + c]);
            }
            for (int64_t t = end - 1; t >= begin; --t) {
                const Gates q = scan_gates(rate, dtb, to_f32(static_cast<const T*>(p.a)[t * p.a_stride + c]),
                                           to_f32(static_cast<const T*>(p.b)[t * p.b_stride + c]));
                const float x = to_f32(static_cast<const T*>(p.x)[t * p.x_stride + c]);
                const float G = to_f32(static_cast<const T*>(d.dy)[t * d.dy_stride + c]) + e;
                e = q.g * G;
                const float dl = e * before[t - begin];
                const float da = -dl * rate / (1.0f + expf(-q.z));
                sA += dl * q.l;
                sdt += da;
                static_cast<T*>(d.dx)[t * d.dx_stride + c] = from_f32<T>(G * q.beta);
                static_cast<T*>(d.da)[t * d.da_stride + c] = from_f32<T>(da);
                static_cast<T*>(d.db)[t * d.db_stride + c] = from_f32<T>(G * x * q.beta * (1.0f - q.beta));
            }
            end = begin;
        }
        if (d.d_state) d.d_state[n * p.channels + c] = e;
        d.dA_part[n * p.channels + c] = sA;
        d.dt_part[n * p.channels + c] = sdt;
    }
}

// Rows that belong to no sequence: out rows (and gradients) are zeros.
template <typename T>
__global__ void gdn_scan_zero_uncovered_kernel(const ScanParams p, T* o0, int64_t s0, T* o1, int64_t s1, T* o2,
                                               int64_t s2) {
    int64_t lo = p.seqs > 0 ? scan_cu(p, 0) : 0, hi = p.seqs > 0 ? scan_cu(p, p.seqs) : 0;
    for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
        if (t >= lo && t < hi) continue;
        for (int c = threadIdx.x; c < p.channels; c += blockDim.x) {
            o0[t * s0 + c] = from_f32<T>(0.0f);
            if (o1) o1[t * s1 + c] = from_f32<T>(0.0f);
            if (o2) o2[t * s2 + c] = from_f32<T>(0.0f);
        }
    }
}

__global__ void gdn_scan_sum_parts_kernel(const float* a, const float* b, float* oa, float* ob, int64_t n, int channels) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= channels) return;
    float sa = 0.0f, sb = 0.0f;
    for (int64_t i = 0; i < n; ++i) {
        sa += a[i * channels + c];
        sb += b[i * channels + c];
    }
    oa[c] = sa;
    ob[c] = sb;
}

// One or a few tokens per sequence: element (sequence, channel) per thread.
// The thread reads its state element before it writes it, so state may be
// new_state.
template <typename T>
__global__ void __launch_bounds__(128) gdn_scan_step_kernel(const ScanParams p, int64_t steps) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= p.channels) return;
    const float rate = expf(p.A_log[c]), dtb = p.dt_bias[c];
    for (int64_t n = blockIdx.y; n < p.seqs; n += gridDim.y) {
        float h = p.state[n * p.channels + c];
        for (int64_t t = n * steps; t < (n + 1) * steps; ++t) {
            const Gates q = scan_gates(rate, dtb, to_f32(static_cast<const T*>(p.a)[t * p.a_stride + c]),
                                       to_f32(static_cast<const T*>(p.b)[t * p.b_stride + c]));
            h = q.g * h + q.beta * to_f32(static_cast<const T*>(p.x)[t * p.x_stride + c]);
            static_cast<T*>(p.out)[t * p.out_stride + c] = from_f32<T>(h);
        }
        p.new_state[n * p.channels + c] = h;
    }
}

static size_t scan_backward_workspace_bytes(int64_t tokens, int64_t seqs, int64_t channels) {
    (void)tokens;
    return static_cast<size_t>(2 * (seqs > 0 ? seqs : 1) * channels) * sizeof(float);
}

template <typename T>
static cudaError_t launch_scan(const ScanParams& p, cudaStream_t s) {
    const dim3 grid((p.channels + 127) / 128, static_cast<unsigned>(p.seqs < 65535 ? (p.seqs > 0 ? p.seqs : 1) : 65535));
    gdn_scan_kernel<T><<<grid, 128, 0, s>>>(p);
    if (p.tokens > 0)
        gdn_scan_zero_uncovered_kernel<T><<<static_cast<unsigned>(p.tokens < 1024 ? p.tokens : 1024), 128, 0, s>>>(
            p, static_cast<T*>(p.out), p.out_stride, nullptr, 0, nullptr, 0);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_scan_backward(const ScanParams& p, const ScanGradParams& d, cudaStream_t s) {
    const unsigned gx = (p.channels + 127) / 128;
    const dim3 grid(gx, static_cast<unsigned>(p.seqs < 65535 ? (p.seqs > 0 ? p.seqs : 1) : 65535));
    gdn_scan_backward_kernel<T><<<grid, 128, 0, s>>>(p, d);
    gdn_scan_sum_parts_kernel<<<gx, 128, 0, s>>>(d.dA_part, d.dt_part, d.dA_log, d.ddt_bias, p.seqs, p.channels);
    if (p.tokens > 0)
        gdn_scan_zero_uncovered_kernel<T><<<static_cast<unsigned>(p.tokens < 1024 ? p.tokens : 1024), 128, 0, s>>>(
            p, static_cast<T*>(d.dx), d.dx_stride, static_cast<T*>(d.da), d.da_stride, static_cast<T*>(d.db),
            d.db_stride);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_scan_step(const ScanParams& p, int64_t steps, cudaStream_t s) {
    const dim3 grid((p.channels + 127) / 128, static_cast<unsigned>(p.seqs < 65535 ? p.seqs : 65535));
    gdn_scan_step_kernel<T><<<grid, 128, 0, s>>>(p, steps);
    return cudaGetLastError();
}

static bool dtype_ok(int dtype) { return dtype >= GDN_DTYPE_BF16 && dtype <= GDN_DTYPE_F32; }
static uintptr_t dtype_bytes(int dtype) { return dtype == GDN_DTYPE_F32 ? 4 : 2; }

// Argument checks shared by the three entry points, then the kernel parameters.
static int scan_setup(const GdnScanArgs* a, ScanParams& p, bool step) {
    if (a == nullptr) return GDN_ERR_NULL_POINTER;
    if (!dtype_ok(a->dtype)) return GDN_ERR_BAD_DTYPE;
    if (!step && a->cu_seqlens_dtype != GDN_SEQLENS_INT32 && a->cu_seqlens_dtype != GDN_SEQLENS_INT64)
        return GDN_ERR_BAD_DTYPE;
    if (a->total_tokens < 0 || a->total_tokens > 0x7fff0000LL || a->num_seqs < 0 || a->num_seqs > 0x7fff0000LL ||
        a->channels < 1 || a->channels > (1 << 20))
        return GDN_ERR_BAD_SIZE;
    if (!a->A_log || !a->dt_bias || (!step && !a->cu_seqlens)) return GDN_ERR_NULL_POINTER;
    if (a->total_tokens > 0 && (!a->x || !a->a || !a->b)) return GDN_ERR_NULL_POINTER;
    if (a->total_tokens > 1 && (a->x_stride < a->channels || a->a_stride < a->channels || a->b_stride < a->channels))
        return GDN_ERR_BAD_SIZE;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(a->x, es) || !aligned(a->a, es) || !aligned(a->b, es) || !aligned(a->output, es) ||
        !aligned(a->A_log, 4) || !aligned(a->dt_bias, 4) || !aligned(a->state, 4) || !aligned(a->new_state, 4) ||
        !aligned(a->checkpoints, 4) ||
        (!step && !aligned(a->cu_seqlens, a->cu_seqlens_dtype == GDN_SEQLENS_INT64 ? 8 : 4)))
        return GDN_ERR_MISALIGNED;
    p.x = a->x;
    p.a = a->a;
    p.b = a->b;
    p.x_stride = a->x_stride;
    p.a_stride = a->a_stride;
    p.b_stride = a->b_stride;
    p.out_stride = a->output_stride;
    p.A_log = a->A_log;
    p.dt_bias = a->dt_bias;
    p.state = a->state;
    p.cu = a->cu_seqlens;
    p.cu_is_int64 = a->cu_seqlens_dtype == GDN_SEQLENS_INT64;
    p.tokens = a->total_tokens;
    p.seqs = a->num_seqs;
    p.channels = static_cast<int>(a->channels);
    p.out = a->output;
    p.new_state = a->new_state;
    p.ckpt = a->checkpoints;
    return GDN_OK;
}
}  // namespace gdn

extern "C" int gdn_scan_launch(const GdnScanArgs* a, void* stream) {
    ScanParams p;
    if (int rc = scan_setup(a, p, false)) return rc;
    if (a->total_tokens > 0 && !a->output) return GDN_ERR_NULL_POINTER;
    if (a->num_seqs > 0 && !a->new_state) return GDN_ERR_NULL_POINTER;
    if (a->total_tokens > 1 && a->output_stride < a->channels) return GDN_ERR_BAD_SIZE;
    if (a->state != nullptr && a->num_seqs > 0 && a->state == a->new_state) return GDN_ERR_BAD_SIZE;
    if (int rc = check_device()) return rc;
    if (a->num_seqs == 0 && a->total_tokens == 0) return GDN_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_scan<float>(p, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_scan<__half>(p, s)
                                                      : launch_scan<__nv_bfloat16>(p, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" int64_t gdn_scan_checkpoint_rows(int64_t total_tokens) {
    return total_tokens < 0 ? 0 : (total_tokens + kScanCkpt - 1) / kScanCkpt;
}

extern "C" size_t gdn_scan_backward_workspace_size(int64_t total_tokens, int64_t num_seqs, int64_t channels) {
    if (total_tokens < 0 || num_seqs < 0 || channels < 1) return 0;
    return scan_backward_workspace_bytes(total_tokens, num_seqs, channels);
}

extern "C" int gdn_scan_backward_launch(const GdnScanArgs* a, const GdnScanGradArgs* g, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    if (g == nullptr) return GDN_ERR_NULL_POINTER;
    ScanParams p;
    if (int rc = scan_setup(a, p, false)) return rc;
    if (a->total_tokens > 0 && (!g->d_output || !g->dx || !g->da || !g->db || !a->checkpoints))
        return GDN_ERR_NULL_POINTER;
    if (!g->dA_log || !g->d_dt_bias) return GDN_ERR_NULL_POINTER;
    if (a->total_tokens > 1 && (g->d_output_stride < a->channels || g->dx_stride < a->channels ||
                                g->da_stride < a->channels || g->db_stride < a->channels))
        return GDN_ERR_BAD_SIZE;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(g->d_output, es) || !aligned(g->dx, es) || !aligned(g->da, es) || !aligned(g->db, es) ||
        !aligned(g->d_new_state, 4) || !aligned(g->d_state, 4) || !aligned(g->dA_log, 4) || !aligned(g->d_dt_bias, 4))
        return GDN_ERR_MISALIGNED;
    const size_t need = scan_backward_workspace_bytes(a->total_tokens, a->num_seqs, a->channels);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)) return GDN_ERR_WORKSPACE;
    if (int rc = check_device()) return rc;
    ScanGradParams d;
    d.dy = g->d_output;
    d.dy_stride = g->d_output_stride;
    d.dx_stride = g->dx_stride;
    d.da_stride = g->da_stride;
    d.db_stride = g->db_stride;
    d.d_new_state = g->d_new_state;
    d.dx = g->dx;
    d.da = g->da;
    d.db = g->db;
    d.d_state = g->d_state;
    d.dA_part = static_cast<float*>(workspace);
    d.dt_part = d.dA_part + (a->num_seqs > 0 ? a->num_seqs : 1) * a->channels;
    d.dA_log = g->dA_log;
    d.ddt_bias = g->d_dt_bias;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_scan_backward<float>(p, d, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_scan_backward<__half>(p, d, s)
                                                      : launch_scan_backward<__nv_bfloat16>(p, d, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" int gdn_scan_step_launch(const GdnScanArgs* a, int64_t tokens, void* stream) {
    ScanParams p;
    if (int rc = scan_setup(a, p, true)) return rc;
    if (tokens < 1 || tokens > 0x7fff0000LL || a->total_tokens != a->num_seqs * tokens) return GDN_ERR_BAD_SIZE;
    if (a->num_seqs == 0) return check_device();
    if (!a->output || !a->state || !a->new_state) return GDN_ERR_NULL_POINTER;
    if (a->total_tokens > 1 && a->output_stride < a->channels) return GDN_ERR_BAD_SIZE;
    if (int rc = check_device()) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_scan_step<float>(p, tokens, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_scan_step<__half>(p, tokens, s)
                                                      : launch_scan_step<__nv_bfloat16>(p, tokens, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}
