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
#include <string.h>

#include <type_traits>

#include "gdn_common.cuh"
#include "gdn_once.cuh"
#include "gdn_overlap.cuh"
#include "tc05.cuh"

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

// ------------------------------------------------ two channels at a time --
// A thread owns two neighbouring channels; sm_100 multiplies and adds such a
// pair in one instruction (fma.rn.f32x2).
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(F2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ F2 splat2(float a) { return pack2(a, a); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max_keep_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_keep_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float kLog2e = 1.4426950408889634f;

// z -> log2 g = rate softplus(z) of N pairs side by side (a polynomial's
// constants are then in registers once for all of them), with
// softplus(z) = max(z, 0) + log1p(u), u = exp(-|z|) in [0, 1].
// log1p(u) / u is a polynomial, fitted by weighted least squares iterated to
// the smallest maximal relative error (Lawson): 2.2e-7, its constants rounded to
// floats.  lg2.approx is not
// usable here: its error near 1 is absolute (2^-22), and softplus of a
// strongly negative argument is a tiny number whose relative error the
// recurrence multiplies by its memory.
template <int N>
__device__ __forceinline__ void log2_decays(F2 (&z)[N], F2 (&u)[N], F2 rate) {
    constexpr float kLog1p[8] = {0.9999998211860657f, -0.4999740421772003f, 0.33275479078292847f, -0.24495463073253632f, 0.17745240032672882f, -0.10768169909715652f, 0.04408962279558182f, -0.008539206348359585f};
    F2 r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 e = unpack2(mul2(z[i], splat2(kLog2e))), v = unpack2(z[i]);
        u[i] = pack2(ex2_approx(-fabsf(e.x)), ex2_approx(-fabsf(e.y)));
        z[i] = pack2(max_keep_nan(v.x, 0.0f), max_keep_nan(v.y, 0.0f));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = fma2(splat2(kLog1p[7]), u[i], splat2(kLog1p[6]));
#pragma unroll
    for (int d = 5; d >= 0; --d)
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fma2(r[i], u[i], splat2(kLog1p[d]));
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = mul2(rate, fma2(u[i], r[i], z[i]));
}
// t -> 2^t of N pairs, t <= 0.  ex2.approx is within 1.2 units in the last
// place, but off in one direction (measured: by 0.05 of them on average at
// -0.001, 0.2 at -0.01), which a decay's memory of a thousand tokens adds up to
// 1e-5.  So decays above 2^-0.25 are 1 + t q(t), q fitted like the polynomial
// above (3.7e-9; evaluated in floats 0.4 units, 0.001 on average).
template <int N>
__device__ __forceinline__ void exp2_decays(F2 (&t)[N]) {
    constexpr float kExp2[4] = {0.693146824836731f, 0.24021293222904205f, 0.05534094199538231f, 0.008836725726723671f};
    F2 q[N];
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = fma2(splat2(kExp2[3]), t[i], splat2(kExp2[2]));
#pragma unroll
    for (int d = 1; d >= 0; --d)
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = fma2(q[i], t[i], splat2(kExp2[d]));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float2 v = unpack2(t[i]), near = unpack2(fma2(q[i], t[i], splat2(1.0f)));
        t[i] = pack2(v.x > -0.25f ? near.x : ex2_approx(v.x), v.y > -0.25f ? near.y : ex2_approx(v.y));
    }
}
template <int N>
__device__ __forceinline__ void decays(F2 (&z)[N], F2 rate) {
    F2 u[N];
    log2_decays(z, u, rate);
    exp2_decays(z);
}
__device__ __forceinline__ F2 sigmoid2(F2 b) {
    const float2 e = unpack2(mul2(b, splat2(-kLog2e)));
    const float2 d = unpack2(add2(pack2(ex2_approx(e.x), ex2_approx(e.y)), splat2(1.0f)));
    return pack2(rcp_approx(d.x), rcp_approx(d.y));
}
// sigmoid(b) and 1 - sigmoid(b), which the difference would lose from b = 17 on:
// 1 / (1 + e) and e / (1 + e) with e = exp(-b).  Where that overflows, sigmoid(b)
// is flushed to zero, and a finite e keeps its product with it a number.
__device__ __forceinline__ F2 sigmoid2(F2 b, F2& rest) {
    constexpr float kMost = 3.402823466e38f;
    const float2 t = unpack2(mul2(b, splat2(-kLog2e)));
    const F2 e = pack2(min_keep_nan(ex2_approx(t.x), kMost), min_keep_nan(ex2_approx(t.y), kMost));
    const float2 d = unpack2(add2(e, splat2(1.0f)));
    const F2 beta = pack2(rcp_approx(d.x), rcp_approx(d.y));
    rest = mul2(e, beta);
    return beta;
}

template <typename T>
__device__ __forceinline__ F2 load_pair(const void* p);  // two neighbouring elements in shared memory
template <>
__device__ __forceinline__ F2 load_pair<float>(const void* p) { return *static_cast<const F2*>(p); }
template <>
__device__ __forceinline__ F2 load_pair<__half>(const void* p) {
    const float2 v = __half22float2(*static_cast<const __half2*>(p));
    return pack2(v.x, v.y);
}
template <>
__device__ __forceinline__ F2 load_pair<__nv_bfloat16>(const void* p) {
    const uint32_t u = *static_cast<const uint32_t*>(p);
    return pack2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Two neighbouring elements of a row; `pairs`: the row starts on a pair's boundary.
template <typename T>
__device__ __forceinline__ void store_pair(T* p, F2 v, bool pairs, bool ok0, bool ok1) {
    const float2 f = unpack2(v);
    if (pairs && ok1) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float2*>(p) = f;
        } else {
            T e[2] = {from_f32<T>(f.x), from_f32<T>(f.y)};
            *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
        }
    } else {
        if (ok0) p[0] = from_f32<T>(f.x);
        if (ok1) p[1] = from_f32<T>(f.y);
    }
}

// ---------------------------------------------------------------- cluster --
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// A bounded wait of the whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, tc05::mbar_wait(bar, parity));
}
// The last thing every thread of a scan does, also one that gave up a wait: no
// CTA's shared memory goes while a CTA of its cluster can still send to it.
// Where no wait ran out, all that was sent to this CTA has arrived, because it
// waited for it; a warp that gave up stays for what is still on its way (sent
// before the barrier, and under a microsecond from arriving).
__device__ __forceinline__ void leave_cluster(bool gave_up) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (gave_up) {
        record_status(32 /* GDN_ERR_DEVICE_TIMEOUT */);
        constexpr uint64_t kStayNs = 100000;
        const uint64_t t0 = tc05::globaltimer_ns();
        for (uint32_t i = 0; i < tc05::kWaitMaxPolls && tc05::globaltimer_ns() - t0 < kStayNs; ++i) {}
    }
}
// 16 bytes into the same shared address of CTA `rank` of the cluster, counted
// by that CTA's mbarrier at the address of `bar`: neither side needs a fence.
__device__ __forceinline__ void st_cluster_f4(uint32_t a, uint32_t bar, uint32_t rank, float4 v) {
    uint32_t ra, rb;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rb) : "r"(bar), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(ra),
                 "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(rb)
                 : "memory");
}

// The scans' CTAs, one to an SM: map warps and a chain warp, the same number to
// each of the four schedulers, so 96 registers a thread forward (16 warps of
// 128: 3 % slower) and 128 backward.  A lane owns two channels; a warp is one
// strip of 64 channels, or two strips of 32 on different tokens.
constexpr int kScanWarps = 19, kScanThreads = 32 * (kScanWarps + 1);
constexpr int kGradWarps = 15, kGradThreads = 32 * (kGradWarps + 1);
template <int STRIPS>
struct Strips {
    static constexpr int kLanes = 32 / STRIPS, kChannels = 2 * kLanes;
    int strip, lane;  // this thread's strip, and its place in it
    __device__ Strips() : strip((threadIdx.x & 31) / kLanes), lane((threadIdx.x & 31) % kLanes) {}
    // Piece i of a tile (in token order) is strip i % STRIPS of warp i / STRIPS;
    // its word in an array [warps][step / 32][32] at this thread's channels.
    __device__ __forceinline__ int word(int i, int step) const { return i / STRIPS * step + i % STRIPS * kLanes + lane; }
};
// Tokens per map warp and tile: a thread's inputs of the next tile wait in
// registers (forward) and what its gates gave in shared memory (backward).
template <typename T>
constexpr int kScanPiece = sizeof(T) == 4 ? 4 : 8;
constexpr int kGradPiece = 4, kGradRows = kGradWarps * kGradPiece;
constexpr int kScanMaxCluster = 16;

// The carry into every kScanCkpt-th packed token is kept for the backward
// pass, which recomputes the states of a tile from it.
constexpr int kScanCkpt = kGradRows;

struct ScanParams {
    const void* x;
    const void* a;
    const void* b;
    uint32_t x_stride, a_stride, b_stride, out_stride;  // BYTES between tokens
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
    bool x_pairs, a_pairs, b_pairs, out_pairs;  // rows start on a pair of elements' boundary
};

struct ScanGradParams {
    const void* dy;
    uint32_t dy_stride, dx_stride, da_stride, db_stride;  // BYTES between tokens
    const float* d_new_state;  // NULL: zero
    void* dx;
    void* da;
    void* db;
    float* d_state;  // NULL: not wanted
    float* dA_log;
    float* ddt_bias;
    bool dy_pairs, grad_pairs;  // rows start on a pair of elements' boundary (dx, da and db together)
};

// Row t of a tensor with `stride` bytes between rows (one wide multiply-add).
template <typename T>
__device__ __forceinline__ T* row_at(const void* base, int64_t t, uint32_t stride) {
    return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + static_cast<uint64_t>(static_cast<uint32_t>(t)) * stride);
}

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

// A piece of the recurrence is an affine map of the state before it,
// h -> A h + H, as (A0, A1, H0, H1) for a thread's two channels.  A piece in
// which a sequence starts does not depend on the state before it: A = -0
// says so (decays are >= +0).  The fast forms multiply all the same, which
// drops a finite state; an infinity or a NaN would cross into the next sequence
// as a NaN, so a chain that ends in one is done again with the forms that
// select.
__device__ __forceinline__ bool is_start(float a) { return __float_as_uint(a) == 0x80000000u; }
__device__ __forceinline__ F2 apply_map(float4 m, F2 h) { return fma2(pack2(m.x, m.y), h, pack2(m.z, m.w)); }
// Decays are positive, but a piece's product of them can fall below the least
// float: an infinite state stays what it is (0 times it would be a NaN) until
// the sequence ends.
__device__ __forceinline__ float select_one(float A, float H, float h, float r) {
    return is_start(A) ? H : fabsf(h) > 3.402823466e38f && A >= 0.0f ? h + H : r;
}
__device__ __noinline__ F2 apply_map_select(float4 m, F2 h) {
    const float2 r = unpack2(apply_map(m, h)), v = unpack2(h);
    return pack2(select_one(m.x, m.z, v.x, r.x), select_one(m.y, m.w, v.y, r.y));
}
// The same without that, for the backward pass: beside an infinity its gradients
// are not finite either way.
__device__ __forceinline__ F2 apply_map_start(float4 m, F2 h) {
    const float2 r = unpack2(apply_map(m, h));
    return pack2(is_start(m.x) ? m.z : r.x, is_start(m.y) ? m.w : r.y);
}
struct Map2 {
    F2 A, H;
};
__device__ __forceinline__ bool has_nan(F2 v) {
    const float2 f = unpack2(v);
    return !(f.x == f.x) || !(f.y == f.y);
}
__device__ __forceinline__ bool all_finite(F2 v) {
    const float2 f = unpack2(v);
    return fabsf(f.x) <= 3.402823466e38f && fabsf(f.y) <= 3.402823466e38f;
}
// The product of n pieces' maps, and to before[.] the product of those ahead
// of each (out of line: the slow form).
template <int STRIPS>
__device__ __noinline__ Map2 chain_select(const float4* maps, int n, int step, float4* before) {
    const Strips<STRIPS> me;
    Map2 r = {splat2(1.0f), splat2(0.0f)};
    for (int i = 0; i < n; ++i) {
        const float4 m = maps[me.word(i, step)];
        const float2 a = unpack2(r.A), h = unpack2(r.H);
        if (i % STRIPS == me.strip) before[me.word(i, 32)] = make_float4(a.x, a.y, h.x, h.y);
        r.H = apply_map_select(m, r.H);
        r.A = pack2(is_start(m.x) ? m.x : a.x * m.x, is_start(m.y) ? m.y : a.y * m.y);
    }
    return r;
}
// The state behind n pieces
__device__ __noinline__ F2 fold_select(const float4* maps, int n, int step, F2 h) {
    for (int i = 0; i < n; ++i) h = apply_map_select(maps[i * step], h);
    return h;
}

// The sequences' offsets: the caller's, or (up to kScanCuMost sequences) a copy
// in shared memory as 32-bit integers, where a search takes a tenth of the time.
constexpr int kScanCuMost = 1023;
struct Offsets {
    const void* cu;
    bool is64;
    int seqs;
    __device__ __forceinline__ int64_t at(int n) const {
        return is64 ? static_cast<const int64_t*>(cu)[n] : static_cast<const int32_t*>(cu)[n];
    }
};
// Every thread calls; a barrier has to follow before the offsets are used.
__device__ __forceinline__ Offsets scan_offsets(const ScanParams& p, int* copy) {
    if (p.seqs > kScanCuMost) return {p.cu, p.cu_is_int64, static_cast<int>(p.seqs)};
    for (int i = threadIdx.x; i <= p.seqs; i += blockDim.x) {
        const int64_t v = scan_cu(p, i);
        copy[i] = v < -1 ? -1 : v > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(v);  // bad ones stay bad
    }
    return {copy, false, static_cast<int>(p.seqs)};
}

// First sequence that ends behind packed token t (seqs if none), by the whole
// warp.  Out of line and, below, in loops that are not unrolled, like
// everything that only pieces with a sequence's start or end need: it is cold
// code whenever it runs, and what it costs is its size.
__device__ __noinline__ int seq_of_token(Offsets o, int64_t t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = o.seqs;
    while (hi - lo > 32) {
        const int step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step - 1;
        const int n = __popc(__ballot_sync(0xffffffffu, i < hi && o.at(i + 1) <= t));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    const int i = lo + lane;
    return lo + __popc(__ballot_sync(0xffffffffu, i < hi && o.at(i + 1) <= t));
}

// Which of W (up to 32) tokens from t on start a sequence, end one,
// belong to one; and the sequence [lo, hi) around the last of them, so that
// tiles inside it need no look at the offsets.
struct Spans {
    uint32_t start, end, covered;
    int lo, hi;
};
template <int W>
constexpr uint32_t kAllTokens = 0xffffffffu >> (32 - W);
__device__ __noinline__ Spans find_spans(Offsets o, int64_t tokens, int64_t t, int width) {
    const int lane = threadIdx.x & 31;
    Spans s = {0, 0, 0, 0, 0};
    const int64_t stop = t + width < tokens ? t + width : tokens;
    if (t >= stop) return s;
    for (int n = seq_of_token(o, t); n < o.seqs;) {
        int64_t b = stop, e = stop;
        if (n + lane < o.seqs) b = o.at(n + lane), e = o.at(n + lane + 1);
        uint32_t st = 0, en = 0, cov = 0;
        int lo = 0, hi = 0;
        if (e > b && b < stop && e > t) {
            if (b >= t) st = 1u << (b - t);
            if (e <= stop) en = 1u << (e - 1 - t);
            const int from = b > t ? static_cast<int>(b - t) : 0, to = static_cast<int>((e < stop ? e : stop) - t);
            cov = (0xffffffffu >> (32 - to)) & (0xffffffffu << from);  // 0 <= from < to <= 32
            if (e > stop) lo = static_cast<int>(b > 0 ? b : 0), hi = static_cast<int>(e < tokens ? e : tokens);
        }
        s.start |= __reduce_or_sync(0xffffffffu, st);
        s.end |= __reduce_or_sync(0xffffffffu, en);
        s.covered |= __reduce_or_sync(0xffffffffu, cov);
        s.lo = max(s.lo, __reduce_max_sync(0xffffffffu, lo));
        s.hi = max(s.hi, __reduce_max_sync(0xffffffffu, hi));
        const int64_t last = __shfl_sync(0xffffffffu, b, 31);
        if (last >= stop) break;
        // On behind the 32, and behind all that are empty where the last of them
        // begins: any number of those can lie at one token, and the other warps'
        // waits are bounded.  So two searches a token at most.
        n = max(n + 32, seq_of_token(o, last));
    }
    return s;
}
// The same, with `s` of an earlier tile: tiles inside one sequence cost two comparisons.
template <int W>
__device__ __forceinline__ void token_spans(const Offsets& o, int64_t tokens, int64_t t, Spans& s) {
    if (t > s.lo && t + W < s.hi) {
        s.start = s.end = 0;
        s.covered = kAllTokens<W>;
    } else {
        s = find_spans(o, tokens, t, W);
    }
}

// Channels c and c + 1 of the state rows of the sequences that packed token t
// (in strip 0) and those `apart` tokens on (in the next strips) belong to;
// `which` has bit i * apart set for the strips that want theirs, the others keep
// `other`.  The whole warp calls; nothing here waits for the rows.
template <int STRIPS>
__device__ __forceinline__ F2 state_of_strips(const Offsets& o, const float* state, int channels, uint32_t which, int apart,
                                              int64_t t, int c, int strip, F2 other) {
#pragma unroll
    for (int i = 0; i < STRIPS; ++i)
        if (which >> (i * apart) & 1) {
            const int n = seq_of_token(o, t + i * apart);
            if (strip == i) {
                float v0 = 0.0f, v1 = 0.0f;
                const float* row = state + static_cast<int64_t>(n) * channels;
                if (state != nullptr && n < o.seqs && c < channels) v0 = row[c];
                if (state != nullptr && n < o.seqs && c + 1 < channels) v1 = row[c + 1];
                other = pack2(v0, v1);
            }
        }
    return other;
}
// Lanes with `mine` store theirs for packed token t's sequence.  The whole warp calls.
__device__ __forceinline__ void store_state_of_strip(const Offsets& o, float* state, int channels, int64_t t, int c, bool mine,
                                                     F2 h) {
    const int n = seq_of_token(o, t);
    if (!mine || state == nullptr || n >= o.seqs) return;
    const float2 v = unpack2(h);
    float* row = state + static_cast<int64_t>(n) * channels;
    if (c < channels) row[c] = v.x;
    if (c + 1 < channels) row[c + 1] = v.y;
}

// Two neighbouring elements as they are stored, read past the L1 cache.
template <typename T>
struct RawPair {
    uint32_t bits;
};
template <>
struct RawPair<float> {
    uint2 bits;
};
template <typename T>
__device__ __forceinline__ RawPair<T> load_raw(const T* p) {
    RawPair<T> r;
    if constexpr (sizeof(T) == 4)
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.bits.x), "=r"(r.bits.y) : "l"(p));
    else
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.bits) : "l"(p));
    return r;
}
template <typename T>
__device__ __forceinline__ RawPair<T> load_raw_part(const T* p, bool ok0, bool ok1) {
    RawPair<T> r;
    T e[2] = {from_f32<T>(0.0f), from_f32<T>(0.0f)};
    if (ok0) e[0] = p[0];
    if (ok1) e[1] = p[1];
    memcpy(&r, e, sizeof(e));
    return r;
}
template <typename T>
__device__ __forceinline__ F2 raw_to_f2(RawPair<T> r) { return load_pair<T>(&r); }

// Sequences without a token pass their state on; bad offsets are reported.
__device__ __forceinline__ void scan_empty_sequences(const ScanParams& p, const float* from, float* to, int c0, int c1,
                                                     int first, int step) {
    c1 = min(p.channels, c1);
    for (int64_t n = first; n < p.seqs; n += step) {
        int64_t t0, t1;
        scan_bounds(p, n, t0, t1);
        if (t0 == t1 && to)
            for (int c = c0; c < c1; ++c) to[n * p.channels + c] = from ? from[n * p.channels + c] : 0.0f;
    }
}

// The packed scan in one pass over the data.  A cluster of R CTAs takes 64
// (or 32) channels and walks the packed tokens, whatever sequences they belong
// to, R tiles at a time: ragged batches and one long sequence load the GPU alike.
//   map warp    g and u = beta x of its piece of the tile's tokens, chained
//               into the maps from the piece's start, to shared memory (its
//               own words: no other warp reads them but the piece's last);
//               then the states and outputs of its piece of the tile before.
//               The next tile's inputs are on their way meanwhile.
//   chain warp  the tile's W maps chained, their product sent to every CTA of
//               the cluster (distributed shared memory, counted by an mbarrier
//               there: no fence, no cluster-wide barrier), and behind all R of
//               them the state at the tile's start, always chained in the same
//               order (the same bits on every run).
// So the gates' arithmetic, which is what the kernel is made of, has a whole
// tile's time to hide the cluster's exchange behind.
// 85 warp instructions per token and pair of channels, about 35 of them gates and
// chains, which at full issue on every SM would take 79 us of the first case below.
// It takes longer because clusters fill 128 of the 148 SMs and those issue in 63 %
// of their slots: with five warps to a scheduler the fixed latencies of dependent
// instructions (1.8 of a warp's stalls per issue; special-function pipe 1.1,
// memory 0.5) are not all hidden.  Measured (bf16): 1 x 16384 x 4096 145 us, 3.7
// TB/s of inputs and outputs, 56 % of the copy rate; 1 x 40000 x 1024 99 us; 32 x
// 64..2048 x 2048 177 us.  A thread per sequence and channel took 42 ms for the
// second.
template <typename T, int STRIPS>
__global__ void __launch_bounds__(kScanThreads, 1) gdn_scan_kernel(const ScanParams p) {
    constexpr int W = kScanWarps, kPiece = kScanPiece<T>, kRows = W * kPiece, kTile = STRIPS * kRows;
    constexpr int kSpan = STRIPS * kPiece;  // a warp's tokens
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ F2 s_in[2][32];  // the state at the tile's start
    __shared__ __align__(8) uint64_t s_bar[6];
    __shared__ int s_cu[kScanCuMost + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int R = cluster_size(), rank = cluster_rank();
    const Strips<STRIPS> me;
    float4* maps = reinterpret_cast<float4*>(smem);  // [2][kRows][32]: of each token, from its piece's start
    float4* befores = maps + 2 * kRows * 32;         // [2][W][32]: of each piece, from the tile's start
    float4* ranks = befores + 2 * W * 32;            // [2][R][32]: the cluster's tiles
    const int c0 = blockIdx.y * me.kChannels, c = c0 + 2 * me.lane;
    const bool ok0 = c < p.channels, ok1 = c + 1 < p.channels;
    const uint32_t full = tc05::smem_u32(s_bar), ready = full + 16, arrived = full + 32;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc05::mbar_init(full + 8 * i, W);
            tc05::mbar_init(ready + 8 * i, 1);
            tc05::mbar_init(arrived + 8 * i, 1);
            tc05::mbar_expect_tx(arrived + 8 * i, R * 512);
        }
        tc05::fence_mbar_init();
    }
    const int tokens = static_cast<int>(p.tokens);
    const int tiles = (tokens + kTile - 1) / kTile, steps = (tiles + R - 1) / R;
    const T* x0 = static_cast<const T*>(p.x) + c;
    const T* a0 = static_cast<const T*>(p.a) + c;
    const T* b0 = static_cast<const T*>(p.b) + c;
    T* out0 = static_cast<T*>(p.out) + c;
    const bool all_channels = c0 + me.kChannels <= p.channels;
    const bool whole = p.x_pairs && p.a_pairs && p.b_pairs && all_channels;
    constexpr int kBatch = 4;
    RawPair<T> x[kPiece], a[kPiece], b[kPiece];
    auto fetch = [&](int k, int from) {  // kBatch tokens of tile k
        const int w0 = (k * R + rank) * kTile + warp * kSpan, t0 = w0 + me.strip * kPiece;
        if (whole && k < steps && w0 + kSpan <= tokens) {
#pragma unroll
            for (int j = from; j < from + kBatch; ++j) {
                x[j] = load_raw(row_at<const T>(x0, t0 + j, p.x_stride));
                a[j] = load_raw(row_at<const T>(a0, t0 + j, p.a_stride));
                b[j] = load_raw(row_at<const T>(b0, t0 + j, p.b_stride));
            }
        } else {
#pragma unroll
            for (int j = from; j < from + kBatch; ++j) {
                const bool live = k < steps && t0 + j < tokens;
                x[j] = load_raw_part(row_at<const T>(x0, t0 + j, p.x_stride), live && ok0, live && ok1);
                a[j] = load_raw_part(row_at<const T>(a0, t0 + j, p.a_stride), live && ok0, live && ok1);
                b[j] = load_raw_part(row_at<const T>(b0, t0 + j, p.b_stride), live && ok0, live && ok1);
            }
        }
    };
    if (warp < W) {
#pragma unroll
        for (int i = 0; i < kPiece; i += kBatch) fetch(0, i);
    }
    const Offsets offsets = scan_offsets(p, s_cu);
    cluster_arrive();
    const F2 dtb = pack2(ok0 ? p.dt_bias[c] : 0.0f, ok1 ? p.dt_bias[c + 1] : 0.0f);
    const F2 rate = pack2(ok0 ? -kLog2e * expf(p.A_log[c]) : 0.0f, ok1 ? -kLog2e * expf(p.A_log[c + 1]) : 0.0f);
    scan_empty_sequences(p, p.state, p.new_state, c0, c0 + me.kChannels, rank * blockDim.x + threadIdx.x, R * blockDim.x);
    cluster_wait();  // every CTA of the cluster runs and has its barriers

    bool gave_up = false;
    if (warp == W) {
        F2 carry = splat2(0.0f);
        for (int k = 0; k < steps; ++k) {
            const int buf = k & 1, phase = k >> 1 & 1;
            if ((gave_up = !warp_wait(full + 8 * buf, phase))) break;
            const float4* last = maps + (buf * kRows + kPiece - 1) * 32;  // a piece's whole map is its last token's
            float4* before = befores + buf * W * 32;
            F2 A = splat2(1.0f), H = splat2(0.0f);
            uint32_t sx = 0, sy = 0;  // the sign of A, kept apart: the product would lose it in two starts
            const auto factor = [&] {
                const float2 a = unpack2(A);
                return make_float2(__uint_as_float((__float_as_uint(a.x) & 0x7fffffffu) | (sx & 0x80000000u)),
                                   __uint_as_float((__float_as_uint(a.y) & 0x7fffffffu) | (sy & 0x80000000u)));
            };
#pragma unroll
            for (int i = 0; i < STRIPS * W; ++i) {
                const float4 m = last[me.word(i, kPiece * 32)];
                const float2 va = factor(), vh = unpack2(H);
                if (i % STRIPS == me.strip) before[me.word(i, 32)] = make_float4(va.x, va.y, vh.x, vh.y);
                H = apply_map(m, H);
                A = mul2(A, pack2(m.x, m.y));
                sx |= __float_as_uint(m.x), sy |= __float_as_uint(m.y);
            }
            const float2 signed_A = factor();
            A = pack2(signed_A.x, signed_A.y);
            if (__any_sync(0xffffffffu, has_nan(A) || has_nan(H))) {
                const Map2 all = chain_select<STRIPS>(last, STRIPS * W, kPiece * 32, before);
                A = all.A, H = all.H;
            }
            const float2 va = unpack2(A), vh = unpack2(H);
            const uint32_t to = tc05::smem_u32(ranks + (buf * R + rank) * 32 + lane);
            // A slot is written again two tiles on: by then this CTA has every
            // CTA's map of tile k + 1, sent after that CTA had read tile k's.
            for (int r = 0; r < R; ++r)
                st_cluster_f4(to, arrived + 8 * buf, r, make_float4(va.x, va.y, vh.x, vh.y));
            if ((gave_up = !warp_wait(arrived + 8 * buf, phase))) break;
            if (lane == 0) tc05::mbar_expect_tx(arrived + 8 * buf, R * 512);
            const float4* all = ranks + buf * R * 32 + lane;
            F2 in = carry;
#pragma unroll 4
            for (int r = 0; r < rank; ++r) in = apply_map(all[r * 32], in);
            F2 next = in;
#pragma unroll 4
            for (int r = rank; r < R; ++r) next = apply_map(all[r * 32], next);
            if (__any_sync(0xffffffffu, has_nan(next))) {
                in = fold_select(all, rank, 32, carry);
                next = fold_select(all + rank * 32, R - rank, 32, in);
            }
            s_in[buf][lane] = in;
            __syncwarp();
            if (lane == 0) tc05::mbar_arrive(ready + 8 * buf);
            carry = next;
            if (p.ckpt && k == 0 && rank == 0 && me.strip == 0) {  // ahead of the first token, for completeness
                if (ok0) p.ckpt[c] = 0.0f;
                if (ok1) p.ckpt[c + 1] = 0.0f;
            }
        }
    } else {
        Spans span = {0, 0, 0, 0, 0};
        uint32_t ends = 0;  // of the tile before
        for (int k = 0; k <= steps; ++k) {
            if (k < steps) {
                const int w0 = (k * R + rank) * kTile + warp * kSpan, buf = k & 1;
                token_spans<kSpan>(offsets, tokens, w0, span);
                const uint32_t special = span.start | (~span.covered & kAllTokens<kSpan>);
                float4* m = maps + (buf * kRows + warp * kPiece) * 32 + lane;
                F2 A = splat2(1.0f), H = splat2(0.0f);  // the map up to each token
#pragma unroll
                for (int i = 0; i < kPiece; i += kBatch) {
                    F2 z[kBatch], u[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        z[j] = add2(raw_to_f2<T>(a[i + j]), dtb);
                        u[j] = mul2(sigmoid2(raw_to_f2<T>(b[i + j])), raw_to_f2<T>(x[i + j]));
                    }
                    fetch(k + 1, i);
                    decays(z, rate);
                    auto put = [&](int j) {
                        const float2 va = unpack2(A), vh = unpack2(H);
                        m[(i + j) * 32] = make_float4(va.x, va.y, vh.x, vh.y);
                    };
                    if (special == 0) {
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) {
                            A = mul2(A, z[j]);
                            H = fma2(z[j], H, u[j]);
                            put(j);
                        }
                    } else {  // g and u for now
#pragma unroll
                        for (int j = 0; j < kBatch; ++j) {
                            const float2 vg = unpack2(z[j]), vu = unpack2(u[j]);
                            m[(i + j) * 32] = make_float4(vg.x, vg.y, vu.x, vu.y);
                        }
                    }
                }
                if (special) {
                    const uint32_t fresh = special >> me.strip * kPiece, covered = span.covered >> me.strip * kPiece;
                    A = splat2(1.0f);
                    H = splat2(0.0f);
#pragma unroll 1
                    for (int j = 0; j < kPiece; ++j) {
                        const float4 gu = m[j * 32];
                        const F2 g = pack2(gu.x, gu.y), u = pack2(gu.z, gu.w);
                        const F2 before = state_of_strips<STRIPS>(offsets, p.state, p.channels, span.start >> j, kPiece, w0 + j, c,
                                                                  me.strip, H);
                        A = fresh >> j & 1 ? splat2(-0.0f) : mul2(A, g);
                        H = covered >> j & 1 ? fma2(g, before, u) : splat2(0.0f);
                        const float2 va = unpack2(A), vh = unpack2(H);
                        m[j * 32] = make_float4(va.x, va.y, vh.x, vh.y);
                    }
                }
                __syncwarp();
                if (lane == 0) tc05::mbar_arrive(full + 8 * buf);
            }
            if (k > 0) {
                const int buf = (k - 1) & 1, w0 = ((k - 1) * R + rank) * kTile + warp * kSpan, t0 = w0 + me.strip * kPiece;
                if ((gave_up = !warp_wait(ready + 8 * buf, (k - 1) >> 1 & 1))) break;
                const float4* m = maps + (buf * kRows + warp * kPiece) * 32 + lane;
                const float4 before = befores[(buf * W + warp) * 32 + lane];
                const F2 tile_in = s_in[buf][lane];
                F2 in = apply_map(before, tile_in), h[kPiece];
                const bool finite = !__any_sync(0xffffffffu, !all_finite(tile_in) || !all_finite(in));
                if (finite) {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) h[j] = apply_map(m[j * 32], in);
                } else {
                    in = apply_map_select(before, tile_in);
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) h[j] = apply_map_select(m[j * 32], in);
                }
                // the piece's token whose state is the next checkpoint, if it has one
                const int kept = kScanCkpt - 1 - t0 % kScanCkpt;
                if (p.ckpt && kept < kPiece && t0 + kept + 1 < tokens) {
                    F2 v = h[0];
#pragma unroll
                    for (int j = 1; j < kPiece; ++j)
                        if (j == kept) v = h[j];
                    float* ck = p.ckpt + static_cast<int64_t>((t0 + kept + 1) / kScanCkpt) * p.channels + c;
                    if (ok0) ck[0] = unpack2(v).x;
                    if (ok1) ck[1] = unpack2(v).y;
                }
                T* out = row_at<T>(out0, t0, p.out_stride);
                if (w0 + kSpan <= tokens && p.out_pairs && all_channels) {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) store_pair(row_at<T>(out, j, p.out_stride), h[j], true, true, true);
                } else {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j)
                        if (t0 + j < tokens) store_pair(row_at<T>(out, j, p.out_stride), h[j], p.out_pairs, ok0, ok1);
                }
#pragma unroll 1
                for (uint32_t left = ends; left; left &= left - 1) {  // sequences that end here
                    const int t = __ffs(left) - 1;
                    store_state_of_strip(offsets, p.new_state, p.channels, w0 + t, c, me.strip == t / kPiece,
                                         apply_map_select(m[t % kPiece * 32], in));
                }
            }
            ends = span.end;
        }
    }
    leave_cluster(gave_up);
}

// What the gates of a backward tile gave, per token and lane: log2 g, beta and
// 1 - beta, sigmoid(z) and the two inputs that are needed again, x and dy, in 40
// bytes.  A thread reads only what it wrote.
constexpr size_t kGradTileBytes = 2 * kGradRows * 32 * 40;
template <typename T>
struct GradTile {
    float4* base;
    float2* rests;
    __device__ GradTile(unsigned char* smem, int lane)
        : base(reinterpret_cast<float4*>(smem) + lane),
          rests(reinterpret_cast<float2*>(smem + 2 * kGradRows * 32 * 32) + lane) {}
    __device__ __forceinline__ void put(int i, F2 t, F2 beta, F2 rest, F2 sig, RawPair<T> x, RawPair<T> dy) {
        const float2 a = unpack2(t), b = unpack2(beta), c = unpack2(sig);
        base[2 * i * 32] = make_float4(a.x, a.y, b.x, b.y);
        base[(2 * i + 1) * 32] = make_float4(c.x, c.y, __uint_as_float(x.bits), __uint_as_float(dy.bits));
        rests[i * 32] = unpack2(rest);
    }
    __device__ __forceinline__ void get(int i, F2& t, F2& beta, F2& rest, F2& sig, F2& x, F2& dy) const {
        const float4 a = base[2 * i * 32], b = base[(2 * i + 1) * 32];
        const float2 c = rests[i * 32];
        t = pack2(a.x, a.y);
        beta = pack2(a.z, a.w);
        rest = pack2(c.x, c.y);
        sig = pack2(b.x, b.y);
        x = raw_to_f2<T>({__float_as_uint(b.z)});
        dy = raw_to_f2<T>({__float_as_uint(b.w)});
    }
};
// With 8 bytes each for x and dy there is room (in clusters of any size) for
// the smaller of beta and 1 - beta, which gives the other; its sign says which.
template <>
struct GradTile<float> {
    float4* base;
    float2* sigs;
    __device__ GradTile(unsigned char* smem, int lane)
        : base(reinterpret_cast<float4*>(smem) + lane),
          sigs(reinterpret_cast<float2*>(smem + 2 * kGradRows * 32 * 32) + lane) {}
    static __device__ __forceinline__ float smaller(float beta, float rest) { return beta > rest ? -rest : beta; }
    __device__ __forceinline__ void put(int i, F2 t, F2 beta, F2 rest, F2 sig, RawPair<float> x, RawPair<float> dy) {
        const float2 a = unpack2(t), b = unpack2(beta), r = unpack2(rest);
        base[2 * i * 32] = make_float4(a.x, a.y, smaller(b.x, r.x), smaller(b.y, r.y));
        base[(2 * i + 1) * 32] = make_float4(__uint_as_float(x.bits.x), __uint_as_float(x.bits.y),
                                             __uint_as_float(dy.bits.x), __uint_as_float(dy.bits.y));
        sigs[i * 32] = unpack2(sig);
    }
    __device__ __forceinline__ void get(int i, F2& t, F2& beta, F2& rest, F2& sig, F2& x, F2& dy) const {
        const float4 a = base[2 * i * 32], b = base[(2 * i + 1) * 32];
        const float2 c = sigs[i * 32];
        const float lo0 = fabsf(a.z), lo1 = fabsf(a.w), hi0 = 1.0f - lo0, hi1 = 1.0f - lo1;
        const bool rest0 = __float_as_int(a.z) < 0, rest1 = __float_as_int(a.w) < 0;
        t = pack2(a.x, a.y);
        beta = pack2(rest0 ? hi0 : lo0, rest1 ? hi1 : lo1);
        rest = pack2(rest0 ? lo0 : hi0, rest1 ? lo1 : hi1);
        sig = pack2(c.x, c.y);
        x = pack2(b.x, b.y);
        dy = pack2(b.z, b.w);
    }
};

// The backward pass, built like the forward one, from the last tile to the
// first.  The gradient that reaches a piece from behind obeys a recurrence of
// its own, e -> g (dy + e), so a piece has two maps: of the state before it
// (the tile's own comes from the forward pass's checkpoint) and of the
// gradient behind it (exchanged over the cluster).  A map warp computes the
// gates once, keeps what the gradients need of them in shared memory, and
// writes its piece's gradients a tile later, when both ends are known.  The
// sums over tokens stay in registers to the end, and are added over the CTA's
// warps and the cluster's CTAs in order.  Bound like the forward pass: 160 warp
// instructions per token and pair of channels in 63 % of the slots; measured
// (bf16): 1 x 16384 x 4096 273 us, 3.4 TB/s; 8 x 4096 x 1024 184 us.
template <typename T, int STRIPS>
__global__ void __launch_bounds__(kGradThreads, 1) gdn_scan_backward_kernel(const ScanParams p, const ScanGradParams d) {
    constexpr int W = kGradWarps, kPiece = kGradPiece, kRows = kGradRows, kTile = STRIPS * kRows, kSpan = STRIPS * kPiece;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float4 s_ends[2][32];  // the state before the tile, the gradient behind it
    __shared__ __align__(8) uint64_t s_bar[7];
    __shared__ int s_cu[kScanCuMost + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int R = cluster_size(), rank = cluster_rank();
    GradTile<T> vals(smem, lane);
    const Strips<STRIPS> me;
    float4* state_maps = reinterpret_cast<float4*>(smem + kGradTileBytes);  // [2][W][32], and then what precedes
    float4* grad_maps = state_maps + 2 * W * 32;                                 // [2][W][32], and then what follows
    float4* ranks = grad_maps + 2 * W * 32;                                      // [2][R][32]
    float4* cta_sums = ranks + 2 * R * 32;  // [R][32], the first CTA's: others write while it still works
    const int c0 = blockIdx.y * me.kChannels, c = c0 + 2 * me.lane;
    const bool ok0 = c < p.channels, ok1 = c + 1 < p.channels;
    const uint32_t full = tc05::smem_u32(s_bar), ready = full + 16, arrived = full + 32, summed = full + 48;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc05::mbar_init(full + 8 * i, W);
            tc05::mbar_init(ready + 8 * i, 1);
            tc05::mbar_init(arrived + 8 * i, 1);
            tc05::mbar_expect_tx(arrived + 8 * i, R * 512);
        }
        tc05::mbar_init(summed, 1);
        tc05::mbar_expect_tx(summed, R * 512);
        tc05::fence_mbar_init();
    }
    const Offsets offsets = scan_offsets(p, s_cu);
    cluster_arrive();
    const int tokens = static_cast<int>(p.tokens);
    const int tiles = (tokens + kTile - 1) / kTile, steps = (tiles + R - 1) / R;
    scan_empty_sequences(p, d.d_new_state, d.d_state, c0, c0 + me.kChannels, rank * blockDim.x + threadIdx.x, R * blockDim.x);
    cluster_wait();  // every CTA of the cluster runs and has its barriers
    // first token of the CTA's tile of step k; before the first token when there is none left
    auto tile_start = [&](int k) { return (tiles - 1 - (k * R + rank)) * kTile; };

    F2 sum_A = splat2(0.0f), sum_dt = splat2(0.0f);
    bool gave_up = false;
    if (warp == W) {
        F2 carry = splat2(0.0f);
        auto checkpoint = [&](int k) {
            const int t = tile_start(k);
            if (k >= steps || t < 0) return splat2(0.0f);
            const float* ck = p.ckpt + static_cast<int64_t>(t / kScanCkpt) * p.channels;
            return pack2(ok0 ? ck[c] : 0.0f, ok1 ? ck[c + 1] : 0.0f);
        };
        F2 state = checkpoint(0);
        for (int k = 0; k < steps; ++k) {
            const int buf = k & 1, phase = k >> 1 & 1;
            const F2 state_in = state;
            state = checkpoint(k + 1);
            if ((gave_up = !warp_wait(full + 8 * buf, phase))) break;
            // In place: a piece's map makes way for what comes before it (a lane's
            // words are its own).
            auto chain = [&](float4* m, int step) {  // a word every `step`
                constexpr int kAhead = 5;            // maps read together
                static_assert(W % kAhead == 0, "whole batches");
                Map2 all = {splat2(1.0f), splat2(0.0f)};
#pragma unroll
                for (int i = 0; i < STRIPS * W; i += kAhead, m += kAhead * step) {
                    float4 e[kAhead];
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) e[j] = m[j * step];
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        const float2 va = unpack2(all.A), vh = unpack2(all.H);
                        m[j * step] = make_float4(va.x, va.y, vh.x, vh.y);
                        const F2 A = pack2(e[j].x, e[j].y);
                        const float2 r = unpack2(fma2(A, all.H, pack2(e[j].z, e[j].w))), a = unpack2(mul2(all.A, A));
                        all.H = pack2(is_start(e[j].x) ? e[j].z : r.x, is_start(e[j].y) ? e[j].w : r.y);
                        all.A = pack2(is_start(e[j].x) ? e[j].x : a.x, is_start(e[j].y) ? e[j].y : a.y);
                    }
                }
                return all;
            };
            // Pieces in token order are kLanes words apart.  With two strips, the
            // lanes of one chain the states, forward, and those of the other the
            // gradients, backward, in one go.
            float4* first_state = state_maps + buf * W * 32 + me.lane;
            float4* last_grad = grad_maps + buf * W * 32 + (STRIPS * W - 1) * me.kLanes + me.lane;
            const bool states = STRIPS > 1 && me.strip == 0;
            const Map2 all_grad = chain(states ? first_state : last_grad, states ? me.kLanes : -me.kLanes);
            float2 va = unpack2(all_grad.A), vh = unpack2(all_grad.H);
            if (STRIPS > 1) {
                va.x = __shfl_sync(0xffffffffu, va.x, lane | 16), va.y = __shfl_sync(0xffffffffu, va.y, lane | 16);
                vh.x = __shfl_sync(0xffffffffu, vh.x, lane | 16), vh.y = __shfl_sync(0xffffffffu, vh.y, lane | 16);
            }
            const uint32_t to = tc05::smem_u32(ranks + (buf * R + rank) * 32 + lane);
            // A slot is written again two tiles on: by then this CTA has every
            // CTA's map of the tile between, sent after that CTA had read this one's.
            for (int r = 0; r < R; ++r)
                st_cluster_f4(to, arrived + 8 * buf, r, make_float4(va.x, va.y, vh.x, vh.y));
            if (STRIPS == 1) chain(first_state, me.kLanes);
            if ((gave_up = !warp_wait(arrived + 8 * buf, phase))) break;
            if (lane == 0) tc05::mbar_expect_tx(arrived + 8 * buf, R * 512);
            const float4* every = ranks + buf * R * 32 + lane;
            F2 in = carry;
#pragma unroll 4
            for (int r = 0; r < rank; ++r) in = apply_map(every[r * 32], in);
            F2 next = in;
#pragma unroll 4
            for (int r = rank; r < R; ++r) next = apply_map(every[r * 32], next);
            if (__any_sync(0xffffffffu, has_nan(next))) {
                in = fold_select(every, rank, 32, carry);
                next = fold_select(every + rank * 32, R - rank, 32, in);
            }
            const float2 h = unpack2(state_in), e = unpack2(in);
            s_ends[buf][lane] = make_float4(h.x, h.y, e.x, e.y);
            __syncwarp();
            if (lane == 0) tc05::mbar_arrive(ready + 8 * buf);
            carry = next;
        }
    } else {
        const F2 dtb = pack2(ok0 ? p.dt_bias[c] : 0.0f, ok1 ? p.dt_bias[c + 1] : 0.0f);
        const float2 decay = make_float2(ok0 ? expf(p.A_log[c]) : 0.0f, ok1 ? expf(p.A_log[c + 1]) : 0.0f);
        const F2 rate = pack2(-kLog2e * decay.x, -kLog2e * decay.y), minus_decay = pack2(-decay.x, -decay.y);
        const bool all_channels = c0 + me.kChannels <= p.channels;
        const bool whole = p.x_pairs && p.a_pairs && p.b_pairs && d.dy_pairs && all_channels;
        RawPair<T> x[kPiece], a[kPiece], b[kPiece], dy[kPiece];
        auto fetch = [&](int k) {
            const int w0 = k < steps ? tile_start(k) + warp * kSpan : -kTile, t0 = w0 + me.strip * kPiece;
            const T* x0 = static_cast<const T*>(p.x) + c;
            const T* a0 = static_cast<const T*>(p.a) + c;
            const T* b0 = static_cast<const T*>(p.b) + c;
            const T* dy0 = static_cast<const T*>(d.dy) + c;
            if (whole && w0 >= 0 && w0 + kSpan <= tokens) {
#pragma unroll
                for (int j = 0; j < kPiece; ++j) {
                    x[j] = load_raw(row_at<const T>(x0, t0 + j, p.x_stride));
                    a[j] = load_raw(row_at<const T>(a0, t0 + j, p.a_stride));
                    b[j] = load_raw(row_at<const T>(b0, t0 + j, p.b_stride));
                    dy[j] = load_raw(row_at<const T>(dy0, t0 + j, d.dy_stride));
                }
            } else {
#pragma unroll
                for (int j = 0; j < kPiece; ++j) {
                    const bool live = w0 >= 0 && t0 + j < tokens;
                    x[j] = load_raw_part(row_at<const T>(x0, t0 + j, p.x_stride), live && ok0, live && ok1);
                    a[j] = load_raw_part(row_at<const T>(a0, t0 + j, p.a_stride), live && ok0, live && ok1);
                    b[j] = load_raw_part(row_at<const T>(b0, t0 + j, p.b_stride), live && ok0, live && ok1);
                    dy[j] = load_raw_part(row_at<const T>(dy0, t0 + j, d.dy_stride), live && ok0, live && ok1);
                }
            }
        };
        fetch(0);
        Spans span = {0, 0, 0, 0, 0};
        struct {
            uint32_t start, end, covered;
        } done = {0, 0, 0};  // of the tile before
        for (int k = 0; k <= steps; ++k) {
            if (k < steps) {
                const int w0 = tile_start(k) + warp * kSpan, buf = k & 1;
                if (w0 >= 0)
                    token_spans<kSpan>(offsets, tokens, w0, span);
                else
                    span = {0, 0, 0, 0, 0};
                const bool special = (span.start | span.end | (~span.covered & kAllTokens<kSpan>)) != 0;
                F2 z[kPiece], g[kPiece], e[kPiece];
#pragma unroll
                for (int j = 0; j < kPiece; ++j) g[j] = z[j] = add2(raw_to_f2<T>(a[j]), dtb);
                log2_decays(g, e, rate);
                F2 A = splat2(1.0f), H = splat2(0.0f), B = splat2(1.0f), E = splat2(0.0f);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) {
                    // sigmoid(z) = 1 / (1 + e) or e / (1 + e), e = exp(-|z|)
                    const float2 v = unpack2(z[j]), w = unpack2(e[j]);
                    const float2 q = make_float2(rcp_approx(1.0f + w.x), rcp_approx(1.0f + w.y));
                    const F2 sig = pack2(v.x < 0.0f ? w.x * q.x : q.x, v.y < 0.0f ? w.y * q.y : q.y);
                    F2 rest;
                    const F2 beta = sigmoid2(raw_to_f2<T>(b[j]), rest);
                    vals.put(buf * kRows + warp * kPiece + j, g[j], beta, rest, sig, x[j], dy[j]);
                    z[j] = mul2(beta, raw_to_f2<T>(x[j]));
                }
                exp2_decays(g);
                if (!special) {
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) {
                        A = mul2(A, g[j]);
                        H = fma2(g[j], H, z[j]);
                    }
                    B = A;
#pragma unroll
                    for (int j = kPiece - 1; j >= 0; --j) E = mul2(g[j], add2(raw_to_f2<T>(dy[j]), E));
                } else {
                    const int at = me.strip * kPiece;
                    F2 t, beta, rest, sig, xs, dys;
#pragma unroll 1
                    for (int j = 0; j < kPiece; ++j) {
                        vals.get(buf * kRows + warp * kPiece + j, t, beta, rest, sig, xs, dys);
                        const bool covered = span.covered >> (at + j) & 1, start = span.start >> (at + j) & 1;
                        F2 g1[1] = {t};
                        exp2_decays(g1);
                        H = state_of_strips<STRIPS>(offsets, p.state, p.channels, span.start >> j, kPiece, w0 + j, c, me.strip, H);
                        A = start || !covered ? splat2(-0.0f) : mul2(A, g1[0]);
                        H = covered ? fma2(g1[0], H, mul2(beta, xs)) : splat2(0.0f);
                    }
#pragma unroll 1
                    for (int j = kPiece - 1; j >= 0; --j) {
                        vals.get(buf * kRows + warp * kPiece + j, t, beta, rest, sig, xs, dys);
                        const bool covered = span.covered >> (at + j) & 1, end = span.end >> (at + j) & 1;
                        F2 g1[1] = {t};
                        exp2_decays(g1);
                        E = state_of_strips<STRIPS>(offsets, d.d_new_state, p.channels, span.end >> j, kPiece, w0 + j, c, me.strip, E);
                        B = end || !covered ? splat2(-0.0f) : mul2(B, g1[0]);
                        E = covered ? mul2(g1[0], add2(dys, E)) : splat2(0.0f);
                    }
                }
                fetch(k + 1);
                const float2 va = unpack2(A), vh = unpack2(H), vb = unpack2(B), ve = unpack2(E);
                state_maps[(buf * W + warp) * 32 + lane] = make_float4(va.x, va.y, vh.x, vh.y);
                grad_maps[(buf * W + warp) * 32 + lane] = make_float4(vb.x, vb.y, ve.x, ve.y);
                __syncwarp();
                if (lane == 0) tc05::mbar_arrive(full + 8 * buf);
            }
            if (k > 0 && tile_start(k - 1) >= 0) {
                const int buf = (k - 1) & 1, w0 = tile_start(k - 1) + warp * kSpan, t0 = w0 + me.strip * kPiece;
                if ((gave_up = !warp_wait(ready + 8 * buf, (k - 1) >> 1 & 1))) break;
                const float4 ends = s_ends[buf][lane];
                const F2 tile_h = pack2(ends.x, ends.y), tile_e = pack2(ends.z, ends.w);
                const float4 hm = state_maps[(buf * W + warp) * 32 + lane], em = grad_maps[(buf * W + warp) * 32 + lane];
                F2 h = apply_map(hm, tile_h), e = apply_map(em, tile_e);
                if (__any_sync(0xffffffffu, !all_finite(tile_h) || !all_finite(tile_e))) {
                    h = apply_map_start(hm, tile_h);
                    e = apply_map_start(em, tile_e);
                }
                T* dx = row_at<T>(static_cast<T*>(d.dx) + c, t0, d.dx_stride);
                T* da = row_at<T>(static_cast<T*>(d.da) + c, t0, d.da_stride);
                T* db = row_at<T>(static_cast<T*>(d.db) + c, t0, d.db_stride);
                const int row0 = buf * kRows + warp * kPiece;
                // one token's gradients from the state before it; e moves on to the token before
                const auto token = [&](F2 g, F2 before, F2 beta, F2 rest, F2 sig, F2 xs, F2 dys, F2& vx, F2& va, F2& vb) {
                    const F2 G = add2(dys, e);
                    e = mul2(g, G);
                    const F2 dl = mul2(e, before);
                    vx = mul2(G, beta);
                    va = mul2(mul2(dl, minus_decay), sig);
                    vb = mul2(mul2(vx, xs), rest);
                    return dl;
                };
                if ((done.start | done.end) == 0 && done.covered == kAllTokens<kSpan> && all_channels && d.grad_pairs) {
                    F2 g[kPiece], t[kPiece], beta[kPiece], rest[kPiece], sig[kPiece], xs[kPiece], dys[kPiece], before[kPiece];
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) {
                        vals.get(row0 + j, t[j], beta[j], rest[j], sig[j], xs[j], dys[j]);
                        g[j] = t[j];
                    }
                    exp2_decays(g);
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) {
                        before[j] = h;
                        h = fma2(g[j], h, mul2(beta[j], xs[j]));
                    }
#pragma unroll
                    for (int j = kPiece - 1; j >= 0; --j) {
                        F2 vx, va, vb;
                        const F2 dl = token(g[j], before[j], beta[j], rest[j], sig[j], xs[j], dys[j], vx, va, vb);
                        sum_A = fma2(dl, t[j], sum_A);
                        sum_dt = add2(sum_dt, va);
                        store_pair(row_at<T>(dx, j, d.dx_stride), vx, true, true, true);
                        store_pair(row_at<T>(da, j, d.da_stride), va, true, true, true);
                        store_pair(row_at<T>(db, j, d.db_stride), vb, true, true, true);
                    }
                } else {
                    const int at = me.strip * kPiece;
                    F2 before[kPiece], t, beta, rest, sig, xs, dys;
#pragma unroll 1
                    for (int j = 0; j < kPiece; ++j) {
                        vals.get(row0 + j, t, beta, rest, sig, xs, dys);
                        F2 g[1] = {t};
                        exp2_decays(g);
                        h = state_of_strips<STRIPS>(offsets, p.state, p.channels, done.start >> j, kPiece, w0 + j, c, me.strip, h);
                        before[j] = h;
                        h = done.covered >> (at + j) & 1 ? fma2(g[0], h, mul2(beta, xs)) : splat2(0.0f);
                    }
#pragma unroll 1
                    for (int j = kPiece - 1; j >= 0; --j) {
                        vals.get(row0 + j, t, beta, rest, sig, xs, dys);
                        F2 g[1] = {t}, vx, va, vb;
                        exp2_decays(g);
                        e = state_of_strips<STRIPS>(offsets, d.d_new_state, p.channels, done.end >> j, kPiece, w0 + j, c, me.strip, e);
                        const F2 dl = token(g[0], before[j], beta, rest, sig, xs, dys, vx, va, vb);
                        if (done.covered >> (at + j) & 1) {
                            sum_A = fma2(dl, t, sum_A);
                            sum_dt = add2(sum_dt, va);
                        } else {
                            vx = va = vb = e = splat2(0.0f);
                        }
#pragma unroll
                        for (int i = 0; i < STRIPS; ++i)
                            if (done.start >> (i * kPiece + j) & 1)
                                store_state_of_strip(offsets, d.d_state, p.channels, w0 + i * kPiece + j, c, me.strip == i, e);
                        if (t0 + j < tokens) {
                            store_pair(row_at<T>(dx, j, d.dx_stride), vx, d.grad_pairs, ok0, ok1);
                            store_pair(row_at<T>(da, j, d.da_stride), va, d.grad_pairs, ok0, ok1);
                            store_pair(row_at<T>(db, j, d.db_stride), vb, d.grad_pairs, ok0, ok1);
                        }
                    }
                }
            }
            done = {span.start, span.end, span.covered};
        }
    }
    // sums over the CTA's warps, in order, then over the cluster's CTAs
    __syncthreads();
    const float2 va = unpack2(sum_A), vd = unpack2(sum_dt);
    float4 part = make_float4(va.x, va.y, vd.x, vd.y);
    if (STRIPS > 1) {  // the other strip's tokens
        part.x += __shfl_xor_sync(0xffffffffu, part.x, 16);
        part.y += __shfl_xor_sync(0xffffffffu, part.y, 16);
        part.z += __shfl_xor_sync(0xffffffffu, part.z, 16);
        part.w += __shfl_xor_sync(0xffffffffu, part.w, 16);
    }
    float4* sums = state_maps + lane;  // nobody reads the maps any more
    if (warp < W) sums[warp * 32] = part;
    __syncthreads();
    auto add_up = [](const float4* v, int n) {
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int i = 0; i < n; ++i) {
            const float4 e = v[i * 32];
            s.x += e.x, s.y += e.y, s.z += e.z, s.w += e.w;
        }
        return s;
    };
    if (warp == 0) st_cluster_f4(tc05::smem_u32(cta_sums + rank * 32 + lane), summed, 0, add_up(sums, W));
    if (warp == 0 && rank == 0) {
        if (warp_wait(summed, 0)) {
            const float4 s = add_up(cta_sums + lane, R);
            constexpr float kLn2 = 0.6931471805599453f;  // l = ln 2 log2 g
            if (me.strip == 0 && ok0) d.dA_log[c] = s.x * kLn2, d.ddt_bias[c] = s.z;
            if (me.strip == 0 && ok1) d.dA_log[c + 1] = s.y * kLn2, d.ddt_bias[c + 1] = s.w;
        } else {
            gave_up = true;
        }
    }
    leave_cluster(gave_up);
}

// One or a few tokens per sequence, V channels of one sequence per thread (4
// where every row starts on a boundary of four elements, else 1).  All of a
// thread's reads of a token come before its writes, so state may be new_state.
// 256 x 4096 bf16: 3.9 us (16.8 MB: 4.3 TB/s), 8.4 with one channel per thread;
// 8 x 1024: 2.1 us, the launch.
template <typename T, int V>
__global__ void __launch_bounds__(128) gdn_scan_step_kernel(const ScanParams p, int steps) {
    const int c = (blockIdx.x * blockDim.x + threadIdx.x) * V;
    if (c >= p.channels) return;
    constexpr int P = V == 1 ? 1 : V / 2;  // pairs; a lone channel is its pair's first
    using Row = std::conditional_t<V == 1, T, std::conditional_t<sizeof(T) == 4, uint4, uint2>>;
    const auto pairs = [](const Row& r, F2 (&f)[P]) {
        if constexpr (V == 1) {
            f[0] = pack2(to_f32(r), 0.0f);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = load_pair<T>(reinterpret_cast<const T*>(&r) + 2 * i);
        }
    };
    const auto floats = [](const float* q, F2 (&f)[P]) {
        if constexpr (V == 1) {
            f[0] = pack2(*q, 0.0f);
        } else {
            const float4 v = *reinterpret_cast<const float4*>(q);
            f[0] = pack2(v.x, v.y);
            f[1] = pack2(v.z, v.w);
        }
    };
    F2 rate[P], dtb[P];
    floats(p.A_log + c, rate);
    floats(p.dt_bias + c, dtb);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float2 v = unpack2(rate[i]);
        rate[i] = pack2(-kLog2e * expf(v.x), -kLog2e * expf(v.y));
    }
    for (int64_t n = blockIdx.y; n < p.seqs; n += gridDim.y) {
        F2 h[P];
        floats(p.state + n * p.channels + c, h);
        for (int64_t t = n * steps; t < (n + 1) * steps; ++t) {
            const Row rx = *reinterpret_cast<const Row*>(row_at<const T>(p.x, t, p.x_stride) + c);
            const Row ra = *reinterpret_cast<const Row*>(row_at<const T>(p.a, t, p.a_stride) + c);
            const Row rb = *reinterpret_cast<const Row*>(row_at<const T>(p.b, t, p.b_stride) + c);
            F2 x[P], z[P], b[P];
            pairs(rx, x);
            pairs(ra, z);
            pairs(rb, b);
#pragma unroll
            for (int i = 0; i < P; ++i) z[i] = add2(z[i], dtb[i]);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                F2 one[1] = {z[i]};
                decays(one, rate[i]);
                h[i] = fma2(one[0], h[i], mul2(sigmoid2(b[i]), x[i]));
            }
            T* out = row_at<T>(p.out, t, p.out_stride) + c;
            if constexpr (V == 1) {
                *out = from_f32<T>(unpack2(h[0]).x);
            } else {
                T e[V];
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 v = unpack2(h[i]);
                    e[2 * i] = from_f32<T>(v.x);
                    e[2 * i + 1] = from_f32<T>(v.y);
                }
                *reinterpret_cast<Row*>(out) = *reinterpret_cast<const Row*>(e);
            }
        }
        float* ns = p.new_state + n * p.channels + c;
        const float2 v = unpack2(h[0]);
        if constexpr (V == 1) {
            *ns = v.x;
        } else {
            const float2 w = unpack2(h[1]);
            *reinterpret_cast<float4*>(ns) = make_float4(v.x, v.y, w.x, w.y);
        }
    }
}

// `kernel` with gridDim = (cluster, groups of channels); `attr` outlives the launch.
static cudaLaunchConfig_t scan_config(int cluster, unsigned groups, int threads, size_t smem, cudaStream_t s, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, groups);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = cluster;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}
// Clusters of `n` CTAs of `kernel` that run at once (below 1: none, or not
// known), asked once per device and size; the kernel's attributes are set with
// it, for `most` bytes of shared memory.
using ClusterCounts = std::atomic<int>[kScanMaxCluster + 1];
template <typename Kernel>
static int active_clusters(Kernel kernel, int n, int threads, size_t smem, size_t most, ClusterCounts* counts) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    return asked_once(counts[dev][n], [&] {
        cudaLaunchAttribute attr[1];
        const cudaLaunchConfig_t cfg = scan_config(n, 1, threads, smem, nullptr, attr);
        int got = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)) == cudaSuccess &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) == cudaSuccess)
            return got > 0 ? got : -1;
        (void)cudaGetLastError();  // the query's own: the launch has to find none
        return 0;
    });
}

// CTAs per cluster, and the tiles that a CTA then walks one after another.  A
// cluster's CTAs sit in one GPC, so how many clusters run at once depends on
// their size in steps (on a B200 33 clusters of 4, 22 of 6, 15 of 8 or 9); the
// size with the fewest tiles in a row, waves x tiles / size, is taken.  `active`
// gives the clusters that run at once.
struct ClusterShape {
    int size;
    int64_t steps;
};
template <typename Active>
static ClusterShape scan_cluster(int64_t tiles, int64_t groups, Active active) {
    ClusterShape best = {0, INT64_MAX};
    for (int r = 1; r <= kScanMaxCluster && (r == 1 || r <= tiles); ++r) {
        const int64_t n = active(r);
        if (n < 1) continue;
        const int64_t steps = (groups + n - 1) / n * ((tiles + r - 1) / r);
        if (steps < best.steps) best = {r, steps};
    }
    return best;
}

// A kernel with one and with two strips to a warp: `rows` tokens per strip and
// tile, smem(r) bytes in clusters of r.  Two strips of 32 channels make twice
// the groups and half the tiles: better clusters for few channels (1 x 40000 x
// 1024: 16 groups in clusters of 6 fill 96 SMs, 32 in clusters of 4 fill 128; 110
// and 89 us with 15 map warps and shorter gates, 99 with two strips as it is now).
template <typename Smem, typename... Params, typename... Args>
static cudaError_t launch_scan_clusters(void (*one)(Params...), void (*two)(Params...), ClusterCounts (*counts)[64],
                                        int64_t tokens, int rows, int threads, int channels, Smem smem, cudaStream_t s, Args... args) {
    const int64_t groups[2] = {(channels + 63) / 64, (channels + 31) / 32};
    void (*const kernels[2])(Params...) = {one, two};
    ClusterShape shape[2];
    for (int i = 0; i < 2; ++i) {
        const int tile = rows * (i + 1);
        shape[i] = scan_cluster((tokens + tile - 1) / tile, groups[i], [&](int n) {
            return active_clusters(kernels[i], n, threads, smem(n), smem(kScanMaxCluster), counts[i]);
        });
    }
    const int i = shape[1].steps < shape[0].steps ? 1 : 0;
    if (shape[i].size == 0) return cudaErrorInvalidConfiguration;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = scan_config(shape[i].size, static_cast<unsigned>(groups[i]), threads, smem(shape[i].size), s, attr);
    return cudaLaunchKernelEx(&cfg, kernels[i], static_cast<Params>(args)...);
}

template <typename T>
static cudaError_t launch_scan(const ScanParams& p, cudaStream_t s) {
    constexpr int kRows = kScanWarps * kScanPiece<T>;
    static ClusterCounts counts[2][64];
    const auto smem = [](int r) { return (2 * kRows + 2 * kScanWarps + 2 * r) * 32 * sizeof(float4); };
    return launch_scan_clusters(gdn_scan_kernel<T, 1>, gdn_scan_kernel<T, 2>, counts, p.tokens, kRows, kScanThreads, p.channels, smem, s, p);
}

template <typename T>
static cudaError_t launch_scan_backward(const ScanParams& p, const ScanGradParams& d, cudaStream_t s) {
    static ClusterCounts counts[2][64];
    const auto smem = [](int r) { return kGradTileBytes + (2 * 2 * kGradWarps + 3 * r) * 32 * sizeof(float4); };
    return launch_scan_clusters(gdn_scan_backward_kernel<T, 1>, gdn_scan_backward_kernel<T, 2>, counts, p.tokens, kGradRows,
                                kGradThreads, p.channels, smem, s, p, d);
}

template <typename T>
static cudaError_t launch_scan_step(const ScanParams& p, int64_t steps, cudaStream_t s) {
    const auto rows = [](const void* q, uint32_t stride) { return aligned(q, 4 * sizeof(T)) && stride % (4 * sizeof(T)) == 0; };
    const bool vec = p.channels % 4 == 0 && rows(p.x, p.x_stride) && rows(p.a, p.a_stride) && rows(p.b, p.b_stride) &&
                     rows(p.out, p.out_stride) && aligned(p.state, 16) && aligned(p.new_state, 16) && aligned(p.A_log, 16) &&
                     aligned(p.dt_bias, 16);
    const int per_cta = vec ? 512 : 128;
    const dim3 grid((p.channels + per_cta - 1) / per_cta, static_cast<unsigned>(p.seqs < 65535 ? p.seqs : 65535));
    if (vec)
        gdn_scan_step_kernel<T, 4><<<grid, 128, 0, s>>>(p, static_cast<int>(steps));
    else
        gdn_scan_step_kernel<T, 1><<<grid, 128, 0, s>>>(p, static_cast<int>(steps));
    return cudaGetLastError();
}

static bool dtype_ok(int dtype) { return dtype >= GDN_DTYPE_BF16 && dtype <= GDN_DTYPE_F32; }
static uintptr_t dtype_bytes(int dtype) { return dtype == GDN_DTYPE_F32 ? 4 : 2; }

// Elements between tokens: the kernels hold the bytes in 32 bits.
static bool stride_ok(int64_t stride) { return stride >= 0 && stride <= (1 << 29); }

// Every row starts on a boundary of two elements, so a pair is one access.
static bool rows_in_pairs(const void* q, int64_t stride, uintptr_t es) { return aligned(q, 2 * es) && stride % 2 == 0; }

static int64_t checkpoint_rows(int64_t tokens) { return (tokens + kScanCkpt - 1) / kScanCkpt; }

// What the three entry points read.
static Operands scan_inputs(const GdnScanArgs* a, bool step) {
    const int64_t es = static_cast<int64_t>(dtype_bytes(a->dtype)), T = a->total_tokens, N = a->num_seqs, C = a->channels;
    Operands o;
    o.read(a->x, T, a->x_stride * es, C * es);
    o.read(a->a, T, a->a_stride * es, C * es);
    o.read(a->b, T, a->b_stride * es, C * es);
    o.read(a->A_log, 1, 0, C * 4);
    o.read(a->dt_bias, 1, 0, C * 4);
    o.read(a->state, N, C * 4, C * 4);
    if (!step) o.read(a->cu_seqlens, 1, 0, (N + 1) * (a->cu_seqlens_dtype == GDN_SEQLENS_INT64 ? 8 : 4));
    return o;
}

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
    if (!stride_ok(a->x_stride) || !stride_ok(a->a_stride) || !stride_ok(a->b_stride) || !stride_ok(a->output_stride))
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
    p.x_stride = static_cast<uint32_t>(a->x_stride * es);
    p.a_stride = static_cast<uint32_t>(a->a_stride * es);
    p.b_stride = static_cast<uint32_t>(a->b_stride * es);
    p.out_stride = static_cast<uint32_t>(a->output_stride * es);
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
    p.x_pairs = rows_in_pairs(a->x, a->x_stride, es);
    p.a_pairs = rows_in_pairs(a->a, a->a_stride, es);
    p.b_pairs = rows_in_pairs(a->b, a->b_stride, es);
    p.out_pairs = rows_in_pairs(a->output, a->output_stride, es);
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
    Operands o = scan_inputs(a, false);
    const int64_t es = static_cast<int64_t>(dtype_bytes(a->dtype)), C = a->channels;
    o.write(a->output, a->total_tokens, a->output_stride * es, C * es);
    o.write(a->new_state, a->num_seqs, C * 4, C * 4);
    o.write(a->checkpoints, checkpoint_rows(a->total_tokens), C * 4, C * 4);
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    if (a->num_seqs == 0 && a->total_tokens == 0) return GDN_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_scan<float>(p, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_scan<__half>(p, s)
                                                      : launch_scan<__nv_bfloat16>(p, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}

extern "C" int64_t gdn_scan_checkpoint_rows(int64_t total_tokens) {
    return total_tokens < 0 ? 0 : checkpoint_rows(total_tokens);
}

extern "C" int gdn_scan_backward_launch(const GdnScanArgs* a, const GdnScanGradArgs* g, void* stream) {
    if (g == nullptr) return GDN_ERR_NULL_POINTER;
    ScanParams p;
    if (int rc = scan_setup(a, p, false)) return rc;
    if (a->total_tokens > 0 && (!g->d_output || !g->dx || !g->da || !g->db || !a->checkpoints))
        return GDN_ERR_NULL_POINTER;
    if (!g->dA_log || !g->d_dt_bias) return GDN_ERR_NULL_POINTER;
    if (!stride_ok(g->d_output_stride) || !stride_ok(g->dx_stride) || !stride_ok(g->da_stride) || !stride_ok(g->db_stride))
        return GDN_ERR_BAD_SIZE;
    if (a->total_tokens > 1 && (g->d_output_stride < a->channels || g->dx_stride < a->channels ||
                                g->da_stride < a->channels || g->db_stride < a->channels))
        return GDN_ERR_BAD_SIZE;
    const uintptr_t es = dtype_bytes(a->dtype);
    if (!aligned(g->d_output, es) || !aligned(g->dx, es) || !aligned(g->da, es) || !aligned(g->db, es) ||
        !aligned(g->d_new_state, 4) || !aligned(g->d_state, 4) || !aligned(g->dA_log, 4) || !aligned(g->d_dt_bias, 4))
        return GDN_ERR_MISALIGNED;
    Operands o = scan_inputs(a, false);
    const int64_t size = static_cast<int64_t>(es), T = a->total_tokens, N = a->num_seqs, C = a->channels;
    o.read(g->d_output, T, g->d_output_stride * size, C * size);
    o.read(g->d_new_state, N, C * 4, C * 4);
    o.read(a->checkpoints, checkpoint_rows(T), C * 4, C * 4);
    o.write(g->dx, T, g->dx_stride * size, C * size);
    o.write(g->da, T, g->da_stride * size, C * size);
    o.write(g->db, T, g->db_stride * size, C * size);
    o.write(g->dA_log, 1, 0, C * 4);
    o.write(g->d_dt_bias, 1, 0, C * 4);
    o.write(g->d_state, N, C * 4, C * 4);
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    ScanGradParams d;
    d.dy = g->d_output;
    d.dy_stride = static_cast<uint32_t>(g->d_output_stride * es);
    d.dx_stride = static_cast<uint32_t>(g->dx_stride * es);
    d.da_stride = static_cast<uint32_t>(g->da_stride * es);
    d.db_stride = static_cast<uint32_t>(g->db_stride * es);
    d.d_new_state = g->d_new_state;
    d.dx = g->dx;
    d.da = g->da;
    d.db = g->db;
    d.d_state = g->d_state;
    d.dA_log = g->dA_log;
    d.ddt_bias = g->d_dt_bias;
    d.dy_pairs = rows_in_pairs(g->d_output, g->d_output_stride, es);
    d.grad_pairs = rows_in_pairs(g->dx, g->dx_stride, es) && rows_in_pairs(g->da, g->da_stride, es) &&
                   rows_in_pairs(g->db, g->db_stride, es);
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
    Operands o = scan_inputs(a, true);
    const int64_t es = static_cast<int64_t>(dtype_bytes(a->dtype)), C = a->channels;
    o.write(a->output, a->total_tokens, a->output_stride * es, C * es, true);
    o.write(a->new_state, a->num_seqs, C * 4, C * 4, true);
    if (!o.apart()) return GDN_ERR_OVERLAP;
    if (int rc = check_device()) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = a->dtype == GDN_DTYPE_F32   ? launch_scan_step<float>(p, tokens, s)
                          : a->dtype == GDN_DTYPE_F16 ? launch_scan_step<__half>(p, tokens, s)
                                                      : launch_scan_step<__nv_bfloat16>(p, tokens, s);
    return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
}
