// Log-probability (and entropy) of one chosen token per row of logits, and its gradient (gfx950).
//
//   z = x / T,  p = softmax(z),  lp = log p[token],  H = -sum p log p
//   d(g lp + h H) / dx_i = (g ([i == token] - p_i) - h p_i (log p_i + H)) / T
//
// Forward reads the logits once: every thread keeps the running maximum m of what it has read, s = sum exp(z - m) and
// t = sum exp(z - m) (x - m), rescaled when the maximum grows, and these triples are merged over the row's threads and, when
// a row is split, its parts.  lp = (x[token] - m) / T - log s and H = log s - t / (s T).  What backward needs of a row is
// m, log s and H; it reads the logits again and writes the gradient.  All sums are fp32, in a fixed order.
//
// Rows: -inf entries have probability 0; a row with nothing else (m stays at the lowest float, s = 0) has lp = -inf, H = 0
// and a gradient of zeros.  NaN or +inf in a row gives NaN, as softmax does.  A token outside [0, V), or equal to the
// padding value, gives lp = H = 0 and a gradient of zeros, and its logits are not read.
#include "rows.h"
#include <float.h>

#define LP_LOG2E 1.4426950408889634f
#define LP_MAX_GRID (1 << 20)          // workgroups of a launch; each takes every LP_MAX_GRID-th unit of work

struct LogpRows {
    const void* x;
    const int64_t* tokens;
    int64_t rows, inner, ld_inner, ld_outer;     // row r starts at element (r / inner) * ld_outer + (r % inner) * ld_inner
    int64_t ignore;
    int32_t V, parts;                            // parts: workgroups of a row
    int64_t chunk;                               // elements of a part, a multiple of 16 bytes' worth
    float c, inv_t;                              // log2(e) / T, 1 / T
};

template <int DT> __device__ __forceinline__ const typename Elem<DT>::type* logp_row(const LogpRows& P, int64_t row) {
    return (const typename Elem<DT>::type*)P.x + (row / P.inner) * P.ld_outer + (row % P.inner) * P.ld_inner;
}
__device__ __forceinline__ bool logp_live(const LogpRows& P, int64_t token) {
    return token >= 0 && token < P.V && token != P.ignore;
}

// Elements in front of a row's first 16-byte boundary.  Forward, the parts of a row start there and the first one takes these as
// well: pieces that straddle cache lines cost a fifth of the bandwidth (8192 x 50001 bf16: 136 us, aligned 108).  Backward, with
// two pieces a thread, finding the boundary costs more than it gives (253 us, aligned 267).
template <int DT> __device__ __forceinline__ int logp_head(const typename Elem<DT>::type* row, int32_t V) {
    constexpr int N = Elem<DT>::N, SIZE = 16 / N;
    const int n = (N - (int)((uintptr_t)row % 16) / SIZE) % N;
    return n < V ? n : V;
}

// m: maximum, at least the lowest float (so that differences of maxima are numbers); s, t: sums relative to it
struct Mst { float m, s, t; };

__device__ __forceinline__ Mst mst_rescale(Mst a, float m, float c) {
    const float d = a.m - m, f = __builtin_amdgcn_exp2f(d * c);
    // (f = 0: the side has no weight left, while its d may be infinite; a NaN goes on in s)
    return {m, a.s * f, f > 0.f ? f * (a.t + a.s * d) : 0.f};
}
__device__ __forceinline__ Mst mst_merge(Mst a, Mst b, float c) {
    const float m = fmaxf(a.m, b.m);
    a = mst_rescale(a, m, c);
    b = mst_rescale(b, m, c);
    return {m, a.s + b.s, a.t + b.t};
}
template <int W> __device__ __forceinline__ Mst mst_reduce(Mst a, float c) {      // over W lanes of a wave
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1)
        a = mst_merge(a, {__shfl_xor(a.m, d, W), __shfl_xor(a.s, d, W), __shfl_xor(a.t, d, W)}, c);
    return a;
}

template <int CNT, bool ENT> __device__ __forceinline__ void mst_add(Mst& a, const float* f, float c) {
    float vm = a.m;
#pragma unroll
    for (int i = 0; i < CNT; i++) vm = fmaxf(vm, f[i]);
    if (vm > a.m) a = mst_rescale(a, vm, c);
#pragma unroll
    for (int i = 0; i < CNT; i++) {
        const float d = f[i] - a.m, e = __builtin_amdgcn_exp2f(d * c);
        a.s += e;
        if (ENT) a.t = fmaf(e, fmaxf(d, -FLT_MAX), a.t);
    }
}

template <int DT>
__device__ __forceinline__ void logp_finish(const LogpRows& P, int64_t row, int64_t token, Mst a, float* logp, float* entropy,
                                            float4* stats) {
    const float logs = logf(a.s);                            // -inf for a row that nothing is left of
    const bool empty = a.s == 0.f;
    const float xt = elem_get<DT>(logp_row<DT>(P, row) + token);
    const float H = empty ? 0.f : logs - P.inv_t * (a.t / a.s);
    // (in 64 bits: the difference of two floats may be none, and is one again over the temperature)
    logp[row] = empty ? -INFINITY : (float)(((double)xt - (double)a.m) * (double)P.inv_t - (double)logs);
    if (entropy) entropy[row] = H;
    stats[row] = make_float4(a.m, logs, H, 0.f);
}

// G threads a row: 8 to 64 of a wave, 256 / G rows a workgroup; or the whole workgroup (G = 256), for one part of a row.
template <int DT, int G, bool ENT, bool NT>
__global__ __launch_bounds__(256) void logp_forward_kernel(LogpRows P, float* __restrict__ logp, float* __restrict__ entropy,
                                                           float4* __restrict__ stats, float4* __restrict__ partial) {
    typedef typename Elem<DT>::type T;
    constexpr int N = Elem<DT>::N, U = 4, W = G < 64 ? G : 64;
    __shared__ Mst wave[4];
    const int lane = threadIdx.x % G;
    const int64_t units = G == 256 ? P.rows * P.parts : (P.rows + 256 / G - 1) / (256 / G);
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t row = G == 256 ? unit / P.parts : unit * (256 / G) + threadIdx.x / G;
        const int part = G == 256 ? (int)(unit % P.parts) : 0;
        if (row >= P.rows) continue;                         // (G < 256: the last workgroup's unused groups)
        const int64_t token = P.tokens[row];
        if (!logp_live(P, token)) {                          // the same for all threads of the row
            if (lane == 0 && part == 0) {
                logp[row] = 0.f;
                if (entropy) entropy[row] = 0.f;
                stats[row] = make_float4(0.f, -INFINITY, 0.f, 0.f);
            }
            continue;
        }
        const T* x = logp_row<DT>(P, row);
        const int head = logp_head<DT>(x, P.V);
        const int64_t lo = head + part * P.chunk, hi = lo + P.chunk < P.V ? lo + P.chunk : P.V;
        const int64_t nv = hi > lo ? (hi - lo) / N : 0;
        Mst a = {-FLT_MAX, 0.f, 0.f};
        if (part == 0 && lane < head) {
            const float f = elem_get<DT>(x + lane);
            mst_add<1, ENT>(a, &f, P.c);
        }
        int64_t v = lane;
        for (; v + (U - 1) * G < nv; v += U * G) {
            u32x4 r[U];
            float f[U * N];
#pragma unroll
            for (int k = 0; k < U; k++) r[k] = vec_load_as<DT, NT>(x + lo + (v + k * G) * N);
#pragma unroll
            for (int k = 0; k < U * N; k++) f[k] = vec_get<DT>(r[k / N], k % N);
            mst_add<U * N, ENT>(a, f, P.c);
        }
        for (; v < nv; v += G) {
            const u32x4 r = vec_load_as<DT, NT>(x + lo + v * N);
            float f[N];
#pragma unroll
            for (int k = 0; k < N; k++) f[k] = vec_get<DT>(r, k);
            mst_add<N, ENT>(a, f, P.c);
        }
        for (int64_t i = lo + nv * N + lane; i < hi; i += G) {
            const float f = elem_get<DT>(x + i);
            mst_add<1, ENT>(a, &f, P.c);
        }
        a = mst_reduce<W>(a, P.c);
        if (G == 256) {
            if (threadIdx.x % 64 == 0) wave[threadIdx.x / 64] = a;
            __syncthreads();
            a = mst_merge(mst_merge(wave[0], wave[1], P.c), mst_merge(wave[2], wave[3], P.c), P.c);
            __syncthreads();                                 // (the next unit writes `wave` again)
        }
        if (lane == 0) {
            if (G == 256 && P.parts > 1) partial[unit] = make_float4(a.m, a.s, a.t, 0.f);
            else logp_finish<DT>(P, row, token, a, logp, entropy, stats);
        }
    }
}

// one wave a row: merges the row's parts
template <int DT>
__global__ __launch_bounds__(64) void logp_merge_kernel(LogpRows P, float* __restrict__ logp, float* __restrict__ entropy,
                                                        float4* __restrict__ stats, const float4* __restrict__ partial) {
    const int64_t row = blockIdx.x;
    const int64_t token = P.tokens[row];
    if (!logp_live(P, token)) return;                        // (written by the forward kernel)
    Mst a = {-FLT_MAX, 0.f, 0.f};
    for (int k = threadIdx.x; k < P.parts; k += 64) {
        const float4 q = partial[row * P.parts + k];
        a = mst_merge(a, {q.x, q.y, q.z}, P.c);
    }
    a = mst_reduce<64>(a, P.c);
    if (threadIdx.x == 0) logp_finish<DT>(P, row, token, a, logp, entropy, stats);
}

// dx_i = p_i (a + b (x_i - m)) (+ g / T at the token), p_i = 2^((x_i - m) c - log2 s);
// a = -(g + h (H - log s)) / T, b = -h / T^2
template <int DT, int G, bool ENT, bool NT>
__global__ __launch_bounds__(256) void logp_backward_kernel(LogpRows P, const float4* __restrict__ stats,
                                                            const float* __restrict__ gp, const float* __restrict__ hp,
                                                            typename Elem<DT>::type* __restrict__ dx) {
    typedef typename Elem<DT>::type T;
    constexpr int N = Elem<DT>::N;
    const int lane = threadIdx.x % G;
    const int64_t units = G == 256 ? P.rows * P.parts : (P.rows + 256 / G - 1) / (256 / G);
    for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int64_t row = G == 256 ? unit / P.parts : unit * (256 / G) + threadIdx.x / G;
        const int part = G == 256 ? (int)(unit % P.parts) : 0;
        if (row >= P.rows) continue;
        const int64_t token = P.tokens[row];
        const T* x = logp_row<DT>(P, row);
        T* out = dx + row * P.V;
        const int64_t lo = part * P.chunk, hi = lo + P.chunk < P.V ? lo + P.chunk : P.V;
        const int64_t nv = (hi - lo) / N;
        const float4 st = stats[row];
        if (!logp_live(P, token) || st.y == -INFINITY) {     // padding, or a row that nothing is left of
            const u32x4 zero = {0, 0, 0, 0};
            for (int64_t v = lane; v < nv; v += G) vec_store_as<DT, NT>(out + lo + v * N, zero);
            for (int64_t i = lo + nv * N + lane; i < hi; i += G) elem_put<DT>(out + i, 0.f);
            continue;
        }
        const float g = gp ? gp[row] : 0.f, h = ENT ? hp[row] : 0.f;
        const float m = st.x, l2 = st.y * LP_LOG2E, gt = g * P.inv_t;
        const float a = ENT ? -P.inv_t * (g + h * (st.z - st.y)) : -gt, b = -h * P.inv_t * P.inv_t;
        auto grad = [&](float xv) {
            const float d = xv - m, p = __builtin_amdgcn_exp2f(fmaf(d, P.c, -l2));
            if (!ENT) return p * a;
            return p == 0.f ? 0.f : p * fmaf(b, d, a);       // (p = 0: d may be infinite)
        };
        for (int64_t v = lane; v < nv; v += G) {
            const int64_t i = lo + v * N;
            const u32x4 r = vec_load_as<DT, NT>(x + i);
            float f[N];
#pragma unroll
            for (int k = 0; k < N; k++) f[k] = grad(vec_get<DT>(r, k)) + (i + k == token ? gt : 0.f);
            vec_store_as<DT, NT>(out + i, vec_make<DT>(f));
        }
        for (int64_t i = lo + nv * N + lane; i < hi; i += G)
            elem_put<DT>(out + i, grad(elem_get<DT>(x + i)) + (i == token ? gt : 0.f));
    }
}

// Threads of a row: as many lanes as leave each about two 16-byte pieces, the whole workgroup above 512 pieces.
static int logp_group(int32_t V, int32_t dtype) {
    const int64_t vecs = ((int64_t)V * (dtype == VQA_F32 ? 4 : 2) + 15) / 16;
    return vecs <= 16 ? 8 : vecs <= 32 ? 16 : vecs <= 64 ? 32 : vecs <= 512 ? 64 : 256;
}
// Forward: rows are split while the launch has fewer than 1024 workgroups (four per CU) and a part keeps a 16-byte piece
// per thread.
static int64_t logp_forward_chunk(int64_t rows, int32_t V, int32_t dtype) {
    if (logp_group(V, dtype) < 256) return V;
    const int64_t piece = 256 * (dtype == VQA_F32 ? 4 : 8), pieces = (V + piece - 1) / piece;
    const int64_t parts = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    return parts >= pieces ? piece : (pieces + parts - 1) / parts * piece;
}

extern "C" int64_t vqa_token_logp_workspace(int64_t rows, int32_t V, int32_t dtype) {
    if (rows <= 0 || V <= 0 || !rows_dtype_ok(dtype)) return 0;
    const int64_t chunk = logp_forward_chunk(rows, V, dtype), parts = (V + chunk - 1) / chunk;
    return parts > 1 ? 4 * rows * parts : 0;
}

static int logp_args(LogpRows& P, const char* who, const void* x, int64_t inner, int64_t ld_inner, int64_t ld_outer,
                     const int64_t* tokens, int64_t rows, int32_t V, int32_t dtype, float temperature, int64_t ignore,
                     const void* stats) {
    if (!x || !tokens || !stats || rows < 0 || V <= 0 || inner <= 0 || !rows_dtype_ok(dtype) || !(temperature > 0.f) ||
        !(temperature < INFINITY) || (uintptr_t)x % (dtype == VQA_F32 ? 4 : 2) || (uintptr_t)tokens % 8 ||
        (uintptr_t)stats % 16) {
        vqa_set_error(std::string(who) + ": bad argument");
        return VQA_EINVAL;
    }
    P.x = x;
    P.tokens = tokens;
    P.rows = rows;
    P.inner = inner;
    P.ld_inner = ld_inner;
    P.ld_outer = ld_outer;
    P.ignore = ignore;
    P.V = V;
    P.inv_t = (float)(1.0 / (double)temperature);
    P.c = (float)(1.4426950408889634 / (double)temperature);
    return VQA_OK;
}

// Whether the logits are too many to stay in the last-level cache (256 MiB) from one pass to the next: then they are read,
// and the gradient is written, past it (4096 x 131072 bf16: forward 162 -> 148 us, backward 312 -> 302; 2048 x 32768 fp16, which
// stay: backward 36 -> 40).
static bool logp_streams(const LogpRows& P, int dtype) {
    return (double)P.rows * P.V * (dtype == VQA_F32 ? 4 : 2) > 256.0 * (1 << 20);
}
template <int DT, int G, bool NT>
static void logp_forward_as(const LogpRows& P, dim3 grid, float* logp, float* entropy, float4* stats, float4* ws, hipStream_t s) {
    if (entropy) hipLaunchKernelGGL((logp_forward_kernel<DT, G, true, NT>), grid, dim3(256), 0, s, P, logp, entropy, stats, ws);
    else hipLaunchKernelGGL((logp_forward_kernel<DT, G, false, NT>), grid, dim3(256), 0, s, P, logp, entropy, stats, ws);
}
template <int DT, int G>
static void logp_forward_launch(const LogpRows& P, dim3 grid, float* logp, float* entropy, float4* stats, float4* ws, hipStream_t s) {
    if (G == 256 && logp_streams(P, DT)) logp_forward_as<DT, G, G == 256>(P, grid, logp, entropy, stats, ws, s);
    else logp_forward_as<DT, G, false>(P, grid, logp, entropy, stats, ws, s);
}
template <int DT, int G, bool NT>
static void logp_backward_as(const LogpRows& P, dim3 grid, const float4* stats, const float* g, const float* h, void* dx,
                             hipStream_t s) {
    typedef typename Elem<DT>::type T;
    if (h) hipLaunchKernelGGL((logp_backward_kernel<DT, G, true, NT>), grid, dim3(256), 0, s, P, stats, g, h, (T*)dx);
    else hipLaunchKernelGGL((logp_backward_kernel<DT, G, false, NT>), grid, dim3(256), 0, s, P, stats, g, h, (T*)dx);
}
template <int DT, int G>
static void logp_backward_launch(const LogpRows& P, dim3 grid, const float4* stats, const float* g, const float* h, void* dx,
                                 hipStream_t s) {
    if (G == 256 && logp_streams(P, DT)) logp_backward_as<DT, G, G == 256>(P, grid, stats, g, h, dx, s);
    else logp_backward_as<DT, G, false>(P, grid, stats, g, h, dx, s);
}
#define LOGP_GROUPS(FN, DT, ...)                             \
    switch (G) {                                             \
        case 8: FN<DT, 8>(__VA_ARGS__); break;               \
        case 16: FN<DT, 16>(__VA_ARGS__); break;             \
        case 32: FN<DT, 32>(__VA_ARGS__); break;             \
        case 64: FN<DT, 64>(__VA_ARGS__); break;             \
        default: FN<DT, 256>(__VA_ARGS__);                   \
    }
#define LOGP_DISPATCH(FN, ...)                                        \
    if (dtype == VQA_BF16) { LOGP_GROUPS(FN, VQA_BF16, __VA_ARGS__) } \
    else if (dtype == VQA_F16) { LOGP_GROUPS(FN, VQA_F16, __VA_ARGS__) } \
    else { LOGP_GROUPS(FN, VQA_F32, __VA_ARGS__) }

static dim3 logp_grid(const LogpRows& P, int G) {
    const int64_t units = G == 256 ? P.rows * P.parts : (P.rows + 256 / G - 1) / (256 / G);
    return dim3((unsigned)(units < LP_MAX_GRID ? units : LP_MAX_GRID));
}

extern "C" int vqa_token_logp(const void* x, int64_t inner, int64_t ld_inner, int64_t ld_outer, const int64_t* tokens,
                              float* logp, float* entropy, float* stats, float* workspace, int64_t rows, int32_t V,
                              int32_t dtype, float temperature, int64_t ignore, void* stream) {
    LogpRows P;
    if (int rc = logp_args(P, "vqa_token_logp", x, inner, ld_inner, ld_outer, tokens, rows, V, dtype, temperature, ignore, stats))
        return rc;
    P.chunk = logp_forward_chunk(rows, V, dtype);
    P.parts = (int32_t)((V + P.chunk - 1) / P.chunk);
    if (!logp || (P.parts > 1 && (!workspace || (uintptr_t)workspace % 16))) {
        vqa_set_error("vqa_token_logp: bad argument");
        return VQA_EINVAL;
    }
    if (rows == 0) return VQA_OK;
    const int G = logp_group(V, dtype);
    const dim3 grid = logp_grid(P, G);
    LOGP_DISPATCH(logp_forward_launch, P, grid, logp, entropy, (float4*)stats, (float4*)workspace, (hipStream_t)stream)
    ROWS_CHECK_LAUNCH("vqa_token_logp");
    if (P.parts > 1) {                                       // (then there are fewer than 1024 rows)
#define MERGE(DT)                                                                                                  \
    hipLaunchKernelGGL(logp_merge_kernel<DT>, dim3((unsigned)rows), dim3(64), 0, (hipStream_t)stream, P, logp,     \
                       entropy, (float4*)stats, (const float4*)workspace)
        if (dtype == VQA_BF16) MERGE(VQA_BF16);
        else if (dtype == VQA_F16) MERGE(VQA_F16);
        else MERGE(VQA_F32);
#undef MERGE
        ROWS_CHECK_LAUNCH("vqa_token_logp");
    }
    return VQA_OK;
}

extern "C" int vqa_token_logp_backward(const void* x, int64_t inner, int64_t ld_inner, int64_t ld_outer, const int64_t* tokens,
                                       const float* stats, const float* g, const float* h, void* dx, int64_t rows, int32_t V,
                                       int32_t dtype, float temperature, int64_t ignore, void* stream) {
    LogpRows P;
    if (int rc = logp_args(P, "vqa_token_logp_backward", x, inner, ld_inner, ld_outer, tokens, rows, V, dtype, temperature,
                           ignore, stats))
        return rc;
    if (!dx || (uintptr_t)dx % (dtype == VQA_F32 ? 4 : 2)) {
        vqa_set_error("vqa_token_logp_backward: bad argument");
        return VQA_EINVAL;
    }
    if (rows == 0) return VQA_OK;
    const int G = logp_group(V, dtype);
    // a workgroup's part of a long row: two 16-byte pieces a thread (with four, 4096 x 131072 bf16 took 340 us, with two 312)
    P.chunk = G == 256 ? 2 * 256 * (dtype == VQA_F32 ? 4 : 8) : V;
    P.parts = (int32_t)((V + P.chunk - 1) / P.chunk);
    const dim3 grid = logp_grid(P, G);
    LOGP_DISPATCH(logp_backward_launch, P, grid, (const float4*)stats, g, h, dx, (hipStream_t)stream)
    ROWS_CHECK_LAUNCH("vqa_token_logp_backward");
    return VQA_OK;
}
