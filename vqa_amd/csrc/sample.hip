// One token per row of logits, drawn with given uniform numbers under temperature, top-k, top-p and min-p (gfx950).
//
// The tokens of a row stand in descending order of their logits, equal logits by index; token i weighs
// w_i = exp((x_i - max) / T).  top-k, min-p and top-p each keep a prefix of that order (top_k tokens; w >= min_p; the tokens
// whose exclusive cumulative weight is below top_p times the weight of what the other two keep), so all together do.  The
// answer is the first token whose inclusive cumulative weight exceeds u times the kept weight.
//
// Nothing is sorted.  A weight is an integer, w rounded to a multiple of 2^-s with V 2^s < 2^63, and a function of the logit
// alone: sums are exact and the same in any order, atomics included.  Each of the three questions - the k-th token, the last
// token of the nucleus, the drawn one - asks which token of the order holds place t, counted in tokens or in weight; a
// radix search over order-preserving integer keys answers it: a histogram of the keys' leading bits (tokens and weight per
// bin, in LDS), the bin that holds t, a histogram of the next bits of that bin's keys, and so on to a single key; equal keys
// weigh the same, so the place among them is a division.
//
// exp is evaluated in 64 bits: a draw compares sums of up to V weights with u times their sum, and with fp32 exponentials
// (2^-22) one row in ten of a flat distribution over 10^5 tokens would get a neighbouring token.
#include "rows.h"

struct SampleArgs {
    const void* x;
    int64_t ld, rows;
    const float* u;
    const float* temperature;      // per row, or null: the scalar
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    double temperature_s, top_p_s, min_p_s;
    int32_t top_k_s, V, shift;     // shift: s
    int64_t* token;
    int64_t ld_token;
    float* logp;                   // or null
};

// Order-preserving keys.  Keys up to MASKED stand for -inf and NaN: tokens that are never drawn.  -0 and +0 are equal.
template <int DT> struct Keys {
    static constexpr int BITS = 16;
    static constexpr uint32_t INF = DT == VQA_BF16 ? 0x7F80u : 0x7C00u;
    static constexpr uint32_t MASKED = 0x7FFFu - INF, TOP = 0x8000u | INF;
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        const uint32_t a = u & 0x7FFFu;
        const uint32_t k = (u & 0x8000u) && a ? 0x7FFFu - a : 0x8000u | a;
        return a > INF ? 0 : k;
    }
    static __device__ __forceinline__ double value(uint32_t k) {
        const uint16_t u = (uint16_t)(k & 0x8000u ? k & 0x7FFFu : 0xFFFFu - k);
        if constexpr (DT == VQA_BF16) return (double)bf2f(u);
        else return (double)(float)__builtin_bit_cast(_Float16, u);
    }
};
template <> struct Keys<VQA_F32> {
    static constexpr int BITS = 32;
    static constexpr uint32_t INF = 0x7F800000u, MASKED = 0x7FFFFFFFu - INF, TOP = 0x80000000u | INF;
    static __device__ __forceinline__ uint32_t of(uint32_t u) {
        const uint32_t a = u & 0x7FFFFFFFu;
        const uint32_t k = (u >> 31) && a ? 0x7FFFFFFFu - a : 0x80000000u | a;
        return a > INF ? 0 : k;
    }
    static __device__ __forceinline__ double value(uint32_t k) {
        return (double)__uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : 0xFFFFFFFFu - k);
    }
};
template <int DT> __device__ __forceinline__ uint32_t vec_raw(u32x4 v, int i) {
    if constexpr (DT == VQA_F32) return v[i];
    else return (i & 1) ? v[i >> 1] >> 16 : v[i >> 1] & 0xFFFFu;
}
template <int DT> __device__ __forceinline__ uint32_t key_at(const typename Elem<DT>::type* x, int64_t i) {
    if constexpr (DT == VQA_F32) return Keys<DT>::of(__float_as_uint(x[i]));
    else return Keys<DT>::of(x[i]);
}

// What a row's weights are made of.
template <int DT> struct Weights {
    uint32_t top;                  // the largest key
    double max, inv_t, min_z;      // min_z: log(min_p)
    double magic;                  // 2^(52 - s): w + magic holds w 2^s in its last bits
    __device__ __forceinline__ double z(uint32_t k) const {
        if (top == Keys<DT>::TOP) return k == top ? 0.0 : -INFINITY;         // +inf takes all the weight
        return (Keys<DT>::value(k) - max) * inv_t;
    }
    __device__ __forceinline__ uint64_t of_z(double zz) const {
        return (uint64_t)(__double_as_longlong(exp(zz) + magic) - __double_as_longlong(magic));
    }
    __device__ __forceinline__ uint64_t of(uint32_t k) const { return of_z(z(k)); }
};

struct RowParams { double t, top_p, min_p, u; int32_t k; bool greedy; };
__device__ __forceinline__ RowParams row_params(const SampleArgs& P, int64_t row) {
    RowParams r;
    r.t = P.temperature ? (double)P.temperature[row] : P.temperature_s;
    r.top_p = P.top_p ? (double)P.top_p[row] : P.top_p_s;
    r.min_p = P.min_p ? (double)P.min_p[row] : P.min_p_s;
    r.k = P.top_k ? P.top_k[row] : P.top_k_s;
    r.u = (double)P.u[row];
    r.greedy = !(r.t > 0.0);
    return r;
}
template <int DT> __device__ __forceinline__ Weights<DT> row_weights(const RowParams& r, uint32_t top, int shift) {
    Weights<DT> w;
    w.top = top;
    w.max = Keys<DT>::value(top);
    w.inv_t = 1.0 / r.t;
    w.min_z = r.min_p > 0.0 ? log(r.min_p < 1.0 ? r.min_p : 1.0) : -INFINITY;
    w.magic = __longlong_as_double((long long)(1023 + 52 - shift) << 52);
    return w;
}
// the first place that the nucleus does not hold, in weight: places below it are kept (at least one is)
__device__ __forceinline__ uint64_t nucleus_end(double top_p, uint64_t total) {
    if (!(top_p > 0.0)) return 1;
    const double e = ceil(top_p * (double)total);
    return e < 1.0 ? 1 : e < (double)total ? (uint64_t)e : total;
}
__device__ __forceinline__ uint64_t drawn_place(double u, uint64_t total) {
    const double t = u * (double)total;
    if (!(t > 0.0)) return 0;
    return t < (double)total && (uint64_t)t < total ? (uint64_t)t : total - 1;
}
template <int DT>
__device__ __forceinline__ void sample_put(const SampleArgs& P, int64_t row, int64_t token, double logp) {
    P.token[row * P.ld_token] = token;
    if (P.logp) P.logp[row] = (float)logp;
}

// ------------------------------------------------------------------------------------------------------------------------
// V <= 64: one wave a row, one token a lane.  A lane adds up what stands before its token by looking at every other one.
template <int DT> __global__ __launch_bounds__(256) void sample_wave_kernel(SampleArgs P) {
    typedef typename Elem<DT>::type T;
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < P.rows; row += (int64_t)gridDim.x * 4) {
        const T* x = (const T*)P.x + row * P.ld;
        const uint32_t key = lane < P.V ? key_at<DT>(x, lane) : 0;
        uint32_t top = key;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if (top <= Keys<DT>::MASKED) {
            if (lane == 0) sample_put<DT>(P, row, -1, -INFINITY);
            continue;
        }
        const RowParams r = row_params(P, row);
        if (r.greedy) {
            const uint64_t m = __ballot(key == top);
            if (lane == 0) sample_put<DT>(P, row, __ffsll((unsigned long long)m) - 1, 0.0);
            continue;
        }
        const Weights<DT> W = row_weights<DT>(r, top, P.shift);
        const double z = key > Keys<DT>::MASKED ? W.z(key) : -INFINITY;
        const bool in = key > Keys<DT>::MASKED && z >= W.min_z;
        const uint64_t w = in ? W.of_z(z) : 0;
        int before = 0;
        uint64_t mass = 0;                                   // (of what stands before; tokens that are out weigh nothing)
        for (int l = 0; l < P.V; l++) {
            const uint32_t kl = __builtin_amdgcn_readlane(key, l);
            const uint64_t wl = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)w, l) |
                                ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(w >> 32), l) << 32);
            if (kl > key || (kl == key && l < lane)) {
                before++;
                mass += wl;
            }
        }
        auto sum = [](uint64_t v) {
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, d);
            return v;
        };
        const bool kept = in && (r.k <= 0 || before < r.k);
        uint64_t total = sum(kept ? w : 0);
        if (r.top_p < 1.0 || r.top_p != r.top_p) {
            const uint64_t end = nucleus_end(r.top_p, total);
            total = sum(kept && mass < end ? w : 0);
        }
        const uint64_t t = drawn_place(r.u, total);
        const uint64_t m = __ballot(kept && mass <= t && t < mass + w);      // exactly one lane
        const int at = __ffsll((unsigned long long)m) - 1;
        if (lane == at) sample_put<DT>(P, row, lane, z - log((double)total) + (double)P.shift * 0.6931471805599453);
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// Any V: a workgroup of BT threads a row.
#define SAMPLE_BINS 2048

struct Hist {
    uint32_t cnt[SAMPLE_BINS];
    unsigned long long mass[SAMPLE_BINS];
};
struct Place {                     // the key that holds a place of the order
    uint32_t key;
    uint64_t cnt_above, mass_above;      // tokens and weight in front of the first token with that key
};
struct SampleShared {
    Hist h1, h2;
    unsigned long long scan_c[16], scan_m[16];
    uint32_t red[16];
    uint32_t bin;
    unsigned long long cnt_above, mass_above;
    int64_t found;
};

template <int BT> struct Row {
    // the bin of `h` (of `bins` ones) that holds place t, from the top, with c / m in front of the highest bin; all threads
    static __device__ void find_bin(SampleShared& S, const Hist& h, int bins, bool by_mass, uint64_t t, uint64_t c, uint64_t m) {
        constexpr int WAVES = BT / 64;
        const int tid = threadIdx.x, per = (bins + BT - 1) / BT;
        uint64_t sc = 0, sm = 0;
        for (int r = 0; r < per; r++) {
            const int b = bins - 1 - (tid * per + r);
            if (b >= 0) {
                sc += h.cnt[b];
                sm += h.mass[b];
            }
        }
        uint64_t ic = sc, im = sm;                           // inclusive over the wave
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t oc = __shfl_up((unsigned long long)ic, d), om = __shfl_up((unsigned long long)im, d);
            if ((tid & 63) >= d) {
                ic += oc;
                im += om;
            }
        }
        if ((tid & 63) == 63) {
            S.scan_c[tid >> 6] = ic;
            S.scan_m[tid >> 6] = im;
        }
        __syncthreads();
        c += ic - sc;
        m += im - sm;
        for (int w = 0; w < WAVES; w++)
            if (w < (tid >> 6)) {
                c += S.scan_c[w];
                m += S.scan_m[w];
            }
        const uint64_t lo = by_mass ? m : c, hi = lo + (by_mass ? sm : sc);
        if (lo <= t && t < hi) {                             // exactly one thread
            for (int r = 0; r < per; r++) {
                const int b = bins - 1 - (tid * per + r);
                if (b < 0) break;
                const uint64_t hc = h.cnt[b], hm = h.mass[b];
                if (t < (by_mass ? m + hm : c + hc)) {
                    S.bin = (uint32_t)b;
                    S.cnt_above = c;
                    S.mass_above = m;
                    break;
                }
                c += hc;
                m += hm;
            }
        }
        __syncthreads();
    }
    static __device__ void clear(Hist& h, int bins) {
        for (int b = threadIdx.x; b < bins; b += BT) {
            h.cnt[b] = 0;
            h.mass[b] = 0;
        }
    }
    template <int DT, typename F> static __device__ __forceinline__ void each(const typename Elem<DT>::type* x, int V, F f) {
        constexpr int N = Elem<DT>::N;
        const int nv = V / N;
        for (int v = threadIdx.x; v < nv; v += BT) {
            const u32x4 r = vec_load<DT>(x + (int64_t)v * N);
#pragma unroll
            for (int k = 0; k < N; k++) f(Keys<DT>::of(vec_raw<DT>(r, k)), v * N + k);
        }
        for (int i = nv * N + threadIdx.x; i < V; i += BT) f(key_at<DT>(x, i), i);
    }
    // histogram of (key >> shift) & (bins - 1) over the tokens that pass min-p and whose key >> up is `prefix`
    template <int DT>
    static __device__ void count(Hist& h, const typename Elem<DT>::type* x, int V, const Weights<DT>& W, int shift, int bins,
                                 int up, uint32_t prefix) {
        each<DT>(x, V, [&](uint32_t key, int) {
            if (key <= Keys<DT>::MASKED || (up < 32 && (key >> up) != prefix)) return;
            const double z = W.z(key);
            if (!(z >= W.min_z)) return;
            const uint32_t b = (key >> shift) & (uint32_t)(bins - 1);
            atomicAdd(&h.cnt[b], 1u);
            const uint64_t w = W.of_z(z);
            if (w) atomicAdd(&h.mass[b], (unsigned long long)w);
        });
    }
    template <int DT>
    static __device__ Place find(SampleShared& S, const typename Elem<DT>::type* x, int V, const Weights<DT>& W, bool by_mass, uint64_t t) {
        constexpr int B = Keys<DT>::BITS;
        Place p;
        find_bin(S, S.h1, SAMPLE_BINS, by_mass, t, 0, 0);
        uint32_t prefix = S.bin;
        int low = B - 11;                                    // bits that are still open
        while (low > 0) {
            const int bits = low > 11 ? 11 : low, bins = 1 << bits;
            const uint64_t c = S.cnt_above, m = S.mass_above;
            clear(S.h2, bins);
            __syncthreads();
            count<DT>(S.h2, x, V, W, low - bits, bins, low, prefix);
            __syncthreads();
            find_bin(S, S.h2, bins, by_mass, t, c, m);
            prefix = (prefix << bits) | S.bin;
            low -= bits;
        }
        p.key = prefix;
        p.cnt_above = S.cnt_above;
        p.mass_above = S.mass_above;
        __syncthreads();
        return p;
    }
    // index of the (j + 1)-th token with this key: every wave counts a contiguous piece of the row, then the right one
    // looks closer
    template <int DT>
    static __device__ int64_t locate(SampleShared& S, const typename Elem<DT>::type* x, int V, uint32_t key, uint64_t j) {
        constexpr int WAVES = BT / 64;
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const int piece = ((V + WAVES - 1) / WAVES + 63) / 64 * 64;
        const int64_t lo = (int64_t)wave * piece, hi = lo + piece < V ? lo + piece : V;
        uint32_t n = 0;
        for (int64_t i = lo + lane; i < hi; i += 64) n += key_at<DT>(x, i) == key;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) n += __shfl_xor((int)n, d);
        if (lane == 0) S.red[wave] = n;
        __syncthreads();
        uint64_t before = 0;
        for (int w = 0; w < wave; w++) before += S.red[w];
        if (before <= j && j < before + n) {
            for (int64_t i = lo + lane; i - lane < hi; i += 64) {
                uint64_t m = __ballot(i < hi && key_at<DT>(x, i) == key);
                const uint64_t c = __popcll((unsigned long long)m);
                if (j < before + c) {
                    for (uint64_t skip = j - before; skip > 0; skip--) m &= m - 1;
                    if (lane == 0) S.found = i + __ffsll((unsigned long long)m) - 1;
                    break;
                }
                before += c;
            }
        }
        __syncthreads();
        return S.found;
    }
};

template <int DT, int BT> __global__ __launch_bounds__(BT) void sample_row_kernel(SampleArgs P) {
    typedef typename Elem<DT>::type T;
    typedef Row<BT> R;
    __shared__ SampleShared S;
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x) {
        const T* x = (const T*)P.x + row * P.ld;
        uint32_t top = 0;
        R::template each<DT>(x, P.V, [&](uint32_t key, int) { top = max(top, key); });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        __syncthreads();                                     // (the previous row's use of S is over)
        if ((tid & 63) == 0) S.red[tid >> 6] = top;
        R::clear(S.h1, SAMPLE_BINS);
        __syncthreads();
        for (int w = 0; w < BT / 64; w++) top = max(top, S.red[w]);
        __syncthreads();
        if (top <= Keys<DT>::MASKED) {
            if (tid == 0) sample_put<DT>(P, row, -1, -INFINITY);
            continue;
        }
        const RowParams r = row_params(P, row);
        if (r.greedy) {
            const int64_t at = R::template locate<DT>(S, x, P.V, top, 0);
            if (tid == 0) sample_put<DT>(P, row, at, 0.0);
            continue;
        }
        const Weights<DT> W = row_weights<DT>(r, top, P.shift);
        R::template count<DT>(S.h1, x, P.V, W, Keys<DT>::BITS - 11, SAMPLE_BINS, 32, 0);
        __syncthreads();
        uint64_t n = 0, total = 0;
        for (int b = tid & 63; b < SAMPLE_BINS; b += 64) {   // (every wave for itself)
            n += S.h1.cnt[b];
            total += S.h1.mass[b];
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            n += __shfl_xor((unsigned long long)n, d);
            total += __shfl_xor((unsigned long long)total, d);
        }
        if (r.k > 0 && (uint64_t)r.k < n) {
            const Place p = R::template find<DT>(S, x, P.V, W, false, (uint64_t)r.k - 1);
            total = p.mass_above + ((uint64_t)r.k - p.cnt_above) * W.of(p.key);
        }
        if (r.top_p < 1.0 || r.top_p != r.top_p) {
            const uint64_t last = nucleus_end(r.top_p, total) - 1;
            const Place p = R::template find<DT>(S, x, P.V, W, true, last);
            const uint64_t w = W.of(p.key);
            total = p.mass_above + ((last - p.mass_above) / w + 1) * w;
        }
        const uint64_t t = drawn_place(r.u, total);
        const Place p = R::template find<DT>(S, x, P.V, W, true, t);
        const int64_t at = R::template locate<DT>(S, x, P.V, p.key, (t - p.mass_above) / W.of(p.key));
        if (tid == 0) sample_put<DT>(P, row, at, W.z(p.key) - log((double)total) + (double)P.shift * 0.6931471805599453);
    }
}

extern "C" int vqa_sample(const vqa_sample_params* p, void* stream) {
    const int size = p && p->dtype == VQA_F32 ? 4 : 2;
    if (!p || p->rows < 0 || p->V <= 0 || p->V > 1 << 30 || !rows_dtype_ok(p->dtype) || p->ld < 0 ||
        (p->rows > 0 && (!p->logits || !p->u || !p->token)) || (uintptr_t)p->logits % size || (uintptr_t)p->token % 8 ||
        (uintptr_t)p->u % 4 || (uintptr_t)p->temperature % 4 || (uintptr_t)p->top_k % 4 || (uintptr_t)p->top_p % 4 ||
        (uintptr_t)p->min_p % 4 || (uintptr_t)p->logp % 4) {
        vqa_set_error("vqa_sample: bad argument");
        return VQA_EINVAL;
    }
    if (p->rows == 0) return VQA_OK;
    SampleArgs P;
    P.x = p->logits;
    P.ld = p->ld;
    P.rows = p->rows;
    P.u = p->u;
    P.temperature = p->temperature;
    P.top_k = p->top_k;
    P.top_p = p->top_p;
    P.min_p = p->min_p;
    P.temperature_s = p->temperature_value;
    P.top_k_s = p->top_k_value;
    P.top_p_s = p->top_p_value;
    P.min_p_s = p->min_p_value;
    P.V = p->V;
    P.token = p->token;
    P.ld_token = p->ld_token;
    P.logp = p->logp;
    int log_v = 0;
    while (((int64_t)1 << log_v) < p->V) log_v++;
    P.shift = 62 - log_v < 51 ? 62 - log_v : 51;             // V 2^s <= 2^62; w + 2^(52 - s) does not leave its binade
    const hipStream_t s = (hipStream_t)stream;
#define SAMPLE_LAUNCH(DT)                                                                                                 \
    if (p->V <= 64) {                                                                                                     \
        const int64_t wg = (p->rows + 3) / 4;                                                                             \
        hipLaunchKernelGGL(sample_wave_kernel<DT>, dim3((unsigned)(wg < 65536 ? wg : 65536)), dim3(256), 0, s, P);        \
    } else if (p->V <= 8192) {                                                                                            \
        hipLaunchKernelGGL((sample_row_kernel<DT, 256>), dim3((unsigned)(p->rows < 65536 ? p->rows : 65536)), dim3(256), 0, s, P); \
    } else {                                                                                                              \
        hipLaunchKernelGGL((sample_row_kernel<DT, 1024>), dim3((unsigned)(p->rows < 65536 ? p->rows : 65536)), dim3(1024), 0, s, P); \
    }
    if (p->dtype == VQA_BF16) { SAMPLE_LAUNCH(VQA_BF16) }
    else if (p->dtype == VQA_F16) { SAMPLE_LAUNCH(VQA_F16) }
    else { SAMPLE_LAUNCH(VQA_F32) }
#undef SAMPLE_LAUNCH
    ROWS_CHECK_LAUNCH("vqa_sample");
    return VQA_OK;
}
