// One token per row of logits, drawn with given uniform numbers under temperature, top-k, top-p and min-p (gfx950).
//
// The tokens of a row stand in descending order of their logits, equal logits by index; token i weighs
// w_i = exp((x_i - max) / T).  top-k, min-p and top-p each keep a prefix of that order (top_k tokens; w >= min_p; the tokens
// whose exclusive cumulative weight is below top_p times the weight of what the other two keep), so all together do.  The
// answer is the first token whose inclusive cumulative weight exceeds u times the kept weight.
//
// exp is evaluated in 64 bits: a draw compares sums of up to V weights with u times their sum, and with fp32 exponentials
// (2^-22) one row in ten of a flat distribution over 10^5 tokens would get a neighbouring token.  Weights that are summed by
// atomics are integers, w rounded to a multiple of 2^-s with V 2^s < 2^63: sums are exact, the same in any order.
//
// No row is sorted.  Each of the three questions - the k-th token, the last token of the nucleus, the drawn one - asks which
// token of the order holds a place, counted in tokens or in weight.  Three kernels by the size of the vocabulary:
//   V <= 64    sample_wave_kernel: a wave a row, a token a lane, every lane looks at all others
//   V <= 128   sample_list_kernel: a workgroup a row, all tokens in a short sorted list
//   above      sample_row_kernel: a histogram over steps of the logit finds the bins in which the answers lie, and only their
//              tokens are listed and sorted.  No single bound: 512 x 131072 fp32 logits, top-p 0.95, take 101-106 us.  They issue
//              28 M vector instructions, 27 a logit, most of them the histogram's 64-bit arithmetic: 46 us of the 1024 SIMDs at
//              4 cycles each.  LDS accesses that meet in a bank cost 46 k cycles a unit, 19 us.  The row is read twice: 268 MB for
//              the histogram, 43-50 us by themselves, and again for the list, from the last-level cache (553 MB asked for in all).
// radix_row takes what those lists cannot hold: rows with thousands of equal logits around an answer.  It goes by the bits of
// order-preserving integer keys: a histogram of the leading ones (tokens and weight per bin, in LDS), the bin that holds the
// place, a histogram of the next bits of that bin's keys, and so on to a single key; equal keys weigh the same, so the place
// among them is a division.  Each of its passes adds two numbers to LDS per logit, and equal ones wait for each other: 512 x 131072
// bf16 / fp32 take 540 / 680 us at top-k 2100 (top-k 900: 85 / 103), 650 / 910 us with 40 different values, 1.5 / 2.5 ms where all
// logits are equal; 1 x 50001 135 / 156 us at top-k 2100 (top-k 900: 32 / 33).
#include "rows.h"
#include <float.h>

// a bin or a comparison has to come out the same wherever it is computed: no sums fused into products but by fma()
#pragma clang fp contract(off)

#define SPLIT_BINS 4096
#define SPLIT_LIST 2048
#define SPLIT_PARTS 32
struct SplitRow {                  // see sample_row_kernel
    unsigned long long hist[SPLIT_BINS], list[SPLIT_LIST];
    float max[SPLIT_PARTS], min[SPLIT_PARTS];
    uint32_t n, done;              // entries of the list; workgroups that have added theirs
};

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
    SplitRow* split;               // null, or a record per row
    int32_t parts, part_size;
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

// a value that all lanes of the wave agree on, held in scalar registers
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ __forceinline__ double uniform(double v) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}

struct RowParams { double t, top_p, min_p, u; int32_t k; bool nucleus; };
__device__ __forceinline__ RowParams row_params(const SampleArgs& P, int64_t row) {
    RowParams r;
    r.t = uniform(P.temperature ? (double)P.temperature[row] : P.temperature_s);
    r.top_p = uniform(P.top_p ? (double)P.top_p[row] : P.top_p_s);
    r.min_p = uniform(P.min_p ? (double)P.min_p[row] : P.min_p_s);
    r.k = P.top_k ? P.top_k[row] : P.top_k_s;
    const double u = (double)P.u[row];
    r.u = uniform(u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0);
    r.nucleus = !(r.top_p >= 1.0);
    if (!(r.t > 0.0)) {                                      // the first token of the order
        r.t = 1.0;
        r.k = 1;
    }
    r.t = r.t > 1e-290 ? r.t : 1e-290;                       // (1 / t is finite; floats that differ are 1e-45 apart or more)
    return r;
}
template <int DT> __device__ __forceinline__ Weights<DT> row_weights(const RowParams& r, uint32_t top, int shift) {
    Weights<DT> w;
    w.top = __builtin_amdgcn_readfirstlane(top);
    w.max = uniform(Keys<DT>::value(top));
    w.inv_t = uniform(1.0 / r.t);
    w.min_z = r.min_p > 0.0 ? uniform(log(r.min_p < 1.0 ? r.min_p : 1.0)) : -INFINITY;
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
        const Weights<DT> W = row_weights<DT>(r, top, P.shift);
        const double z = key > Keys<DT>::MASKED ? W.z(key) : -INFINITY;
        const bool in = key > Keys<DT>::MASKED && z >= W.min_z;
        const uint64_t w = in ? W.of_z(z) : 0;
        int before = 0;
        uint64_t mass = 0;                                   // (of what stands before; tokens that are out weigh nothing)
        const uint64_t mine = ((uint64_t)key << 32) | (uint32_t)~lane;       // larger: before
        auto look = [&](int l) {                             // without a branch: a compare, two selects, two sums
            const uint64_t other = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane(key, l) << 32) | (uint32_t)~l;
            const uint64_t wl = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(w >> 32), l) << 32) |
                                (uint32_t)__builtin_amdgcn_readlane((uint32_t)w, l);
            before += other > mine;
            mass += other > mine ? wl : 0;
        };
        int l = 0;
        for (; l + 4 <= P.V; l += 4) {
#pragma unroll
            for (int k = 0; k < 4; k++) look(l + k);
        }
        for (; l < P.V; l++) look(l);
        auto sum = [](uint64_t v) {
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, d);
            return v;
        };
        const bool kept = in && (r.k <= 0 || before < r.k);
        uint64_t total = sum(kept ? w : 0);
        if (r.nucleus) {
            const uint64_t end = nucleus_end(r.top_p, total);
            total = sum(kept && mass < end ? w : 0);
        }
        const uint64_t t = drawn_place(r.u, total);
        const uint64_t m = __ballot(kept && mass <= t && t < mass + w);      // exactly one lane
        const int at = __ffsll((unsigned long long)m) - 1;
        if (lane == at) sample_put<DT>(P, row, lane, z - log(ldexp((double)total, -P.shift)));
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// Radix search, for any V: a workgroup of BT threads a row.
template <int RB> struct Hist {
    uint32_t cnt[1 << RB];
    unsigned long long mass[1 << RB];
};
struct Place {                     // the key that holds a place of the order
    uint32_t key;
    uint64_t cnt_above, mass_above;      // tokens and weight in front of the first token with that key
};
template <int RB> struct RadixShared {
    Hist<RB> h1, h2;
    unsigned long long scan_c[16], scan_m[16];
    uint32_t red[16];
    uint32_t bin;
    unsigned long long cnt_above, mass_above;
    int64_t found;
};

// RB: bits of the key that a level looks at
template <int BT, int RB> struct Radix {
    typedef RadixShared<RB> Shared;
    // the bin of `h` (of `bins` ones) that holds place t, from the top, with c / m in front of the highest bin; all threads
    static __device__ void find_bin(Shared& S, const Hist<RB>& h, int bins, bool by_mass, uint64_t t, uint64_t c, uint64_t m) {
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
    static __device__ void clear(Hist<RB>& h, int bins) {
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
    static __device__ void count(Hist<RB>& h, const typename Elem<DT>::type* x, int V, const Weights<DT>& W, int shift, int bins,
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
    static __device__ Place find(Shared& S, const typename Elem<DT>::type* x, int V, const Weights<DT>& W, bool by_mass, uint64_t t) {
        constexpr int B = Keys<DT>::BITS;
        Place p;
        find_bin(S, S.h1, (1 << RB), by_mass, t, 0, 0);
        uint32_t prefix = S.bin;
        int low = B - RB;                                    // bits that are still open
        while (low > 0) {
            const int bits = low > RB ? RB : low, bins = 1 << bits;
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
    static __device__ int64_t locate(Shared& S, const typename Elem<DT>::type* x, int V, uint32_t key, uint64_t j) {
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

// The whole answer for one row, not masked as a whole, by radix search; all threads of the workgroup.  Not inlined: rows that
// come here are rare, and the kernels that call it keep their registers.
template <int DT, int BT, int RB> __device__ __attribute__((noinline)) void radix_row(LDS_AS void* lds, SampleArgs P, int64_t row) {
    typedef typename Elem<DT>::type T;
    typedef Radix<BT, RB> R;
    typename R::Shared& S = *(typename R::Shared*)(LDS_AS typename R::Shared*)lds;
    const int tid = threadIdx.x;
    const T* x = (const T*)P.x + row * P.ld;
    const RowParams r = row_params(P, row);
    __syncthreads();                                         // (LDS was somebody else's)
    uint32_t top = 0;
    R::template each<DT>(x, P.V, [&](uint32_t key, int) { top = max(top, key); });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if ((tid & 63) == 0) S.red[tid >> 6] = top;
    R::clear(S.h1, 1 << RB);
    __syncthreads();
    for (int w = 0; w < BT / 64; w++) top = max(top, S.red[w]);
    const Weights<DT> W = row_weights<DT>(r, top, P.shift);
    R::template count<DT>(S.h1, x, P.V, W, Keys<DT>::BITS - RB, 1 << RB, 32, 0);
    __syncthreads();
    uint64_t n = 0, total = 0;
    for (int b = tid & 63; b < 1 << RB; b += 64) {           // (every wave for itself)
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
    if (r.nucleus) {
        const uint64_t last = nucleus_end(r.top_p, total) - 1;
        const Place p = R::template find<DT>(S, x, P.V, W, true, last);
        const uint64_t w = W.of(p.key);
        total = p.mass_above + ((last - p.mass_above) / w + 1) * w;
    }
    const uint64_t t = drawn_place(r.u, total);
    const Place p = R::template find<DT>(S, x, P.V, W, true, t);
    const int64_t at = R::template locate<DT>(S, x, P.V, p.key, (t - p.mass_above) / W.of(p.key));
    if (tid == 0) sample_put<DT>(P, row, at, W.z(p.key) - log(ldexp((double)total, -P.shift)));
}

// ------------------------------------------------------------------------------------------------------------------------
// 64 < V <= LIST_ALL: every token goes on the list.  Above:
//   1. the row's maximum and minimum, or a guess of them;
//   2. a histogram over BINS equal steps of x below the maximum, down to where weights no longer count (e^-WINDOW).  With
//      top-k, of tokens: the list is what is not below the k-th token's bin.  Without, of weight: a token of bin b weighs
//      e^(-b d) e^(-(f - 1/2) d) with 0 <= f < 1, the second factor is a short polynomial and added as an integer; the bin's
//      weight is that sum times e^(-b d), and a scan gives the weight in front of each bin;
//   3. the list: the tokens of the bin that the nucleus ends in and of the bins that the draw can fall into.
// The list (key and index of each token, LIST at most) is sorted in LDS, its weights are added up in order, and nucleus and
// draw are looked up in it.  Rows whose list would be too long - many equal logits - go to the radix search.
#define LIST_ALL 128
#define WINDOW 40.0
#define GUESS_FROM 8192

typedef Keys<VQA_F32> FKeys;       // the list's keys: of the logits as fp32, whatever their type

// Steps of x below the maximum: bin b holds the x with floor(at(x)) = b, at(x) = (max - x) scale + 1/2.
struct Steps {
    double max, scale;             // (the difference first: max * scale may dwarf the 1/2)
    float hi, lo;                  // what the bins hold: lo <= x <= hi
    int bins;
    __device__ __forceinline__ double at(float x) const { return fma(max - (double)x, scale, 0.5); }
    __device__ __forceinline__ uint32_t bin(float x) const { return (uint32_t)at(x); }
    // bin, or a place of its own for what lies below and above the bins
    __device__ __forceinline__ uint32_t slot(float x) const { return x > hi ? bins + 1 : x < lo ? bins : bin(x); }
};

// One wave: the smallest float in [bottom, top] that `in` holds for; it holds for `top`, and for every float above one that
// it holds for.  64 candidates a round.  (Stepping from a guess would not do: next to 0 there are millions of floats within
// the rounding of max - x.)
template <typename F> __device__ __forceinline__ float first_float(float bottom, float top, F in) {
    uint32_t lo = FKeys::of(__float_as_uint(bottom)), hi = FKeys::of(__float_as_uint(top));
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, lane = threadIdx.x & 63;
        const uint32_t mine = lane <= (hi - lo) / step ? lo + lane * step : hi;
        const uint64_t m = __ballot(in((float)FKeys::value(mine)));
        if (m == 0) {
            lo += 63 * step + 1;                             // (then lane 63 was below hi)
        } else {
            const uint32_t first = __ffsll((unsigned long long)m) - 1;
            const uint32_t at = first <= (hi - lo) / step ? lo + first * step : hi;
            lo = first ? lo + (first - 1) * step + 1 : at;
            hi = at;
        }
    }
    return (float)FKeys::value(hi);
}

template <int CAP> struct ListShared {
    unsigned long long list[CAP];        // key << 32 | ~index: descending is the order
    union {
        double w[CAP];
        unsigned long long other[CAP];
    };
    double part[16], total, behind;      // total: the kept weight; behind: the weight up to the nucleus's last bin
    unsigned long long above, below;     // weight, or number, of the tokens outside the bins
    float max[16], min[16], edge[4], lo;
    uint32_t n, top, last, pick, bin_end, bin_lo, bin_hi;
};
template <int BINS> union BinShared {
    unsigned long long mass[BINS];       // weights, or the numbers of tokens
    double front[BINS + 2];              // the weight in front of each bin, of what is below the bins, of what is above
};

// exclusive sums of v over the workgroup's threads, in thread order
template <int BT> __device__ __forceinline__ double scan_threads(double* part, double v, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    double base = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < BT / 64; w++) {
        if (w < wave) base += part[w];
        all += part[w];
    }
    __syncthreads();
    total = all;
    const double before = __shfl_up(inc, 1);
    return lane ? base + before : base;
}

// *out = max(*out, v) where v, or 0, grows with the thread: the wave's last thread that has one asks for it
__device__ __forceinline__ void raise(uint32_t* out, int v) {
    const uint64_t m = __ballot(v > 0);
    if (m && (threadIdx.x & 63) == 63 - __clzll((unsigned long long)m)) atomicMax(out, (uint32_t)v);
}

// Sorts list[0, n), descending; the answer is in `list` or, true, in `other`; both have room for the next multiple of 64.
// Every wave sorts stretches of 64 in registers, then four sorted runs at a time become one: an entry's place among them is the
// sum of its places in each, found by three searches that run side by side.  (Not inlined: the kernels keep their registers.)
template <int BT>
__device__ __attribute__((noinline)) bool sort_runs(LDS_AS unsigned long long* list, LDS_AS unsigned long long* other, int n) {
    const int tid = threadIdx.x, lane = tid & 63, m = (n + 63) & ~63;
    for (int i = tid; i < m; i += BT) {                      // (whole waves: m and i - lane are multiples of 64)
        unsigned long long e = i < n ? list[i] : 0;
#pragma unroll
        for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
            for (int j = k >> 1; j > 0; j >>= 1) {
                const unsigned long long o = __shfl_xor(e, j);
                e = ((lane & j) == 0) == ((lane & k) == 0) ? (o > e ? o : e) : (o < e ? o : e);
            }
        list[i] = e;
    }
    __syncthreads();
    bool swapped = false;
    for (int run = 64; run < n; run *= 4) {
        const LDS_AS unsigned long long* src = swapped ? other : list;
        LDS_AS unsigned long long* dst = swapped ? list : other;
        for (int i = tid; i < m; i += BT) {
            const unsigned long long e = src[i];
            const int base = i & ~(4 * run - 1), mine = (i - base) / run;
            int o[3], len[3], at[3] = {0, 0, 0};
            unsigned long long least[3];                     // equal ones (the padding) keep their order
#pragma unroll
            for (int q = 0; q < 3; q++) {
                const int r = q + (q >= mine);
                o[q] = base + r * run;
                len[q] = min(max(m - o[q], 0), run);
                least[q] = r < mine ? e : e + 1;             // (no key is all ones)
            }
            for (int step = run; step > 0; step >>= 1)
#pragma unroll
                for (int q = 0; q < 3; q++)
                    if (at[q] + step <= len[q] && src[o[q] + at[q] + step - 1] >= least[q]) at[q] += step;
            dst[base + (i - base - mine * run) + at[0] + at[1] + at[2]] = e;
        }
        __syncthreads();
        swapped = !swapped;
    }
    return swapped;
}

// The same; short lists by counting what is larger than each entry, n * n / BT comparisons a thread without a barrier.  (100 x 20000
// fp32 with 1024 threads, counted against merged: top-k 200 20.7 / 22 us, 300 26 / 23, 500 32 / 25.  A bitonic network in LDS, a
// barrier at every longer distance, took 31 us where merging takes 25, top-k 700, and as long for the longest lists, 2000.)
template <int BT> __device__ __forceinline__ bool sort_list(unsigned long long* list, unsigned long long* other, int n) {
    const int tid = threadIdx.x;
    if (n > (BT < 512 ? BT / 2 : 256)) return sort_runs<BT>((LDS_AS unsigned long long*)list, (LDS_AS unsigned long long*)other, n);
    int parts = 2;                                           // threads an entry
    while (parts < 64 && parts * 2 * n <= BT) parts *= 2;
    const int i = tid / parts;
    const unsigned long long mine = i < n ? list[i] : 0;
    int rank = 0;
    if (i < n)
        for (int j = tid % parts; j < n; j += parts) rank += list[j] > mine;
    for (int d = 1; d < parts; d <<= 1) rank += __shfl_xor(rank, d);
    if (i < n && tid % parts == 0) other[rank] = mine;       // (entries differ: so do ranks)
    __syncthreads();
    return true;
}

// Nucleus and draw in the sorted list of n tokens.  Without `front` the list holds all that is kept but for the nucleus;
// with it, front[b] is the weight in front of bin b, `total` all weight, and the list holds the bins that matter.
template <int DT, int BT, int CAP>
__device__ __forceinline__ void finish_list(ListShared<CAP>& L, bool swapped, const SampleArgs& P, int64_t row,
                                            const RowParams& r, const Weights<VQA_F32>& W, int n, double* front, const Steps& S,
                                            double total) {
    const unsigned long long* list = swapped ? L.other : L.list;         // (sorted; the weights take the other place)
    double* weight = swapped ? (double*)L.list : L.w;
    const int tid = threadIdx.x, per = (n + BT - 1) / BT, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    double sum = 0.0, listed;
    for (int i = i0; i < i1; i++) {
        const double w = exp(W.z((uint32_t)(list[i] >> 32)));
        weight[i] = w;
        sum += w;
    }
    if (tid == 0) L.last = L.pick = 0;
    const double before = scan_threads<BT>(L.part, sum, listed);
    auto bin_of = [&](int i) { return S.slot((float)FKeys::value((uint32_t)(list[i] >> 32))); };
    if (front) {                                             // front[b] becomes what is in front of the bin beyond the list
        double g = before;
        for (int i = i0; i < i1; i++) {
            const uint32_t b = bin_of(i);
            if (i == 0 || bin_of(i - 1) != b) front[b] -= g;
            g += weight[i];
        }
        __syncthreads();
    } else {
        total = listed;
    }
    auto base = [&](int i) { return front ? front[bin_of(i)] : 0.0; };
    uint32_t last = n - 1;
    if (r.nucleus) {                                         // the last token in front of which less than `end` stands
        const double end = r.top_p * total;
        double g = before;
        int mine = 0;
        for (int i = i0; i < i1; i++) {
            if (base(i) + g < end) mine = i;
            g += weight[i];
        }
        raise(&L.last, mine);
        __syncthreads();
        last = L.last;
        if (i0 <= (int)last && (int)last < i1) {
            double g = before;
            for (int i = i0; i <= (int)last; i++) g += weight[i];
            L.total = base(last) + g;
        }
        __syncthreads();
        total = L.total;
    }
    // drawn: the last kept token that does not start behind t, of those that weigh anything
    const double t = r.u * total;
    double g = before;
    int mine = 0;
    for (int i = i0; i < i1 && i <= (int)last; i++) {
        const double w = weight[i];
        if (w > 0.0 && base(i) + g <= t) mine = i;
        g += w;
    }
    raise(&L.pick, mine);
    __syncthreads();
    if (tid == 0) {
        const unsigned long long e = list[L.pick];
        sample_put<DT>(P, row, (int64_t)(uint32_t)~(uint32_t)e, W.z((uint32_t)(e >> 32)) - log(total));
    }
}

__device__ __forceinline__ unsigned long long list_entry(uint32_t key, int i) {
    return ((unsigned long long)key << 32) | (uint32_t)~i;
}
template <int DT> __device__ __forceinline__ uint32_t float_key(const typename Elem<DT>::type* x, int64_t i) {
    return FKeys::of(__float_as_uint(elem_get<DT>(x + i)));
}

// One row a workgroup, without a loop over rows: the compiler would keep the constants of exp and log in registers around it.
#define GRID_X (1 << 20)
__device__ __forceinline__ int64_t grid_row() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

template <int DT> __global__ __launch_bounds__(2 * LIST_ALL) void sample_list_kernel(SampleArgs P) {
    typedef typename Elem<DT>::type T;
    constexpr int BT = 2 * LIST_ALL;                         // (two threads an entry: sort_list counts)
    __shared__ ListShared<LIST_ALL> L;
    const int tid = threadIdx.x, V = P.V;
    const int64_t row = grid_row();
    if (row >= P.rows) return;
    const T* x = (const T*)P.x + row * P.ld;
    const uint32_t key = tid < V ? float_key<DT>(x, tid) : 0;
    uint32_t top = key;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if ((tid & 63) == 0) L.max[tid >> 6] = __uint_as_float(top);
    if (tid == 0) L.n = 0;
    __syncthreads();
    for (int w = 0; w < BT / 64; w++) top = max(top, __float_as_uint(L.max[w]));
    if (top <= FKeys::MASKED) {
        if (tid == 0) sample_put<DT>(P, row, -1, -INFINITY);
        return;
    }
    const RowParams r = row_params(P, row);
    const Weights<VQA_F32> W = row_weights<VQA_F32>(r, top, P.shift);
    const bool in = key > FKeys::MASKED && W.z(key) >= W.min_z;
    if (tid < LIST_ALL) L.list[tid] = in ? list_entry(key, tid) : 0;
    const uint64_t m = __ballot(in);
    if ((tid & 63) == 0) atomicAdd(&L.n, (uint32_t)__popcll((unsigned long long)m));
    __syncthreads();
    const bool swapped = sort_list<BT>(L.list, L.other, V);
    int n = (int)L.n;
    if (r.k > 0 && r.k < n) n = r.k;
    finish_list<DT, BT, LIST_ALL>(L, swapped, P, row, r, W, n, nullptr, Steps(), 0.0);
}

// Passes over a row.  (Kept short: a pass runs once per row, and instructions that come from memory cost as much as the
// row.  With the row held in registers and its passes unrolled, 75 KB of code, a row of 50001 took 12 us in the last pass
// alone, 6 with these loops.)
template <int DT, int BT> struct RowPass {
    typedef typename Elem<DT>::type T;
    static constexpr int N = Elem<DT>::N;
    const T* x;
    int V, nv;
    __device__ __forceinline__ RowPass(const T* x_, int V_) : x(x_), V(V_), nv(V_ / N) {}
    // calls f(x) with a sixteenth of the logits or more, in stretches all over the row
    template <typename F> __device__ __forceinline__ void some(F f) const {
#pragma unroll 4
        for (int v = threadIdx.x; v < nv; v += 16 * BT) {
            const u32x4 r = vec_load<DT>(x + (int64_t)v * N);
#pragma unroll
            for (int q = 0; q < N; q++) f(vec_get<DT>(r, q), 0);
        }
    }
    // calls f(x, index) with every logit as a float; four pieces of 16 bytes on their way at a time
    template <typename F> __device__ __forceinline__ void each(F f) const {
        constexpr int U = 4;
        int v = threadIdx.x;
#pragma unroll 1
        for (; v + (U - 1) * BT < nv; v += U * BT) {
            u32x4 r[U];
#pragma unroll
            for (int k = 0; k < U; k++) r[k] = vec_load<DT>(x + (int64_t)(v + k * BT) * N);
#pragma unroll
            for (int k = 0; k < U; k++)
#pragma unroll
                for (int q = 0; q < N; q++) f(vec_get<DT>(r[k], q), (v + k * BT) * N + q);
        }
#pragma unroll 1
        for (; v < nv; v += BT) {
            const u32x4 r = vec_load<DT>(x + (int64_t)v * N);
#pragma unroll
            for (int q = 0; q < N; q++) f(vec_get<DT>(r, q), v * N + q);
        }
#pragma unroll 1
        for (int i = nv * N + threadIdx.x; i < V; i += BT) f(elem_get<DT>(x + i), i);
    }
};

template <int BT, int BINS> struct BinScan {
    static constexpr int PER = BINS / BT;
    // front[b]: `above` and the sum of v over the bins before b; v: the thread's bins, read from where front goes
    static __device__ __forceinline__ double scan(BinShared<BINS>& B, double* part, const double (&v)[PER], double above) {
        double sum = 0.0, total;
#pragma unroll
        for (int k = 0; k < PER; k++) sum += v[k];
        double g = above + scan_threads<BT>(part, sum, total);
#pragma unroll
        for (int k = 0; k < PER; k++) {
            B.front[threadIdx.x * PER + k] = g;
            g += v[k];
        }
        return total;
    }
    // the last bin with something in it that starts in front of (or, `upto`, at) t
    static __device__ __forceinline__ void last_bin(const BinShared<BINS>& B, const double (&v)[PER], uint32_t* out, double t, bool upto) {
        int mine = 0;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const double g = B.front[threadIdx.x * PER + k];
            if (v[k] > 0.0 && (upto ? g <= t : g < t)) mine = threadIdx.x * PER + k;
        }
        raise(out, mine);
    }
};

// WHOLE: one workgroup does a row.  Few long rows are split over P.parts workgroups each, in three launches that meet in
// SplitRow, a workspace per row: MAXIMUM, HISTOGRAM and COLLECT do a pass over their part each, and the workgroup that comes
// last to the row's list does the rest.  What depends on the whole row is computed by each of its workgroups anew.
enum SamplePhase { WHOLE, MAXIMUM, HISTOGRAM, COLLECT };
template <int DT, int BT, int BINS, int LIST, SamplePhase PHASE> __global__ __launch_bounds__(BT, 4) void sample_row_kernel(SampleArgs P) {
    typedef typename Elem<DT>::type T;
    constexpr int PER = BINS / BT;
    constexpr bool SPLIT = PHASE != WHOLE;
    constexpr int RB = BINS >= 4096 ? 11 : 10;
    __shared__ union {
        struct {
            ListShared<LIST> L;
            BinShared<BINS> B;
        } s;
        RadixShared<RB> radix;
    } shared;
    ListShared<LIST>& L = shared.s.L;
    BinShared<BINS>& B = shared.s.B;
    const int tid = threadIdx.x, wave = tid >> 6;
    const int part = SPLIT ? blockIdx.x % P.parts : 0;
    const int64_t row = SPLIT ? blockIdx.x / P.parts : grid_row();
    if (row >= P.rows) return;
    SplitRow* const Q = P.split + (SPLIT ? row : 0);
    const int first_index = part * P.part_size;
    const RowPass<DT, BT> H((const T*)P.x + row * P.ld + first_index, SPLIT ? ::min(P.part_size, P.V - first_index) : P.V);
    const RowParams r = row_params(P, row);
    const bool by_count = r.k > 0 && r.k < P.V;
    // The maximum of a whole row costs a pass over memory in which little is computed, and the histogram is bound by
    // arithmetic.  Without min-p (which needs the true maximum) long rows take both passes as one: the bins lie between the
    // largest and the smallest logit of a sixteenth of the row, and the few tokens outside go on the list at once.  If they
    // are not few, it starts again with the whole row's.  (512 x 131072 fp32, top-p: 143 us in two passes, 107 in one;
    // 1024 x 16000 bf16 50 and 44, 1024 x 4096 22.7 and 22.9.  Where it has to start again: 512 x 131072 fp32 152 us instead of 94,
    // 1024 x 16000 bf16, whose 2500 raised logits are also too many for the list, 105 instead of 42.)
    bool guess = PHASE == WHOLE && P.V >= GUESS_FROM && !(r.min_p > 0.0);
    float max, min;
    Weights<VQA_F32> W;
    Steps S;
    double d;                                                // a step of the bins in z
    for (;; guess = false) {
        max = -INFINITY, min = INFINITY;
        if (PHASE == WHOLE || PHASE == HISTOGRAM)
            for (int b = tid; b < BINS; b += BT) B.mass[b] = 0;
        if (tid == 0) {
            L.n = L.top = L.bin_end = L.bin_lo = L.bin_hi = 0;
            L.above = L.below = 0;
        }
        if (PHASE == WHOLE || PHASE == MAXIMUM) {
            auto widen = [&](float f, int) {
                max = fmaxf(max, f);                         // (a NaN is passed over)
                min = fminf(min, f >= -FLT_MAX ? f : INFINITY);
            };
            if (guess) H.some(widen);
            else H.each(widen);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) {
                max = fmaxf(max, __shfl_xor(max, d));
                min = fminf(min, __shfl_xor(min, d));
            }
            if ((tid & 63) == 0) {
                L.max[wave] = max;
                L.min[wave] = min;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < BT / 64; w++) {
                max = fmaxf(max, L.max[w]);
                min = fminf(min, L.min[w]);
            }
        } else {
            __syncthreads();
            for (int q = 0; q < P.parts; q++) {
                max = fmaxf(max, Q->max[q]);
                min = fminf(min, Q->min[q]);
            }
        }
        if (PHASE == MAXIMUM) {
            for (int b = part * BT + tid; b < BINS; b += P.parts * BT) Q->hist[b] = 0;
            if (tid == 0) {
                Q->max[part] = max;
                Q->min[part] = min;
                if (part == 0) Q->n = Q->done = 0;
            }
            return;
        }
        max = uniform(max);
        min = uniform(min);
        if (max == -INFINITY || max == INFINITY || max == min) {
            if (guess) {
                __syncthreads();                             // (L.max is written again)
                continue;
            }
            if (max == -INFINITY) {
                if (tid == 0 && part == 0) sample_put<DT>(P, row, -1, -INFINITY);
            } else if (PHASE == WHOLE || (PHASE == COLLECT && part == 0)) {
                radix_row<DT, BT, RB>((LDS_AS void*)&shared, P, row);
            }
            return;
        }
        W = row_weights<VQA_F32>(r, FKeys::of(__float_as_uint(max)), P.shift);
        const bool cut = (double)max - (double)min > WINDOW * r.t;
        const double range = uniform(cut ? WINDOW * r.t : (double)max - (double)min);
        S.max = W.max;
        S.scale = uniform((BINS - 1) / range);
        S.hi = max;
        S.lo = min;
        S.bins = BINS;
        if (r.min_p > 0.0 || cut) {
            if (wave == 0) {
                const float f = first_float(min, max, [&](float f) {
                    return (double)max - (double)f <= range && ((double)f - W.max) * W.inv_t >= W.min_z;
                });
                if (tid == 0) L.lo = f;
            }
            __syncthreads();
            S.lo = uniform(L.lo);
        }
        d = uniform(W.inv_t / S.scale);
        if (PHASE == WHOLE || PHASE == HISTOGRAM) {
            const float lo = S.lo;
            // (what is further down than WINDOW weighs nothing)
            const float least = guess && !cut ? uniform(fmaxf((float)((double)max - WINDOW * r.t), -FLT_MAX)) : lo;
            auto outside = [&](float f, int i) {
                if ((f > max) | ((f < lo) & (f >= least))) {
                    const uint32_t at = atomicAdd(&L.n, 1u);
                    if (at < LIST) L.list[at] = list_entry(FKeys::of(__float_as_uint(f)), i);
                }
            };
            if (by_count) {
                H.each([&](float f, int i) {
                    if ((f >= lo) & (f <= max)) atomicAdd((uint32_t*)&B.mass[S.bin(f)], 1u);
                    else if (PHASE == WHOLE) outside(f, i);
                });
            } else {
                // e^(-(f - 1/2) d) for 0 <= f < 1: the series around 1/2, in powers of f (and `magic` on top)
                const double c1 = -d, c2 = d * d * 0.5, c3 = d * d * d * (-1.0 / 6.0), c4 = d * d * d * d * (1.0 / 24.0);
                constexpr bool FIFTH = BINS < 4096;          // (d / 2)^5 / 5! is 2^-45 with 4096 bins, 2^-35 with 1024
                const double c5 = FIFTH ? d * d * d * d * d * (-1.0 / 120.0) : 0.0;
                const double a4 = uniform(c4 - 2.5 * c5), a3 = uniform(c3 - 2.0 * c4 + 2.5 * c5);
                const double a2 = uniform(c2 - 1.5 * c3 + 1.5 * c4 - 1.25 * c5);
                const double a1 = uniform(c1 - c2 + 0.75 * c3 - 0.5 * c4 + 0.3125 * c5);
                const double a0 = uniform(1.0 - 0.5 * c1 + 0.25 * c2 - 0.125 * c3 + 0.0625 * c4 - 0.03125 * c5 + W.magic);
                const long long magic = __double_as_longlong(W.magic);
                H.each([&](float f, int i) {
                    if ((f >= lo) & (f <= max)) {
                        const double a = S.at(f), e = __builtin_amdgcn_fract(a);
                        const double q = FIFTH ? fma(e, c5, a4) : a4;
                        const double p = fma(e, fma(e, fma(e, fma(e, q, a3), a2), a1), a0);
                        atomicAdd(&B.mass[(uint32_t)a], (unsigned long long)(__double_as_longlong(p) - magic));
                    } else if (PHASE == WHOLE) {
                        outside(f, i);
                    }
                });
            }
            __syncthreads();
        }
        if (!guess || L.n <= LIST / 2) break;
        __syncthreads();
    }
    if (PHASE == HISTOGRAM) {
        for (int b = tid; b < BINS; b += BT)
            if (B.mass[b]) atomicAdd(&Q->hist[b], B.mass[b]);
        return;
    }
    double above = 0.0, below = 0.0, bins_top = 1.0;         // outside the bins; the weight of the bins' largest logit
    if (guess && L.n > 0) {
        const uint32_t guessed = W.top;
        for (uint32_t i = tid; i < L.n; i += BT) atomicMax(&L.top, (uint32_t)(L.list[i] >> 32));
        __syncthreads();
        const uint32_t top = ::max(guessed, (uint32_t)__builtin_amdgcn_readfirstlane(L.top));
        if (top == FKeys::TOP) {
            radix_row<DT, BT, RB>((LDS_AS void*)&shared, P, row);
            return;
        }
        W.top = top;
        W.max = uniform(FKeys::value(top));
        bins_top = exp(W.z(guessed));
        for (uint32_t i = tid; i < L.n; i += BT) {
            const uint32_t key = (uint32_t)(L.list[i] >> 32);
            atomicAdd(key > guessed ? &L.above : &L.below, by_count ? 1ull : (unsigned long long)W.of(key));
        }
        __syncthreads();
        above = by_count ? (double)L.above : ldexp((double)L.above, -P.shift);
        below = by_count ? (double)L.below : ldexp((double)L.below, -P.shift);
    }
    // the weight, or with top-k the number, of the tokens in each bin
    double v[PER];
    {
        double weight = by_count ? 1.0 : ldexp(bins_top * exp(-d * (tid * PER)), -P.shift);      // 2^-s e^(z of the thread's first bin)
        const double step = by_count ? 1.0 : exp(-d);
#pragma unroll
        for (int q = 0; q < PER; q++) {
            v[q] = (double)(SPLIT ? Q->hist[tid * PER + q] : B.mass[tid * PER + q]) * weight;
            weight *= step;
        }
    }
    const double binned = above + BinScan<BT, BINS>::scan(B, L.part, v, above), total = binned + below;
    if (tid == 0) {
        B.front[BINS] = binned;
        B.front[BINS + 1] = 0.0;
    }
    if (by_count) {
        BinScan<BT, BINS>::last_bin(B, v, &L.bin_hi, (double)r.k, false);        // (or the last bin, where fewer tokens count)
    } else if (r.nucleus) {
        BinScan<BT, BINS>::last_bin(B, v, &L.bin_end, r.top_p * total, false);
        __syncthreads();
        if (tid == (int)L.bin_end / PER) {
            double g = B.front[tid * PER];
#pragma unroll
            for (int q = 0; q < PER; q++)
                if (q <= (int)L.bin_end % PER) g += v[q];
            L.behind = r.top_p * total > binned ? total : g;
        }
        __syncthreads();
        BinScan<BT, BINS>::last_bin(B, v, &L.bin_lo, r.u * B.front[L.bin_end], true);
        BinScan<BT, BINS>::last_bin(B, v, &L.bin_hi, r.u * L.behind, true);
    } else {
        BinScan<BT, BINS>::last_bin(B, v, &L.bin_lo, r.u * total, true);
    }
    __syncthreads();
    // the tokens with edge 0 <= x < edge 1 or edge 2 <= x < edge 3 go on the list
    if (wave < 4) {
        const uint32_t end = L.bin_end;
        const uint32_t first = by_count ? 0 : wave < 2 ? L.bin_lo : end;
        const uint32_t last = by_count ? L.bin_hi : wave >= 2 ? end : r.nucleus ? ::min(L.bin_hi, end) : first;
        float e = INFINITY;
        if (wave < 2 || (r.nucleus && !by_count)) {
            if (!(wave & 1)) e = first_float(S.lo, max, [&](float f) { return S.bin(f) <= last; });
            else if (first > 0) e = first_float(S.lo, max, [&](float f) { return S.bin(f) < first; });
            else e = (float)FKeys::value(FKeys::of(__float_as_uint(max)) + 1);       // (the next float: above it all is listed)
        }
        if ((tid & 63) == 0) L.edge[wave] = e;
    }
    __syncthreads();
    const float e0 = uniform(L.edge[0]), e1 = uniform(L.edge[1]), e2 = uniform(L.edge[2]), e3 = uniform(L.edge[3]);
    H.each([&](float f, int i) {
        if (((f >= e0) & (f < e1)) | ((f >= e2) & (f < e3))) {
            const uint32_t at = atomicAdd(&L.n, 1u);
            if (at < LIST) L.list[at] = list_entry(FKeys::of(__float_as_uint(f)), first_index + i);
        }
    });
    __syncthreads();
    int n = (int)L.n;
    if (SPLIT) {                                             // add them to the row's list; the last workgroup takes it
        if (tid == 0) L.last = atomicAdd(&Q->n, (uint32_t)n);
        __syncthreads();
        // Entries are stored past the L2 cache (atomic, agent scope).  Every wave waits for its own stores before the barrier,
        // which waits for none, as the release of thread 0 waits for those of its own wave only.  (A fence by every wave would
        // write the L2 cache back each time, 43 us for 256 workgroups.)
        for (int i = tid; i < n; i += BT)
            if (i < LIST && L.last + i < LIST)
                __hip_atomic_store(&Q->list[L.last + i], L.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        wait_for_stores();
        __syncthreads();
        if (tid == 0) L.pick = __hip_atomic_fetch_add(&Q->done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if ((int)L.pick != P.parts - 1) return;
        n = (int)__hip_atomic_load(&Q->n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (n > LIST || n == 0) {
        radix_row<DT, BT, RB>((LDS_AS void*)&shared, P, row);
        return;
    }
    if (SPLIT) {
        for (int i = tid; i < n; i += BT) L.list[i] = __hip_atomic_load(&Q->list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
    }
    const bool swapped = sort_list<BT>(L.list, L.other, n);
    if (by_count && r.k < n) n = r.k;
    finish_list<DT, BT, LIST>(L, swapped, P, row, r, W, n, by_count ? nullptr : B.front, S, total);
}

// Workgroups of a row.  A split row pays for three launches and for a scan of its bins in each workgroup of the last: worth it
// from 34304 logits on for a single row, from 131072 for 64 of them, not with more rows.  In us, split against whole, of calls one
// after the other, bf16 / fp32:
//                  top-p 0.9             top-k 50, top-p 0.95
//   1 x 50000      23 24 against 28 26   19 20 against 22 21
//   1 x 131072     25 22 against 45 43   20 20 against 34 34
//   8 x 65536      28 27 against 32 33   21 21 against 24 27
//   32 x 65536     37 35 against 36 31   28 29 against 24 25   (whole)
//   32 x 98304     38 39 against 44 41   30 31 against 31 30
//   64 x 98304     43 43 against 45 40   33 34 against 30 31   (whole)
//   64 x 131072    45 48 against 52 50   35 37 against 35 35
static int sample_parts(int64_t rows, int32_t V) {
    if (rows <= 0 || rows > 64 || V < 32768 + 1536 * rows) return 1;
    const int64_t by_rows = 256 / rows, by_size = V / 8192;
    const int64_t parts = by_rows < by_size ? by_rows : by_size;
    return (int)(parts < SPLIT_PARTS ? parts : SPLIT_PARTS);
}

extern "C" int64_t vqa_sample_workspace(int64_t rows, int32_t V) {
    return sample_parts(rows, V) > 1 ? rows * (int64_t)sizeof(SplitRow) : 0;
}

// The kernel of a whole row of more than LIST_ALL logits, in us (calls one after the other, bf16, top-p 0.9):
//                                      1 x 8192  256 x 4096  256 x 32768  1024 x 4096  1024 x 16384  512 x 65536  1024 x 131072
//   1024 threads, 4096 bins, list 2048  16        17          27           58           74            71           205
//   512 threads, 4096 bins, list 2048   16        15          31           36           51            58           168
//   256 threads, 1024 bins, list 1024   14        14          46           19           37            80           791
// So: 1024 threads for up to 256 rows, one on a unit, above 4096 logits; 256 threads, whose few bins cost little to scan and of
// which eight share a unit, up to 16384 logits, above which the tokens of a bin become too many for its list; else 512.
// The borders are not exact: 257 x 16384 takes 28 us where 512 threads take 25, 4096 x 32768 249 where 256 threads take 196.
extern "C" int vqa_sample(const vqa_sample_params* p, void* stream) {
    const int size = p && p->dtype == VQA_F32 ? 4 : 2;
    const int parts = p ? sample_parts(p->rows, p->V) : 1;
    if (!p || p->rows < 0 || p->V <= 0 || p->V > 1 << 30 || p->rows > (int64_t)GRID_X * 65535 || !rows_dtype_ok(p->dtype) || p->ld < 0 ||
        (p->rows > 0 && (!p->logits || !p->u || !p->token)) || (uintptr_t)p->logits % size || (uintptr_t)p->token % 8 ||
        (uintptr_t)p->u % 4 || (uintptr_t)p->temperature % 4 || (uintptr_t)p->top_k % 4 || (uintptr_t)p->top_p % 4 ||
        (uintptr_t)p->min_p % 4 || (uintptr_t)p->logp % 4 ||
        (parts > 1 && (!p->workspace || (uintptr_t)p->workspace % 8))) {
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
    P.split = (SplitRow*)p->workspace;
    P.parts = parts;
    P.part_size = ((p->V + parts - 1) / parts + 63) / 64 * 64;
    int log_v = 0;
    while (((int64_t)1 << log_v) < p->V) log_v++;
    P.shift = 62 - log_v < 51 ? 62 - log_v : 51;             // V 2^s <= 2^62; w + 2^(52 - s) does not leave its binade
    const hipStream_t s = (hipStream_t)stream;
#define SAMPLE_LAUNCH(DT)                                                                                                 \
    if (p->V <= 64) {                                                                                                     \
        const int64_t wg = (p->rows + 3) / 4;                                                                             \
        hipLaunchKernelGGL(sample_wave_kernel<DT>, dim3((unsigned)(wg < 65536 ? wg : 65536)), dim3(256), 0, s, P);        \
    } else if (p->V <= LIST_ALL) {                                                                                        \
        hipLaunchKernelGGL(sample_list_kernel<DT>, rows_grid, dim3(2 * LIST_ALL), 0, s, P);                               \
    } else {                                                                                                              \
        if (parts > 1) {                                                                                                  \
            SAMPLE_PHASE(DT, MAXIMUM, parts_grid)                                                                         \
            SAMPLE_PHASE(DT, HISTOGRAM, parts_grid)                                                                       \
            SAMPLE_PHASE(DT, COLLECT, parts_grid)                                                                         \
        } else if (p->rows <= 256 && p->V > 4096)                                                                         \
            hipLaunchKernelGGL((sample_row_kernel<DT, 1024, 4096, 2048, WHOLE>), rows_grid, dim3(1024), 0, s, P);         \
        else if (p->V <= 16384)                                                                                           \
            hipLaunchKernelGGL((sample_row_kernel<DT, 256, 1024, 1024, WHOLE>), rows_grid, dim3(256), 0, s, P);           \
        else                                                                                                              \
            hipLaunchKernelGGL((sample_row_kernel<DT, 512, 4096, 2048, WHOLE>), rows_grid, dim3(512), 0, s, P);           \
    }
    const dim3 parts_grid((unsigned)(parts > 1 ? p->rows * parts : 1));
#define SAMPLE_PHASE(DT, PHASE, GRID)                                                                                     \
    hipLaunchKernelGGL((sample_row_kernel<DT, 512, SPLIT_BINS, SPLIT_LIST, PHASE>), GRID, dim3(512), 0, s, P);            \
    ROWS_CHECK_LAUNCH("vqa_sample");
    const dim3 rows_grid((unsigned)(p->rows < GRID_X ? p->rows : GRID_X), (unsigned)((p->rows + GRID_X - 1) / GRID_X));
    if (p->dtype == VQA_BF16) { SAMPLE_LAUNCH(VQA_BF16) }
    else if (p->dtype == VQA_F16) { SAMPLE_LAUNCH(VQA_F16) }
    else { SAMPLE_LAUNCH(VQA_F32) }
#undef SAMPLE_LAUNCH
#undef SAMPLE_PHASE
    ROWS_CHECK_LAUNCH("vqa_sample");
    return VQA_OK;
}
