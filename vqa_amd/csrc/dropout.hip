// Dropout whose mask is never stored: the random bits of an element are a function of (seed, offset, index), so the
// backward pass computes them again (gfx950).
//
// Bits: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011), key = the seed's
// halves, counter = the halves of offset + index / 8 and two zeros.  One block of 128 bits serves 8 elements with 16 bits
// each, low half of a word first: an element is dropped iff its bits are below `threshold`, i.e. with probability
// threshold / 65536, and kept ones are multiplied by 65536 / (65536 - threshold), which keeps the expectation exactly.
// (Ten rounds cost 20 wide products, a quarter-rate instruction each.  With 32 bits per element they would be as expensive
// as the memory traffic of a bf16 pass; with 16 they are half of it.)
//
// Dropped elements become +0 whatever they were (a NaN included).  x and y may be the same buffer.
#include "rows.h"

struct Philox { uint32_t w[4]; };

__device__ __forceinline__ Philox philox10(uint64_t counter, uint64_t seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}
__device__ __forceinline__ bool philox_keep(const Philox& r, int j, uint32_t threshold) {
    return ((r.w[j >> 1] >> ((j & 1) * 16)) & 0xFFFFu) >= threshold;
}

#define DROPOUT_GRID (1 << 23)

// One thread: 8 consecutive elements at a time, a grid-stride apart.
template <int DT>
__global__ __launch_bounds__(256) void dropout_kernel(const typename Elem<DT>::type* x, typename Elem<DT>::type* y, int64_t n,
                                                      uint32_t threshold, float scale, uint64_t seed, uint64_t offset,
                                                      const int64_t* __restrict__ state) {
    constexpr int N = Elem<DT>::N;
    if (state) {
        seed = (uint64_t)state[0];
        offset = (uint64_t)state[1];
    }
    const int64_t step = (int64_t)gridDim.x * 256, blocks = (n + 7) / 8;
    for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += step) {
        const int64_t i = b * 8;
        if (i + 8 <= n) {
            u32x4 v[8 / N];
#pragma unroll
            for (int k = 0; k < 8 / N; k++) v[k] = vec_load<DT>(x + i + k * N);
            const Philox r = philox10(offset + (uint64_t)b, seed);
#pragma unroll
            for (int k = 0; k < 8 / N; k++) {
                float f[N];
#pragma unroll
                for (int j = 0; j < N; j++) f[j] = philox_keep(r, k * N + j, threshold) ? vec_get<DT>(v[k], j) * scale : 0.f;
                vec_store<DT>(y + i + k * N, vec_make<DT>(f));
            }
        } else {
            const Philox r = philox10(offset + (uint64_t)b, seed);
            for (int j = 0; j < 8 && i + j < n; j++)
                elem_put<DT>(y + i + j, philox_keep(r, j, threshold) ? elem_get<DT>(x + i + j) * scale : 0.f);
        }
    }
}

extern "C" int vqa_dropout(const void* x, void* y, int64_t n, int32_t dtype, int32_t threshold, uint64_t seed, uint64_t offset,
                           const int64_t* state, void* stream) {
    const int size = dtype == VQA_F32 ? 4 : 2;
    if ((n > 0 && (!x || !y)) || n < 0 || !rows_dtype_ok(dtype) || threshold < 0 || threshold > 65536 || (uintptr_t)x % size ||
        (uintptr_t)y % size || (uintptr_t)state % 8) {
        vqa_set_error("vqa_dropout: bad argument");
        return VQA_EINVAL;
    }
    if (n == 0) return VQA_OK;
    const float scale = threshold < 65536 ? 65536.f / (float)(65536 - threshold) : 0.f;
    const int64_t want = ((n + 7) / 8 + 255) / 256;
    // (a block of 8 elements a thread, until the launch has 2^31 threads: with 16384 workgroups that loop, 2^28 bf16 elements
    // took 196 us instead of 177)
    const dim3 grid((unsigned)(want < DROPOUT_GRID ? want : DROPOUT_GRID)), block(256);
#define LAUNCH(DT)                                                                                                             \
    hipLaunchKernelGGL(dropout_kernel<DT>, grid, block, 0, (hipStream_t)stream, (const Elem<DT>::type*)x, (Elem<DT>::type*)y, n, \
                       (uint32_t)threshold, scale, seed, offset, state)
    if (dtype == VQA_BF16) LAUNCH(VQA_BF16);
    else if (dtype == VQA_F16) LAUNCH(VQA_F16);
    else LAUNCH(VQA_F32);
#undef LAUNCH
    ROWS_CHECK_LAUNCH("vqa_dropout");
    return VQA_OK;
}
