// policy_common.h - what the translation units of liblobpolicy.so share: errors, packed loads, the description of a segment's walk.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/lobpolicy.h"

namespace lobpolicy {

// ---------------------------------------------------------------------------------------------------------------------------
// host: errors

int fail(int code, const char* format, ...);  // notes the calling thread's message; returns code

inline int launched() {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOBPOLICY_OK : fail(LOBPOLICY_ERR_HIP, "launch: %s", hipGetErrorString(e));
}

#define REQUIRE(condition, ...) \
    do { \
        if (!(condition)) return fail(LOBPOLICY_ERR_ARG, __VA_ARGS__); \
    } while (0)

inline bool aligned(const void* p, int64_t bytes) { return (uintptr_t)p % bytes == 0; }
constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------------------------------------------------------------------
// device: small tools

typedef __bf16 bf16;

template <class T, int W>
struct alignas(sizeof(T) * W < 16 ? sizeof(T) * W : 16) Pack {
    T v[W];
};

// the same from and to any address: the hardware's wide loads and stores need no alignment
template <class T, int W>
__device__ __forceinline__ Pack<T, W> load_anywhere(const T* p) {
    Pack<T, W> x;
    __builtin_memcpy(&x, p, sizeof x);
    return x;
}
template <class T, int W>
__device__ __forceinline__ void store_anywhere(T* p, const Pack<T, W>& x) {
    __builtin_memcpy(p, &x, sizeof x);
}

// element i is x's element i + s, and 0 from behind its end: the end of a row whose length is no multiple of W, loaded as the row's last W elements
template <class T, int W>
__device__ __forceinline__ Pack<T, W> shifted(Pack<T, W> x, int s) {
    static_assert(sizeof x == 8 || sizeof x == 16, "");
    constexpr int bits = 8 * (int)sizeof(T);
    if constexpr (sizeof x == 8) {
        const uint64_t y = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(Pack<T, W>, s >= W ? 0 : y >> (bits * s & 63));
    } else {
        struct Two {
            uint64_t lo, hi;
        } y = __builtin_bit_cast(Two, x);
        const int half = W / 2;
        y.lo = s >= half ? y.hi : y.lo;
        y.hi = s >= half ? 0 : y.hi;
        const int by = bits * (s >= half ? s - half : s) & 63;
        y.lo = s >= W ? 0 : y.lo >> by | y.hi << 1 << (63 - by);
        y.hi >>= by;
        return __builtin_bit_cast(Pack<T, W>, y);
    }
}

template <class T, int W>
__device__ __forceinline__ void load_pack(const T* p, float* out) {
    const Pack<T, W> x = *reinterpret_cast<const Pack<T, W>*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = (float)x.v[i];
}

template <class T, int W>
__device__ __forceinline__ void store_pack(T* p, const float* in) {
    Pack<T, W> x;
#pragma unroll
    for (int i = 0; i < W; ++i) x.v[i] = (T)in[i];
    *reinterpret_cast<Pack<T, W>*>(p) = x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

// ---------------------------------------------------------------------------------------------------------------------------
// decay attention over segments
//
// One recurrence serves the forward pass and all three gradients: with "queries" a, "keys" b and "values" c,
//     S = [cut] ? 0 : e^g S;   S += in_scale b_t c_t^T;   out_t = out_scale a_t^T S
//   out  a = q,  b = k,  c = v   forwards,  S: the state
//   dq   a = do, b = v,  c = k   forwards,  S: the state, transposed
//   dk   a = v,  b = do, c = q   backwards, S: the state's gradient, transposed
//   dv   a = k,  b = q,  c = do  backwards, S: the state's gradient
// Forwards a token with a reset cuts what came before it.  Backwards the gradient passes from token t + 1 to token t with e^g, unless
// t + 1 has a reset; what enters behind the last token (the gradient of the final state) enters without a decay, and what leaves
// in front of token 0 (the gradient of the initial state) leaves with one.

struct Rows {  // one operand: [steps][envs][heads][width], the last dimension contiguous
    const void* data;
    int64_t st, sn, sh;
};

struct Scan {
    Rows a, b, c, out;
    const float* log_decay;
    const uint8_t* reset;
    int64_t reset_st, reset_sn;
    const int32_t* lengths;
    const float* state_in;  // [envs][heads] matrices of da x dc, by the strides below
    float* state_out;
    int64_t in_row, in_col, out_row, out_col;
    int64_t steps, envs;
    int heads, da, dc;
    bool reverse;
    float in_scale, out_scale;
    int64_t part_steps;  // the steps are split into `parts` of this many, each a workgroup's; state_in and state_out are then [unit][part]
    int parts;
    float* carry_out;  // [unit][part]: what comes into the part times this goes out of it, negative: a reset lies in it (the walk without outputs)
};

__device__ __forceinline__ int64_t length_of(const Scan& s, int64_t n) {
    if (!s.lengths) return s.steps;
    const int64_t l = s.lengths[n];
    return l < 0 ? 0 : (l > s.steps ? s.steps : l);
}

// Up to three walks over the same steps in one launch: what one reads the others find in the cache, and few environments fill more of the card.
struct Walks {
    Scan walk[3];
    int count;
};

// One family per type and rows of the state: DA = 32, 64 or 128 holds da.  Every walk's da and dc are the first one's, or (`swapped`: the second and
// third) the first one's the other way round.
template <class T, int DA>
int scan_rows(const Walks& w, bool swapped, hipStream_t stream);

}  // namespace lobpolicy
