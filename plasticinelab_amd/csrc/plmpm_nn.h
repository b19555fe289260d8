// Shared by the policy-training operators (plmpm_scan.hip, plmpm_norm.hip, plmpm_adamw.hip): element types and their conversions, vector
// loads and stores of VW neighbouring elements, sums over a wave and over the waves of a row.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>

#include "../../include/plmpm_policy.h"

int plmpm_fail(const char* fmt, ...);          // plmpm_capi.hip: sets the text of plmpm_last_error, returns -1
#define NN_REQUIRE(cond, ...) do { if (!(cond)) return plmpm_fail(__VA_ARGS__); } while (0)
#define NN_LAUNCHED(what)                                                                                           \
    do {                                                                                                            \
        hipError_t e_ = hipGetLastError();                                                                          \
        if (e_ != hipSuccess) return plmpm_fail("%s: launch failed: %s", what, hipGetErrorString(e_));              \
    } while (0)

namespace plbnn {

struct bf16 { uint16_t v; };
struct f16 { uint16_t v; };

__device__ __forceinline__ float as_f(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
__device__ __forceinline__ uint32_t as_u(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return as_f((uint32_t)x.v << 16); }
#if defined(PLB_HOST_EMUL)
inline float to_f(f16 x) {
    const uint32_t s = (uint32_t)(x.v & 0x8000) << 16, e = (x.v >> 10) & 31, m = x.v & 1023;
    if (e == 31) return as_f(s | 0x7f800000u | (m << 13));
    if (e) return as_f(s | ((e + 112) << 23) | (m << 13));
    const float f = (float)m * 5.9604644775390625e-8f;         // subnormal: m 2^-24
    return s ? -f : f;
}
inline void from_f(float f, bf16& o) {
    const uint32_t u = as_u(f);
    o.v = f != f ? 0x7fc0 : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
inline void from_f(float f, f16& o) {
    const uint32_t u = as_u(f), s = (u >> 16) & 0x8000;
    const float a = std::fabs(f);
    if (f != f) { o.v = 0x7e00; return; }
    if (a >= 65520.0f) { o.v = (uint16_t)(s | 0x7c00); return; }
    if (a < 6.103515625e-5f) { o.v = (uint16_t)(s | (uint32_t)std::nearbyint(a * 16777216.0f)); return; }
    const uint32_t b = as_u(a), r = b + 0xfffu + ((b >> 13) & 1);
    o.v = (uint16_t)(s | ((r - (112u << 23)) >> 13));
}
inline float exp2_fast(float x) { return exp2f(x); }
inline float fract_below_one(float x) { const float f = x - std::floor(x); return f > 0.999999940395355224609375f ? 0.999999940395355224609375f : f; }
inline void sleep_a_little() { __builtin_amdgcn_s_sleep(1); }
inline void wait_for_memory() {}
#else
__device__ __forceinline__ float to_f(f16 x) { _Float16 h; memcpy(&h, &x, 2); return (float)h; }
// round to nearest even, one conversion instruction each
__device__ __forceinline__ void from_f(float f, bf16& o) { const __bf16 h = (__bf16)f; memcpy(&o, &h, 2); }
__device__ __forceinline__ void from_f(float f, f16& o) { const _Float16 h = (_Float16)f; memcpy(&o, &h, 2); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }       // v_exp_f32: within 1 ulp; exponents below -126 give 0
__device__ __forceinline__ float fract_below_one(float x) { return __builtin_amdgcn_fractf(x); }        // v_fract_f32: at most the last float below 1
__device__ __forceinline__ void sleep_a_little() { __builtin_amdgcn_s_sleep(8); }        // 8 x 64 cycles
__device__ __forceinline__ void wait_for_memory() { __builtin_amdgcn_s_waitcnt(0x0f70); }       // vmcnt(0)
#endif
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }

// what comes of `f` is made anew from here on, as with Vec::forget
__device__ __forceinline__ void anew(float& f) {
#if !defined(PLB_HOST_EMUL)
    asm volatile("" : "+v"(f));
#endif
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// 1 / (1 + e^-x): both ends come out right by themselves (e^-x = inf -> 0, 0 -> 1)
__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-kLog2e * x)); }
// A sigmoid s and 1 - s in one number, each to its own last bits: the smaller of the two, q e with e = e^-|x| and q = 1 / (1 + e), with the sign of x.  (From a
// rounded s near 1 the difference cancels: 23 % off at x = 15.7, nothing left above 17.)  s is then what is left of its negative above a whole number,
// one instruction, and s (1 - s) one more.  The smaller side is never 0, whose negative has nothing left: 2^-126 is added where it is multiplied.
__device__ __forceinline__ float both_sides(float x) {
    const float e = exp2_fast(-kLog2e * fabsf(x)), q = __builtin_amdgcn_rcpf(1.0f + e);
    return copysignf(fmaf(e, q, 1.1754943508222875e-38f), x);
}
__device__ __forceinline__ float side_of(float both) { return fract_below_one(-both); }
__device__ __forceinline__ float product_of(float both) { const float t = fabsf(both); return fmaf(-t, t, t); }

// N neighbouring elements as one access of the widest type their bytes allow (up to 16; more: several).  LOOSE: at any element's address -- global
// memory takes accesses of 16 bytes at every alignment, and the compiler makes one of a packed type
template <int BYTES, bool LOOSE = false> struct Wide;
template <> struct Wide<2> { typedef uint16_t type; };
template <> struct Wide<4> { typedef uint32_t type; };
template <> struct Wide<8> { struct alignas(8) type { uint32_t w[2]; }; };
template <> struct Wide<16> { struct alignas(16) type { uint32_t w[4]; }; };
template <> struct Wide<4, true> { struct __attribute__((packed, aligned(2))) type { uint32_t w; }; };
template <> struct Wide<16, true> { struct __attribute__((packed, aligned(2))) type { uint32_t w[4]; }; };
template <class T, int N, bool LOOSE = false> struct Vec {
    static constexpr int bytes = N * (int)sizeof(T), part = bytes > 16 ? 16 : bytes, parts = bytes / part;
    typedef typename Wide<part, LOOSE>::type W;
    W w[parts];
#if !defined(PLB_HOST_EMUL)
    // the same bytes as a vector of words, as the builtins for such accesses take them
    typedef std::conditional_t<(part < 4), uint16_t, uint32_t> Word;
    typedef Word __attribute__((ext_vector_type(part < 4 ? 1 : part / 4), aligned(LOOSE ? 2 : part))) Past;
#endif
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int k = 0; k < parts; ++k) w[k] = reinterpret_cast<const W*>(p)[k];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int k = 0; k < parts; ++k) reinterpret_cast<W*>(p)[k] = w[k];
    }
    // past the caches, for what is not touched again soon: the cache then keeps what is
    __device__ __forceinline__ void load_past(const T* p) {
#if defined(PLB_HOST_EMUL)
        load(p);
#else
#pragma unroll
        for (int k = 0; k < parts; ++k) {
            const Past v = __builtin_nontemporal_load(reinterpret_cast<const Past*>(p) + k);
            memcpy(&w[k], &v, part);
        }
#endif
    }
    __device__ __forceinline__ void store_past(T* p) const {
#if defined(PLB_HOST_EMUL)
        store(p);
#else
#pragma unroll
        for (int k = 0; k < parts; ++k) {
            Past v;
            memcpy(&v, &w[k], part);
            __builtin_nontemporal_store(v, reinterpret_cast<Past*>(p) + k);
        }
#endif
    }
    __device__ __forceinline__ void zero() { memset(w, 0, sizeof(w)); }
    // the elements move down by `n`, zeros behind them (a vector of 4 bytes)
    __device__ __forceinline__ void drop(int n) {
        static_assert(bytes == 4, "one word");
        uint32_t u;
        memcpy(&u, w, 4);
        u >>= 8 * sizeof(T) * n;
        memcpy(w, &u, 4);
    }
    // unpack from here on (else the compiler keeps the floats of an earlier or a later get, twice the registers where elements have 16 bits)
    __device__ __forceinline__ void forget() {
#if !defined(PLB_HOST_EMUL)
        if constexpr (bytes % 4 == 0) {
            uint32_t u[bytes / 4];
            memcpy(u, w, bytes);
#pragma unroll
            for (int k = 0; k < bytes / 4; ++k) asm("" : "+v"(u[k]));
            memcpy(w, u, bytes);
        }
#endif
    }
    __device__ __forceinline__ void get(float* f) const {
        T e[N];
        memcpy(e, w, sizeof(w));
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = to_f(e[k]);
    }
    __device__ __forceinline__ void set(const float* f) {
        T e[N];
#pragma unroll
        for (int k = 0; k < N; ++k) from_f(f[k], e[k]);
        memcpy(w, e, sizeof(w));
    }
};

// a row's address, the same for the whole wave, plus a lane's 32-bit offset: the empty asm keeps the row's address in scalar registers (the compiler
// would otherwise add row and offset once a lane in 64 bits, and hold two vector registers for each of the loads in flight)
template <class T> __device__ __forceinline__ T* at_offset(T* row, unsigned bytes) {
#if defined(PLB_HOST_EMUL)
    return (T*)((char*)row + bytes);
#else
    typedef char __attribute__((address_space(1))) * Global;
    const uint64_t r = (uint64_t)row;
    unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)r), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(r >> 32));
    uint64_t u = ((uint64_t)hi << 32) | lo;
    asm("" : "+s"(u));
    return (T*)(char*)((Global)u + bytes);
#endif
}

// sums over groups of n neighbouring lanes (n a power of two up to 64, the same for the wave), every lane gets its group's: steps within 16 lanes
// are DPP moves (a lane's partner in its pair, its four, its eight, its sixteen), the two above go through LDS crossbar shuffles
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return as_f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)as_u(v), CTRL, 0xf, 0xf, true));
}
template <int K> __device__ __forceinline__ void lane_sums(float (&v)[K], int n) {
    if (n >= 2)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += dpp<0xB1>(v[k]);           // quad_perm 1 0 3 2
    if (n >= 4)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += dpp<0x4E>(v[k]);           // quad_perm 2 3 0 1
    if (n >= 8)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += dpp<0x141>(v[k]);          // row_half_mirror
    if (n >= 16)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += dpp<0x140>(v[k]);          // row_mirror
    if (n >= 32)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], 16);
    if (n >= 64)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], 32);
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, dpp<0xB1>(v));
    v = max(v, dpp<0x4E>(v));
    v = max(v, dpp<0x141>(v));
    v = max(v, dpp<0x140>(v));
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

// host side: bytes that a pointer and a stride (in elements) both keep to
inline int aligned_to(const void* p, int64_t stride, int size) {
    const uint64_t a = (uint64_t)(uintptr_t)p | ((uint64_t)stride * (uint64_t)size);
    return (a & 15) == 0 ? 16 : (a & 7) == 0 ? 8 : (a & 3) == 0 ? 4 : (a & 1) == 0 ? 2 : 1;
}
inline int dtype_size(int dtype) { return dtype == PLMPM_NN_F32 ? 4 : 2; }
inline size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

}  // namespace plbnn
