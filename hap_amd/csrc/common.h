// Shared helpers of the gfx950 kernels: error reporting, element access, launch checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdarg.h>

#include <initializer_list>

#include "../../include/hapmi.h"

typedef __bf16 bf16_t;
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define HAPMI_WAVE 64

int hapmi_set_error(int code, const char *fmt, ...);
int hapmi_sumsq_static_setup();   // elementwise.hip: per-device set-up that hapmi_init runs

#define HAPMI_REQUIRE(cond, code, ...)                           \
    do {                                                         \
        if (!(cond)) return hapmi_set_error((code), __VA_ARGS__); \
    } while (0)

// Refuses outputs that share memory with each other or with an operand that is read (operands that are only read may share).
struct HapmiSpan {
    const void *at;                 // NULL: no such operand
    int64_t bytes;                  // from the first byte to behind the last one
    int64_t row = 0, pitch = 0;     // a strided matrix: bytes of a row, from row to row (0: the whole span is used)
};
// Whether two spans share a byte.  A matrix leaves the gaps between its rows to others: columns beside it in the same buffer
// (equal pitch), or something that fits into one gap.  Matrices of different pitches whose ranges meet count as sharing.
inline bool hapmi_meet(const HapmiSpan &a, const HapmiSpan &b) {
    const uintptr_t x = (uintptr_t)a.at, y = (uintptr_t)b.at;
    if (!x || !y || a.bytes <= 0 || b.bytes <= 0) return false;
    if (x <= y ? y - x >= (uintptr_t)a.bytes : x - y >= (uintptr_t)b.bytes) return false;
    if (a.pitch != b.pitch && a.pitch && b.pitch) return true;
    const uintptr_t pitch = (uintptr_t)(a.pitch ? a.pitch : b.pitch);
    if (!pitch) return true;
    const uintptr_t ra = a.pitch ? (uintptr_t)a.row : (uintptr_t)a.bytes, rb = b.pitch ? (uintptr_t)b.row : (uintptr_t)b.bytes;
    // b's rows begin `d` bytes behind a's, within a pitch: apart if they begin behind a's row and end before a's next one
    const uintptr_t d = x <= y ? (y - x) % pitch : (pitch - (x - y) % pitch) % pitch;
    return d < ra || d + rb > pitch;
}
inline int hapmi_apart(const char *name, std::initializer_list<HapmiSpan> written, std::initializer_list<HapmiSpan> read) {
    for (auto w = written.begin(); w != written.end(); ++w) {
        for (auto o = w + 1; o != written.end(); ++o) HAPMI_REQUIRE(!hapmi_meet(*w, *o), HAPMI_EALIAS, "%s: an output shares memory with another operand", name);
        for (auto &r : read) HAPMI_REQUIRE(!hapmi_meet(*w, r), HAPMI_EALIAS, "%s: an output shares memory with another operand", name);
    }
    return HAPMI_OK;
}

#define HAPMI_CHECK_LAUNCH(name)                                                        \
    do {                                                                                \
        hipError_t e__ = hipGetLastError();                                             \
        if (e__ != hipSuccess)                                                          \
            return hapmi_set_error(HAPMI_ELAUNCH, "%s: %s", (name), hipGetErrorString(e__)); \
    } while (0)

static inline int hapmi_dtype_ok(int dtype) { return dtype == HAPMI_F32 || dtype == HAPMI_BF16; }
static inline int64_t hapmi_elem_size(int dtype) { return dtype == HAPMI_F32 ? 4 : 2; }
static inline int64_t hapmi_cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// element load/store as float for either storage type
template <typename T> __device__ __forceinline__ float ld_f(const T *p, int64_t i);
template <> __device__ __forceinline__ float ld_f<float>(const float *p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float ld_f<bf16_t>(const bf16_t *p, int64_t i) { return (float)p[i]; }
template <typename T> __device__ __forceinline__ void st_f(T *p, int64_t i, float v);
template <> __device__ __forceinline__ void st_f<float>(float *p, int64_t i, float v) { p[i] = v; }
template <> __device__ __forceinline__ void st_f<bf16_t>(bf16_t *p, int64_t i, float v) { p[i] = (bf16_t)v; }

// 16-byte vector of elements: 4 floats or 8 bf16
template <typename T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int N = 4;
    f32x4 v;
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};
template <> struct Vec16<bf16_t> {
    static constexpr int N = 8;
    bf16x8 v;
    __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
    __device__ __forceinline__ void set(int i, float x) { v[i] = (bf16_t)x; }
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

// sum over an aligned group of 2^group_log2 <= 64 lanes, in every lane: exchanges inside a row of 16 lanes ride on the additions
// (DPP: neighbours, pairs, then mirrors, whose lanes hold equal sums), the last two cross rows
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float group_sum(float v, int group_log2) {
    if (group_log2 > 0) v = dpp_add<0xb1>(v);              // quad_perm [1, 0, 3, 2]
    if (group_log2 > 1) v = dpp_add<0x4e>(v);              // quad_perm [2, 3, 0, 1]
    if (group_log2 > 2) v = dpp_add<0x141>(v);             // row_half_mirror
    if (group_log2 > 3) v = dpp_add<0x140>(v);             // row_mirror
    if (group_log2 > 4) v += __shfl_xor(v, 16, 64);
    if (group_log2 > 5) v += __shfl_xor(v, 32, 64);
    return v;
}

// block-wide reductions for blocks of up to 1024 threads (16 waves); `red` is 16 floats of LDS
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = wave_sum(v);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nw = (blockDim.x + 63) >> 6;
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    float t = 0.f;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}
__device__ __forceinline__ float block_max(float v, float *red) {
    v = wave_max(v);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, nw = (blockDim.x + 63) >> 6;
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < nw; ++i) t = fmaxf(t, red[i]);
    return t;
}
