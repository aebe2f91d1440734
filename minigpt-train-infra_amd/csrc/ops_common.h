// ops_common.h -- what the training-step operators' kernels share: element
// types, vector accesses, reductions over lanes, error returns.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "mgopt.h"
#include "mgopt_ops.h"

namespace mgopt {

// Sets the text mgopt_last_error returns on this thread and hands back `code` (mgopt.hip).
int set_error(int code, const std::string& msg);

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error(static_cast<int>(e), std::string(what) + ": " + hipGetErrorString(e));
}

inline bool known_dtype(int32_t d) { return d == MGOPT_F32 || d == MGOPT_F16 || d == MGOPT_BF16; }
inline int dtype_bytes(int32_t d) { return d == MGOPT_F32 ? 4 : 2; }

// A dispatch counts its work-items in 32 bits: the most work-groups of `block` threads that one launch takes.
constexpr uint32_t max_blocks(uint32_t block) { return 0xFFFFFFFFu / block; }

// Calls f with a value of the element type that `dtype` names.
template <typename F>
int with_dtype(int32_t dtype, F&& f) {
    switch (dtype) {
        case MGOPT_F32: return f(float{});
        case MGOPT_F16: return f(_Float16{});
        case MGOPT_BF16: return f(__bf16{});
        default: return set_error(MGOPT_E_INVALID, "bad dtype " + std::to_string(dtype));
    }
}

// N consecutive elements as one access.  The type asks for the element's own
// alignment only: gfx950 takes vector accesses at any address, so rows of odd
// strides keep 16-byte accesses.
template <typename T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
using vec_t = typename Vec<T, N>::type;

template <int N, typename T>
__device__ __forceinline__ void load(float (&f)[N], const T* p) {
    const vec_t<T, N> v = *reinterpret_cast<const vec_t<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = static_cast<float>(v[i]);
}

// Streamed data that nothing reads again soon.
template <int N, typename T>
__device__ __forceinline__ void load_nt(float (&f)[N], const T* p) {
    const vec_t<T, N> v = __builtin_nontemporal_load(reinterpret_cast<const vec_t<T, N>*>(p));
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = static_cast<float>(v[i]);
}

template <int N, typename T>
__device__ __forceinline__ void store(T* p, const float (&f)[N]) {
    vec_t<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<T>(f[i]);
    *reinterpret_cast<vec_t<T, N>*>(p) = v;
}

template <int N, typename T>
__device__ __forceinline__ void store_nt(T* p, const float (&f)[N]) {
    vec_t<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<T>(f[i]);
    __builtin_nontemporal_store(v, reinterpret_cast<vec_t<T, N>*>(p));
}

// The first n of N elements (n may exceed N or be negative), zeros for the others.
template <int N, bool NT = false, typename T>
__device__ __forceinline__ void load_some(float (&f)[N], const T* p, int64_t n) {
    if (n >= N) {
        if constexpr (NT) load_nt<N>(f, p);
        else load<N>(f, p);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
}

template <int N, bool NT = false, typename T>
__device__ __forceinline__ void store_some(T* p, const float (&f)[N], int64_t n) {
    if (n >= N) {
        if constexpr (NT) store_nt<N>(p, f);
        else store<N>(p, f);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) p[i] = static_cast<T>(f[i]);
}

// x of the lane that the DPP control word names, within rows of 16 lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(dpp<CTRL>(__float_as_uint(x)));
}
constexpr int kDppXor1 = 0xB1;         // quad_perm [1,0,3,2]
constexpr int kDppXor2 = 0x4E;         // quad_perm [2,3,0,1]
constexpr int kDppHalfMirror = 0x141;  // lane i of 8 takes lane 7 - i: the other quad, once quads are uniform
constexpr int kDppMirror = 0x140;      // lane i of 16 takes lane 15 - i: the other eight, once eights are uniform

// op over aligned groups of LANES lanes, the result in each of them, in a fixed order.
template <int LANES, typename X, typename Op>
__device__ __forceinline__ X reduce_lanes(X x, Op op) {
    if constexpr (LANES > 1) x = op(x, dpp<kDppXor1>(x));
    if constexpr (LANES > 2) x = op(x, dpp<kDppXor2>(x));
    if constexpr (LANES > 4) x = op(x, dpp<kDppHalfMirror>(x));
    if constexpr (LANES > 8) x = op(x, dpp<kDppMirror>(x));
    if constexpr (LANES > 16) x = op(x, __shfl_xor(x, 16));
    if constexpr (LANES > 32) x = op(x, __shfl_xor(x, 32));
    return x;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32: 1 ulp, tiny results to 0
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }    // v_rcp_f32: 1 ulp, tiny results to 0

// An id of a list of 4- or 8-byte signed integers.
__device__ __forceinline__ int64_t id_at(const void* p, int64_t i, int bytes) {
    return bytes == 8 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

}  // namespace mgopt
