// ops_rms_norm.hip -- the residual's addition and the RMS norm of the sum, its
// backward pass, its output in 8 bits, and rows of any tensor in 8 bits.
//
//     h = round(x + residual)        r = 1 / sqrt(mean(h^2) + eps)        y = (h * r) * weight
//
// h is rounded to the stream's type before it is normed, so that the backward
// pass, which reads the stored h, differentiates what was computed.  With g the
// gradient of y, gw = g * weight and xhat = h * r:
//
//     dx = grad_h + r * (gw - xhat * mean(gw * xhat))        dweight = sum g * xhat
//
// and dx is the gradient of x and of the residual alike.
//
// In 8 bits: with m the largest magnitude of a row of y, scale = m * (1/127) and
// codes = the integers nearest to y * (127 / m), ties to even, all in fp32 and y
// not rounded to the stream's type.  A row with an inf or a NaN has the scale NaN,
// one whose m is below 2^-119, where 127 / m could overflow, counts as zeros.
//
// mean(h^2) is summed in 64 bits: squares of 32-bit values neither overflow nor
// underflow there, and r, rounded to 32 bits once, does not hang on the order of
// the sum but in one of some 2^28 rows, so that the codes are the format's and not
// this kernel's.
//
// The backward pass norms a row before it sums gw * xhat, though a sum of gw * h
// beside the squares' saves a join of the waves: with h near its type's largest values
// that sum passes 32 bits.  On the same inputs over and over, with and without it: 8,192
// rows of 4,096 in bf16 46.5 and 45.7 us, 4,096 of 16,384 119 and 128, 2,048 of 32,768
// in fp32 340 and 301.  (The sum of gw * h in 64 bits: 47, 157 and 342, for the registers.)
//
// Bound by memory.  A row is read once and held by one wave, 256 or 1,024 threads,
// whichever needs no more than a few vectors of 16 bytes a thread.  8,192 rows of
// 4,096 in bf16: 46 us forward (5.9 TB/s); 75 us backward (3.6 TB/s with the weight's
// partial sums) and 8 for the sums of those.  The backward pass with 512 threads a row
// took 79 us and with each next row's loads ahead of this row's sums 85, where this one
// took 72: both cost more registers than they hide latency.
//
// Wide rows do not stay in the registers of 1,024 threads, 128 each: forward, fp32 rows
// over 16,384 in 8 bits spill 12 of them; backward, rows over 16,384 spill 106 (fp32) and
// 118 (2 bytes), fp32 rows over 8,192 23.  On the same inputs over and over, backward:
// 4,096 x 8,192 in bf16 70 us (2.9 TB/s), 4,096 x 16,384 119 (3.4), 2,048 x 32,768 301 (1.3);
// in fp32 100 (4.0), 187 (4.3) and 340 (2.4).
#include "ops_common.h"

namespace mgopt {
namespace {

constexpr float kTiny = 0x1p-119f;
constexpr int kMaxWidth = MGOPT_MAX_NORM_WIDTH;

// N values of a weight of any of the types.
template <int N>
__device__ __forceinline__ void load_weight(float (&f)[N], const void* w, int32_t dtype, int64_t at, int64_t n) {
    if (dtype == MGOPT_F32) load_some<N>(f, static_cast<const float*>(w) + at, n);
    else if (dtype == MGOPT_F16) load_some<N>(f, static_cast<const _Float16*>(w) + at, n);
    else load_some<N>(f, static_cast<const __bf16*>(w) + at, n);
}

// The sum of x over a work-group of BLOCK threads in a fixed order, in each of them; `part` is free again
// when all threads have passed the next barrier.
template <int BLOCK, typename X>
__device__ __forceinline__ X block_sum(X x, X (&part)[BLOCK / 64]) {
    if constexpr (sizeof(X) == 4) {
        x = reduce_lanes<64>(x, [](X a, X b) { return a + b; });
    } else {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d);
    }
    if constexpr (BLOCK > 64) {
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
        __syncthreads();
        x = part[0];
#pragma unroll
        for (int i = 1; i < BLOCK / 64; ++i) x += part[i];
    }
    return x;
}
template <int BLOCK>
__device__ __forceinline__ uint32_t block_max(uint32_t x, uint32_t* part) {
    x = reduce_lanes<64>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
    if constexpr (BLOCK > 64) {
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
        __syncthreads();
        x = part[0];
#pragma unroll
        for (int i = 1; i < BLOCK / 64; ++i) x = max(x, part[i]);
    }
    return x;
}

// The scale of a row whose largest magnitude has the bits m (NaN above inf), and what its values are
// multiplied by for their codes.
struct Scale {
    float scale, inv;
    bool finite;
};
__device__ __forceinline__ Scale scale_of(uint32_t m) {
    const float most = __uint_as_float(m);
    const bool finite = m < 0x7F800000u, zero = most < kTiny;
    return {finite ? (zero ? 0.0f : most * (1.0f / 127.0f)) : __uint_as_float(0x7FC00000u),
            finite && !zero ? 127.0f / most : 0.0f, finite};
}
template <int N>
__device__ __forceinline__ void store_codes(int8_t* at, const float (&y)[N], const Scale& s) {
    uint32_t word[N / 4];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float c = s.finite ? rintf(y[i + k] * s.inv) : 0.0f;
            w |= (static_cast<uint32_t>(static_cast<int>(c)) & 0xFFu) << (8 * k);
        }
        word[i / 4] = w;
    }
    if constexpr (N == 8) *reinterpret_cast<uint2*>(at) = make_uint2(word[0], word[1]);
    else *reinterpret_cast<uint32_t*>(at) = word[0];
}

struct NormArgs {
    const void *x, *residual, *weight;
    int64_t x_stride, residual_stride;
    int64_t rows, width, first_row;
    double eps;
    void *h, *y;
    int8_t* codes;
    int64_t codes_stride;
    float* scales;
    int32_t weight_dtype;
    // backward: x is the gradient of y, residual that of h or NULL, h the stream
    const void* stream;
    int64_t stream_stride;
    void* dx;
    float* partials;        // [work-groups][width], or NULL
};

__device__ __forceinline__ float rstd_of(double sum, int64_t width, double eps) {
    return static_cast<float>(1.0 / sqrt(sum / static_cast<double>(width) + eps));
}

// A row a work-group, NV vectors of N elements a thread.
template <typename T, int BLOCK, int NV, bool CODES>
__global__ __launch_bounds__(BLOCK) void rms_norm_kernel(NormArgs a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ double part[BLOCK / 64];
    __shared__ uint32_t top[BLOCK / 64];
    const int64_t row = a.first_row + blockIdx.x;
    float h[NV][N];
    double sum = 0.0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N, n = a.width - at;
        load_some<N>(h[v], static_cast<const T*>(a.x) + row * a.x_stride + at, n);
        if (a.residual != nullptr) {
            float s[N];
            load_some<N>(s, static_cast<const T*>(a.residual) + row * a.residual_stride + at, n);
#pragma unroll
            for (int i = 0; i < N; ++i) h[v][i] = static_cast<float>(static_cast<T>(h[v][i] + s[i]));
            store_some<N>(static_cast<T*>(a.h) + row * a.width + at, h[v], n);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fma(static_cast<double>(h[v][i]), static_cast<double>(h[v][i]), sum);
    const float r = rstd_of(block_sum<BLOCK>(sum, part), a.width, a.eps);
    uint32_t m = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N, n = a.width - at;
        float w[N];
        load_weight<N>(w, a.weight, a.weight_dtype, at, n);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // beyond the width h is 0 and its product with an infinite r (eps 0, a row of zeros) NaN
            h[v][i] = i < n ? h[v][i] * r * w[i] : 0.0f;
            if constexpr (CODES) m = max(m, __float_as_uint(h[v][i]) & 0x7FFFFFFFu);
        }
        if constexpr (!CODES) store_some<N>(static_cast<T*>(a.y) + row * a.width + at, h[v], n);
    }
    if constexpr (CODES) {
        const Scale s = scale_of(block_max<BLOCK>(m, top));
        if (threadIdx.x == 0) a.scales[row] = s.scale;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N;
            if (at < a.codes_stride) store_codes<N>(a.codes + row * a.codes_stride + at, h[v], s);
        }
    }
}

// Rows of a work-group's own, `gridDim.x` apart; each thread keeps the sums of its columns' weight
// gradients over them.
template <typename T, int BLOCK, int NV>
__global__ __launch_bounds__(BLOCK) void rms_norm_backward_kernel(NormArgs a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ double squares[2][BLOCK / 64];
    __shared__ float dots[2][BLOCK / 64];
    float dw[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) dw[v][i] = 0.0f;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        float h[NV][N], g[NV][N];
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N, n = a.width - at;
            load_some<N>(h[v], static_cast<const T*>(a.stream) + row * a.stream_stride + at, n);
            load_some<N>(g[v], static_cast<const T*>(a.x) + row * a.x_stride + at, n);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) sum = fma(static_cast<double>(h[v][i]), static_cast<double>(h[v][i]), sum);
        // two sets of partial sums in turn: a wave that is a row ahead writes the other one
        const float r = rstd_of(block_sum<BLOCK>(sum, squares[turn]), a.width, a.eps);
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N, n = a.width - at;
            float w[N];
            load_weight<N>(w, a.weight, a.weight_dtype, at, n);
#pragma unroll
            for (int i = 0; i < N; ++i) dot = fmaf(g[v][i] * w[i], h[v][i] * r, dot);
        }
        const float mean = block_sum<BLOCK>(dot, dots[turn]) / static_cast<float>(a.width);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N, n = a.width - at;
            float w[N], d[N];
            load_weight<N>(w, a.weight, a.weight_dtype, at, n);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float xhat = h[v][i] * r;
                dw[v][i] = fmaf(g[v][i], xhat, dw[v][i]);
                d[i] = r * (g[v][i] * w[i] - xhat * mean);
            }
            if (a.residual != nullptr) {
                load_some<N>(w, static_cast<const T*>(a.residual) + row * a.residual_stride + at, n);
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] += w[i];
            }
            store_some<N>(static_cast<T*>(a.dx) + row * a.width + at, d, n);
        }
    }
    if (a.partials == nullptr) return;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int64_t at = (static_cast<int64_t>(v) * BLOCK + threadIdx.x) * N;
        store_some<N>(a.partials + blockIdx.x * a.width + at, dw[v], a.width - at);
    }
}

// Sums the rows of partial weight gradients: a work-group takes kCols columns, its threads rows in turn,
// joined in a fixed order.
constexpr int kCols = 16, kSumBlock = 1024;
__global__ __launch_bounds__(kSumBlock) void norm_weight_kernel(const float* partials, uint32_t rows, int64_t width, void* dw,
                                                                int32_t dtype) {
    __shared__ float part[kSumBlock / kCols][kCols + 1];
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
    const int64_t e = static_cast<int64_t>(blockIdx.x) * kCols + col;
    float x = 0.0f;
    if (e < width) {
#pragma unroll 8
        for (uint32_t r = row; r < rows; r += kSumBlock / kCols) x += partials[static_cast<int64_t>(r) * width + e];
    }
    part[row][col] = x;
    __syncthreads();
    for (int half = kSumBlock / kCols / 2; half > 0; half /= 2) {
        if (row < half) part[row][col] += part[row + half][col];
        __syncthreads();
    }
    if (row != 0 || e >= width) return;
    x = part[0][col];
    if (dtype == MGOPT_F32) static_cast<float*>(dw)[e] = x;
    else if (dtype == MGOPT_F16) static_cast<_Float16*>(dw)[e] = static_cast<_Float16>(x);
    else static_cast<__bf16*>(dw)[e] = static_cast<__bf16>(x);
}

// Rows of any width to codes: read twice, the second time from the cache.
template <typename T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void int8_rows_kernel(NormArgs a) {
    constexpr int N = 16 / sizeof(T);
    __shared__ uint32_t top[BLOCK / 64];
    const int64_t row = a.first_row + blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    uint32_t m = 0;
    float f[N];
    for (int64_t at = threadIdx.x * N; at < a.width; at += BLOCK * N) {
        load_some<N>(f, x + at, a.width - at);
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    }
    const Scale s = scale_of(block_max<BLOCK>(m, top));
    if (threadIdx.x == 0) a.scales[row] = s.scale;
    for (int64_t at = threadIdx.x * N; at < a.codes_stride; at += BLOCK * N) {
        load_some<N>(f, x + at, a.width - at);
        store_codes<N>(a.codes + row * a.codes_stride + at, f, s);
    }
}

template <int V>
using Int = std::integral_constant<int, V>;

// Threads of a row, and vectors of N elements a thread.
template <int N, typename F>
int with_shape(int64_t width, F&& f) {
    const int64_t vecs = (width + N - 1) / N;
    if (vecs <= 64) return f(Int<64>{}, Int<1>{});
    if (vecs <= 128) return f(Int<64>{}, Int<2>{});
    if (vecs <= 256) return f(Int<256>{}, Int<1>{});
    if (vecs <= 512) return f(Int<256>{}, Int<2>{});
    if (vecs <= 1024) return f(Int<256>{}, Int<4>{});
    if (vecs <= 2048) return f(Int<1024>{}, Int<2>{});
    if constexpr (kMaxWidth / N > 4096)
        if (vecs > 4096) return f(Int<1024>{}, Int<8>{});
    return f(Int<1024>{}, Int<4>{});
}

// The launches that cover the rows, one work-group each, in pieces of at most a grid.
template <typename F>
int over_rows(NormArgs& a, int block, const char* what, F&& launch) {
    const int64_t piece = max_blocks(static_cast<uint32_t>(block));
    for (a.first_row = 0; a.first_row < a.rows; a.first_row += piece) {
        launch(dim3(static_cast<uint32_t>(std::min(piece, a.rows - a.first_row))));
        if (int rc = launched(what)) return rc;
    }
    return 0;
}

int check(const char* what, int32_t dtype, int64_t rows, int64_t width, double eps) {
    const std::string w(what);
    if (!known_dtype(dtype)) return set_error(MGOPT_E_INVALID, w + ": bad dtype");
    if (rows < 0 || width < 1) return set_error(MGOPT_E_INVALID, w + ": need rows >= 0 and width >= 1");
    if (!(eps >= 0.0)) return set_error(MGOPT_E_INVALID, w + ": eps must not be negative");
    return 0;
}
int check_codes(const char* what, const int8_t* codes, int64_t stride, int64_t width) {
    if (stride < width || stride % 16 != 0 || reinterpret_cast<uintptr_t>(codes) % 16 != 0)
        return set_error(MGOPT_E_ALIGN, std::string(what) + ": rows of codes need a 16-byte aligned place and stride");
    if (stride - width >= 16) return set_error(MGOPT_E_INVALID, std::string(what) + ": codes_stride is the width rounded up to 16");
    return 0;
}

// Work-groups of the backward pass, each with a row of partial weight gradients: 8 waves a compute unit where a
// row is one wave's, 16 or more for the others.  8,192 rows of 4,096 in bf16, with the sums of the partial
// rows: 80 us with 1,024 work-groups, 109 with 512 and 163 with 256, whose waves do not cover the memory's
// latency.
uint32_t backward_blocks(int64_t rows, int64_t width) {
    const int64_t most = width <= 1024 ? 2048 : width <= 8192 ? 1024 : 256;
    return static_cast<uint32_t>(std::max<int64_t>(1, std::min(rows, most)));
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int mgopt_rms_norm(const void* x_dev, int64_t x_stride, const void* residual_dev, int64_t residual_stride,
                             const void* weight_dev, int32_t weight_dtype, int32_t dtype, int64_t rows, int64_t width,
                             double eps, void* h_dev, void* y_dev, int8_t* codes_dev, int64_t codes_stride, float* scales_dev,
                             void* stream) {
    if (int rc = check("rms_norm", dtype, rows, width, eps)) return rc;
    if (!known_dtype(weight_dtype)) return set_error(MGOPT_E_INVALID, "rms_norm: bad dtype");
    if (width > kMaxWidth) return set_error(MGOPT_E_LIMIT, "rms_norm: rows of more than " + std::to_string(kMaxWidth) + " elements");
    if ((y_dev == nullptr) == (codes_dev == nullptr) && rows > 0)
        return set_error(MGOPT_E_INVALID, "rms_norm: exactly one of y_dev and codes_dev");
    if (rows == 0) return 0;
    if (!x_dev || !weight_dev || (residual_dev == nullptr) != (h_dev == nullptr) || (codes_dev == nullptr) != (scales_dev == nullptr))
        return set_error(MGOPT_E_INVALID, "rms_norm: NULL argument");
    if (codes_dev)
        if (int rc = check_codes("rms_norm", codes_dev, codes_stride, width)) return rc;
    NormArgs a{};
    a.x = x_dev, a.x_stride = x_stride, a.residual = residual_dev, a.residual_stride = residual_stride;
    a.weight = weight_dev, a.weight_dtype = weight_dtype, a.rows = rows, a.width = width, a.eps = eps;
    a.h = h_dev, a.y = y_dev, a.codes = codes_dev, a.codes_stride = codes_stride, a.scales = scales_dev;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int N = 16 / sizeof(T);
        // codes fill their rows up to the stride
        return with_shape<N>(codes_dev ? codes_stride : width, [&](auto block, auto nv) {
            constexpr int B = decltype(block)::value, NV = decltype(nv)::value;
            return over_rows(a, B, "rms_norm", [&](dim3 grid) {
                if (codes_dev) hipLaunchKernelGGL((rms_norm_kernel<T, B, NV, true>), grid, dim3(B), 0, s, a);
                else hipLaunchKernelGGL((rms_norm_kernel<T, B, NV, false>), grid, dim3(B), 0, s, a);
            });
        });
    });
}

MGOPT_API int64_t mgopt_rms_norm_workspace(int64_t rows, int64_t width) {
    if (rows < 0 || width < 1 || width > kMaxWidth) return -1;
    return static_cast<int64_t>(backward_blocks(rows, width)) * width * 4;
}

MGOPT_API int mgopt_rms_norm_backward(const void* grad_y_dev, int64_t grad_y_stride, const void* grad_h_dev,
                                      int64_t grad_h_stride, const void* h_dev, int64_t h_stride, const void* weight_dev,
                                      int32_t weight_dtype, int32_t dtype, int64_t rows, int64_t width, double eps,
                                      void* d_x_dev, void* d_weight_dev, void* workspace_dev, void* stream) {
    if (int rc = check("rms_norm_backward", dtype, rows, width, eps)) return rc;
    if (!known_dtype(weight_dtype)) return set_error(MGOPT_E_INVALID, "rms_norm_backward: bad dtype");
    if (width > kMaxWidth)
        return set_error(MGOPT_E_LIMIT, "rms_norm_backward: rows of more than " + std::to_string(kMaxWidth) + " elements");
    if (rows > 0 && (!grad_y_dev || !h_dev || !weight_dev || !d_x_dev))
        return set_error(MGOPT_E_INVALID, "rms_norm_backward: NULL argument");
    if (d_weight_dev && (!workspace_dev || reinterpret_cast<uintptr_t>(workspace_dev) % 16 != 0))
        return set_error(MGOPT_E_ALIGN, "rms_norm_backward: the workspace must be 16-byte aligned and not NULL");
    NormArgs a{};
    a.x = grad_y_dev, a.x_stride = grad_y_stride, a.residual = grad_h_dev, a.residual_stride = grad_h_stride;
    a.stream = h_dev, a.stream_stride = h_stride, a.weight = weight_dev, a.weight_dtype = weight_dtype;
    a.rows = rows, a.width = width, a.eps = eps, a.dx = d_x_dev;
    a.partials = d_weight_dev ? static_cast<float*>(workspace_dev) : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t blocks = backward_blocks(rows, width);
    if (rows > 0) {
        const int rc = with_dtype(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int N = 16 / sizeof(T);
            return with_shape<N>(width, [&](auto block, auto nv) {
                constexpr int B = decltype(block)::value, NV = decltype(nv)::value;
                hipLaunchKernelGGL((rms_norm_backward_kernel<T, B, NV>), dim3(blocks), dim3(B), 0, s, a);
                return launched("rms_norm_backward");
            });
        });
        if (rc) return rc;
    }
    if (!d_weight_dev) return 0;
    hipLaunchKernelGGL(norm_weight_kernel, dim3(static_cast<uint32_t>((width + kCols - 1) / kCols)), dim3(kSumBlock), 0, s,
                       static_cast<const float*>(workspace_dev), rows > 0 ? blocks : 0, width, d_weight_dev, weight_dtype);
    return launched("rms_norm_backward");
}

MGOPT_API int mgopt_int8_rows(const void* x_dev, int64_t x_stride, int32_t dtype, int64_t rows, int64_t width,
                              int8_t* codes_dev, int64_t codes_stride, float* scales_dev, void* stream) {
    if (int rc = check("int8_rows", dtype, rows, width, 0.0)) return rc;
    if (rows == 0) return 0;
    if (!x_dev || !codes_dev || !scales_dev) return set_error(MGOPT_E_INVALID, "int8_rows: NULL argument");
    if (int rc = check_codes("int8_rows", codes_dev, codes_stride, width)) return rc;
    NormArgs a{};
    a.x = x_dev, a.x_stride = x_stride, a.rows = rows, a.width = width;
    a.codes = codes_dev, a.codes_stride = codes_stride, a.scales = scales_dev;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto block) {
            constexpr int B = decltype(block)::value;
            return over_rows(a, B, "int8_rows", [&](dim3 grid) {
                hipLaunchKernelGGL((int8_rows_kernel<T, B>), grid, dim3(B), 0, s, a);
            });
        };
        return width <= 1024 ? go(Int<64>{}) : go(Int<256>{});
    });
}

}  // extern "C"
