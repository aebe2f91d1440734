// ops_gated_act.hip -- the MLP's activation with an 8-bit checkpoint.
//
// Forward: y = act(gate) * up, or act(gate) without a gate, and, for a
// training pass, what the backward pass needs of the inputs in 8 bits.
// Backward: with the checkpoint's g and u,
//
//     d_gate = dy * u * act'(g)    d_up = dy * act(g)    y = act(g) * u
//
// the last for the weight gradient of the projection that follows, so that a
// program keeps neither gate, up nor y between the passes.
//
// Checkpoint: groups of 128 elements along a row share a scale.  With the
// group's largest magnitude m: scale = m * (1/127), code = the integer nearest
// to x * (127 / m), ties to even, all in fp32.  A group with an inf or a NaN
// has the scale NaN, so that its gradients do too (a loss scaler skips such a
// step); one whose m is below 2^-119, where 127 / m could overflow, counts as zeros.
//
// Bound by memory: forward moves (2 + 1) * b + 2 * (1 + 4/128) bytes per
// element of b bytes, backward (1 + 3) * b + 2 * (1 + 4/128).  8,192 rows of
// 12,288 in bf16: 133 us forward (6.1 TB/s), 179 us backward (5.7).
// A lane takes 16 bytes of each input, 16 or 32 lanes a group of 128, so that a
// group's largest magnitude is a few exchanges within a wave.
#include "ops_common.h"

namespace mgopt {
namespace {

// One wave a work-group, which starts as soon as any SIMD has room: against 256
// threads, at 8,192 rows of 12,288 in bf16, 180 against 189 us for the backward
// pass; at 2,049 of 2,731 in fp16, 12.1 against 14.1 for each.
constexpr int kActBlock = 64;
// A forward pass that moves more than the Infinity Cache holds reads its inputs
// and writes y past the caches: 133 against 145 us at 8,192 rows of 12,288 in
// bf16.  A backward pass right behind it finds less of what it reads in the cache,
// 179 against 167 us, so that the two alone take the same; in a training step
// other passes lie between.  On 100 MB in fp16, whose inputs are still cached, such
// loads cost 15.2 against 12.2 us, and in the backward pass, with its three
// outputs, they and such stores never paid.
constexpr int64_t kStreamBytes = int64_t{256} << 20;
constexpr int kGroup = MGOPT_ACT_GROUP;  // elements per scale
constexpr float kTiny = 0x1p-119f;
constexpr double kGeluInner = 0.7978845608028654;  // sqrt(2 / pi)
constexpr double kGeluCubic = 0.044715;
constexpr double kLog2e = 1.4426950408889634;

// The activation and its derivative.  Both are x * s for a logistic s:
// SiLU's is of x, and GELU's tanh form of v = 2 sqrt(2/pi) (x + 0.044715 x^3),
// as (1 + tanh(v / 2)) / 2 is the logistic function of v; written so, neither
// tail cancels.  exp(-v) overflows to inf for large negative v and s is then 0, as
// it is wherever it would lie below 2^-126: under v = -87.
// An error of v * log2(e) is one of exp(-v) times |v|.  SiLU's has one rounding,
// within |v| 2^-24 of s, and stays in 32 bits.  GELU's v goes through four, and is
// formed in 64 bits, which run at the 32-bit rate here.
template <int ACT>
__device__ __forceinline__ void act(float x, float& a, float& d) {
    float w = x * static_cast<float>(kLog2e), dv = 1.0f;
    if constexpr (ACT == MGOPT_ACT_GELU_TANH) {
        const double y = x, c = 2.0 * kGeluInner * kLog2e;
        w = static_cast<float>(y * fma(y * y, c * kGeluCubic, c));
        dv = static_cast<float>(2.0 * kGeluInner) * fmaf(static_cast<float>(3.0 * kGeluCubic), x * x, 1.0f);
    }
    const float s = rcp_hw(1.0f + exp2_hw(-w));
    a = x * s;
    // s (1 - s) v' x is 0 where x^2 overflowed: s is 0 or 1 there
    const float t = s * (1.0f - s);
    d = t == 0.0f ? s : fmaf(x * t, dv, s);
}

// Rows of vectors: work-group b takes the vectors of column chunk b % chunks
// of `rows_per_block` rows, 1 << shift threads a row.
struct Place {
    int64_t row, col;
};
template <int N>
__device__ __forceinline__ Place place(int64_t first_row, uint32_t chunks, uint32_t shift) {
    const uint32_t rb = blockIdx.x / chunks, cb = blockIdx.x - rb * chunks, t = threadIdx.x;
    return {first_row + static_cast<int64_t>(rb) * (kActBlock >> shift) + (t >> shift),
            (static_cast<int64_t>(cb) * kActBlock + (t & ((1u << shift) - 1))) * N};
}

struct ActArgs {
    const void *gate, *up;         // forward: inputs; backward: gate is grad_out
    int64_t gate_stride, up_stride;
    int64_t rows, width, groups;   // groups of a row
    int8_t* codes;                 // [inputs][rows][groups * 128]
    float* scales;                 // [inputs][rows][groups]
    void *y, *d_gate, *d_up;
    int64_t d_gate_stride, d_up_stride;
    int64_t first_row;             // of this launch
    uint32_t chunks, shift;
};

// N values of a group to codes, the group spread over 128 / N lanes.
template <int N>
__device__ __forceinline__ void pack(const float (&x)[N], int8_t* codes, float* scale, bool first) {
    uint32_t m = 0;  // magnitudes as integers: in their order, NaN above inf
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    m = reduce_lanes<kGroup / N>(m, [](uint32_t a, uint32_t b) { return max(a, b); });
    const float most = __uint_as_float(m);
    const bool finite = m < 0x7F800000u, zero = most < kTiny;
    const float inv = finite && !zero ? 127.0f / most : 0.0f;
    if (first) *scale = finite ? (zero ? 0.0f : most * (1.0f / 127.0f)) : __uint_as_float(0x7FC00000u);
    uint32_t word[N / 4];
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float c = finite ? rintf(x[i + k] * inv) : 0.0f;
            w |= (static_cast<uint32_t>(static_cast<int>(c)) & 0xFFu) << (8 * k);
        }
        word[i / 4] = w;
    }
    if constexpr (N == 8)
        *reinterpret_cast<uint2*>(codes) = make_uint2(word[0], word[1]);
    else
        *reinterpret_cast<uint32_t*>(codes) = word[0];
}

template <int N>
__device__ __forceinline__ void unpack(float (&x)[N], const int8_t* codes, float scale) {
    uint32_t word[N / 4];
    if constexpr (N == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes);
        word[0] = w.x, word[1] = w.y;
    } else {
        word[0] = *reinterpret_cast<const uint32_t*>(codes);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        x[i] = static_cast<float>(static_cast<int8_t>(word[i / 4] >> (8 * (i % 4)) & 0xFFu)) * scale;
}

template <typename T, int ACT, bool GATED, bool PACK, bool STREAM>
__global__ __launch_bounds__(kActBlock) void gated_act_kernel(ActArgs a) {
    constexpr int N = 16 / sizeof(T);
    const Place p = place<N>(a.first_row, a.chunks, a.shift);
    if (p.row >= a.rows || p.col >= a.groups * kGroup) return;  // whole groups of lanes leave together
    const int64_t n = a.width - p.col;
    float g[N], u[N], y[N];
    load_some<N, STREAM>(g, static_cast<const T*>(a.gate) + p.row * a.gate_stride + p.col, n);
    if constexpr (GATED) load_some<N, STREAM>(u, static_cast<const T*>(a.up) + p.row * a.up_stride + p.col, n);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float d;
        act<ACT>(g[i], y[i], d);
        if constexpr (GATED) y[i] *= u[i];
    }
    store_some<N, STREAM>(static_cast<T*>(a.y) + p.row * a.width + p.col, y, n);
    if constexpr (PACK) {
        const int64_t pitch = a.groups * kGroup, at = p.row * pitch + p.col;
        const int64_t group = p.row * a.groups + p.col / kGroup;
        const bool first = p.col % kGroup == 0;
        pack<N>(g, a.codes + at, a.scales + group, first);
        if constexpr (GATED) pack<N>(u, a.codes + a.rows * pitch + at, a.scales + a.rows * a.groups + group, first);
    }
}

template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(kActBlock) void gated_act_backward_kernel(ActArgs a) {
    constexpr int N = 16 / sizeof(T);
    const Place p = place<N>(a.first_row, a.chunks, a.shift);
    const int64_t n = a.width - p.col;
    if (p.row >= a.rows || n <= 0) return;
    const int64_t pitch = a.groups * kGroup, at = p.row * pitch + p.col;
    const int64_t group = p.row * a.groups + p.col / kGroup;
    float dy[N], g[N], u[N];
    load_some<N>(dy, static_cast<const T*>(a.gate) + p.row * a.gate_stride + p.col, n);
    unpack<N>(g, a.codes + at, a.scales[group]);
    if constexpr (GATED) unpack<N>(u, a.codes + a.rows * pitch + at, a.scales[a.rows * a.groups + group]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float v, d;
        act<ACT>(g[i], v, d);
        const float w = dy[i];
        if constexpr (GATED) {
            g[i] = w * u[i] * d;
            dy[i] = w * v;       // d_up
            u[i] = v * u[i];     // y
        } else {
            g[i] = w * d;
            u[i] = v;
        }
    }
    store_some<N>(static_cast<T*>(a.d_gate) + p.row * a.d_gate_stride + p.col, g, n);
    if constexpr (GATED) store_some<N>(static_cast<T*>(a.d_up) + p.row * a.d_up_stride + p.col, dy, n);
    if (a.y != nullptr) store_some<N>(static_cast<T*>(a.y) + p.row * a.width + p.col, u, n);
}

// The launches that cover the rows: threads per row as a power of two up to a
// work-group, in pieces of at most a grid.
template <typename F>
int over_rows(ActArgs a, int vec, F&& launch) {
    const int64_t vecs = a.groups * (kGroup / vec);
    a.shift = 0;
    while ((1 << a.shift) < kActBlock && (int64_t{1} << a.shift) < vecs) ++a.shift;
    const int64_t chunks = (vecs + kActBlock - 1) / kActBlock, per_block = kActBlock >> a.shift;
    if (chunks > max_blocks(kActBlock)) return set_error(MGOPT_E_LIMIT, "gated_act: rows too long");
    a.chunks = static_cast<uint32_t>(chunks);
    const int64_t piece = max_blocks(kActBlock) / chunks * per_block;
    for (a.first_row = 0; a.first_row < a.rows; a.first_row += piece) {
        const int64_t n = a.rows - a.first_row < piece ? a.rows - a.first_row : piece;
        launch(a, dim3(static_cast<uint32_t>((n + per_block - 1) / per_block * chunks)));
        if (int rc = launched("gated_act")) return rc;
    }
    return 0;
}

int check(const char* what, int32_t dtype, int64_t rows, int64_t width, int32_t kind) {
    if (!known_dtype(dtype)) return set_error(MGOPT_E_INVALID, std::string(what) + ": bad dtype");
    if (rows < 0 || width < 1) return set_error(MGOPT_E_INVALID, std::string(what) + ": need rows >= 0 and width >= 1");
    if (kind != MGOPT_ACT_SILU && kind != MGOPT_ACT_GELU_TANH)
        return set_error(MGOPT_E_INVALID, std::string(what) + ": unknown activation");
    return 0;
}

template <int V>
struct Int {
    static constexpr int value = V;
};
template <typename F>
void with_act(int32_t kind, F&& f) {
    if (kind == MGOPT_ACT_SILU) f(Int<MGOPT_ACT_SILU>{});
    else f(Int<MGOPT_ACT_GELU_TANH>{});
}

template <typename F>
void with_flag(bool on, F&& f) {
    if (on) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int mgopt_gated_act(const void* gate_dev, int64_t gate_stride, const void* up_dev, int64_t up_stride,
                              int32_t dtype, int64_t rows, int64_t width, int32_t kind, void* y_dev, int8_t* codes_dev,
                              float* scales_dev, void* stream) {
    if (int rc = check("gated_act", dtype, rows, width, kind)) return rc;
    if (rows == 0) return 0;
    if (!gate_dev || !y_dev || (codes_dev == nullptr) != (scales_dev == nullptr))
        return set_error(MGOPT_E_INVALID, "gated_act: NULL argument");
    if (reinterpret_cast<uintptr_t>(codes_dev) % 8 != 0)
        return set_error(MGOPT_E_ALIGN, "gated_act: codes must be 8-byte aligned");
    ActArgs a{};
    a.gate = gate_dev, a.up = up_dev, a.gate_stride = gate_stride, a.up_stride = up_stride;
    a.rows = rows, a.width = width, a.groups = (width + kGroup - 1) / kGroup;
    a.codes = codes_dev, a.scales = scales_dev, a.y = y_dev;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t inputs = up_dev ? 2 : 1;
    const bool stream_it = rows * width * (dtype_bytes(dtype) * (inputs + 1) + (codes_dev ? inputs : 0)) > kStreamBytes;
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return over_rows(a, 16 / sizeof(T), [&](const ActArgs& b, dim3 grid) {
            with_act(kind, [&](auto k) {
                constexpr int K = decltype(k)::value;
                const dim3 block(kActBlock);
                with_flag(up_dev != nullptr, [&](auto gated) {
                    with_flag(codes_dev != nullptr, [&](auto pack) {
                        with_flag(stream_it, [&](auto streamed) {
                            hipLaunchKernelGGL((gated_act_kernel<T, K, decltype(gated)::value, decltype(pack)::value, decltype(streamed)::value>),
                                               grid, block, 0, s, b);
                        });
                    });
                });
            });
        });
    });
}

MGOPT_API int mgopt_gated_act_backward(const void* grad_out_dev, int64_t grad_out_stride, const int8_t* codes_dev,
                                       const float* scales_dev, int32_t gated, int32_t dtype, int64_t rows, int64_t width,
                                       int32_t kind, void* d_gate_dev, int64_t d_gate_stride, void* d_up_dev,
                                       int64_t d_up_stride, void* y_dev, void* stream) {
    if (int rc = check("gated_act_backward", dtype, rows, width, kind)) return rc;
    if (rows == 0) return 0;
    if (!grad_out_dev || !codes_dev || !scales_dev || !d_gate_dev || (gated != 0) != (d_up_dev != nullptr))
        return set_error(MGOPT_E_INVALID, "gated_act_backward: NULL argument");
    if (reinterpret_cast<uintptr_t>(codes_dev) % 8 != 0)
        return set_error(MGOPT_E_ALIGN, "gated_act_backward: codes must be 8-byte aligned");
    ActArgs a{};
    a.gate = grad_out_dev, a.gate_stride = grad_out_stride;
    a.rows = rows, a.width = width, a.groups = (width + kGroup - 1) / kGroup;
    a.codes = const_cast<int8_t*>(codes_dev), a.scales = const_cast<float*>(scales_dev);
    a.d_gate = d_gate_dev, a.d_gate_stride = d_gate_stride, a.d_up = d_up_dev, a.d_up_stride = d_up_stride, a.y = y_dev;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return over_rows(a, 16 / sizeof(T), [&](const ActArgs& b, dim3 grid) {
            with_act(kind, [&](auto k) {
                constexpr int K = decltype(k)::value;
                const dim3 block(kActBlock);
                if (gated) hipLaunchKernelGGL((gated_act_backward_kernel<T, K, true>), grid, block, 0, s, b);
                else hipLaunchKernelGGL((gated_act_backward_kernel<T, K, false>), grid, block, 0, s, b);
            });
        });
    });
}

}  // extern "C"
