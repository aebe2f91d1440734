// ops_qk_norm_rope.hip -- RMS norm of every query and key head and the rotary
// rotation of the result, in one pass, and the backward pass.
//
// For one head's vector x of D elements, weight w and a token at position p:
//
//     xhat = x / sqrt(mean(x^2) + eps)      n = xhat * w
//     (a, b) -> (a cos - b sin, b cos + a sin)  for the R/2 pairs of n's first R
//                                              elements, cos and sin of p's table row
//
// the pairs being (i, i + R/2), or (2i, 2i + 1) when interleaved.  Backward,
// with g the incoming gradient rotated back and h = g * w:
//
//     dx = (h - xhat * mean(h * xhat)) / sqrt(mean(x^2) + eps)      dw = sum g * xhat
//
// A group of lanes holds a head, each lane VEC pairs of it, so that both halves
// of a pair are in one lane and the mean is a sum over the group.  `parts` groups
// share a token's heads: its cosines, sines and the weights stay in registers
// from head to head.
//
// Bound by memory: forward reads and writes the heads once; backward reads x
// and the gradient and writes dx.  The weights' gradients are summed per lane
// over all of a work-group's tokens, then over lanes and work-groups in a fixed
// order.  8,192 tokens of 32 + 8 heads of 128 in bf16: 36 us forward (4.7 TB/s),
// 48 us backward (5.3 TB/s) and 5 us for the weights' sums, a launch's latency.
#include "ops_common.h"

namespace mgopt {
namespace {

constexpr int kRopeBlock = 256;
constexpr int kWaves = kRopeBlock / 64;
constexpr int kMaxDim = MGOPT_MAX_HEAD_DIM;
constexpr uint32_t kBackwardBlocks = 2048;  // work-groups of the backward pass at most, a row of partial weight gradients each

constexpr uint64_t kMaxTasks = uint64_t{1} << 31;  // tokens times the groups that share a token

struct Args {
    mgopt_qk_args a;
    uint32_t tokens;
    uint32_t lanes;   // of a head: 1 << shift
    uint32_t shift;
    uint32_t parts;   // groups that share a token's heads
    // backward
    uint32_t q_parts, k_parts, q_blocks;
    float* partials;  // [work-groups][dim]
};

// x summed over aligned groups of `lanes` lanes, in each of them.
__device__ __forceinline__ float sum_group(float x, uint32_t lanes) {
    if (lanes > 1) x += dpp<kDppXor1>(x);
    if (lanes > 2) x += dpp<kDppXor2>(x);
    if (lanes > 4) x += dpp<kDppHalfMirror>(x);
    if (lanes > 8) x += dpp<kDppMirror>(x);
    if (lanes > 16) x += __shfl_xor(x, 16);
    if (lanes > 32) x += __shfl_xor(x, 32);
    return x;
}

// Where a lane's VEC pairs lie: VEC elements from a and VEC from b.  Slots past
// the rotated part hold neighbouring elements that are passed through.
struct Slot {
    int a, b;
    bool rotated, on, has_b;
};
template <int VEC, bool INTER>
__device__ __forceinline__ Slot slot_of(uint32_t s, int dim, int rotary) {
    Slot q;
    q.rotated = static_cast<int>(s) * 2 * VEC < rotary;
    if (INTER || !q.rotated) {
        q.a = static_cast<int>(s) * 2 * VEC;
        q.b = q.a + VEC;
    } else {
        q.a = static_cast<int>(s) * VEC;
        q.b = q.a + rotary / 2;
    }
    q.on = static_cast<int>(s) * 2 * VEC < dim;
    q.has_b = q.on && q.b < dim;  // only single elements (VEC 1) can end a head in the middle of a slot
    return q;
}

// The pairs of a slot: a[j], b[j].
template <int VEC, bool INTER>
struct Pairs {
    float a[VEC], b[VEC];

    template <typename T>
    __device__ __forceinline__ void read(const T* p, const Slot& q) {
        float lo[VEC], hi[VEC];
        load<VEC>(lo, p + q.a);
        if (VEC > 1 || q.has_b) load<VEC>(hi, p + q.b);
        else hi[0] = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            a[j] = INTER ? (2 * j < VEC ? lo[2 * j % VEC] : hi[2 * j % VEC]) : lo[j];
            b[j] = INTER ? (2 * j + 1 < VEC ? lo[(2 * j + 1) % VEC] : hi[(2 * j + 1) % VEC]) : hi[j];
        }
        if constexpr (INTER && VEC == 1) b[0] = hi[0];
    }
    template <typename T>
    __device__ __forceinline__ void write(T* p, const Slot& q) const {
        float lo[VEC], hi[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            lo[j] = INTER && VEC > 1 ? (j % 2 ? b[j / 2] : a[j / 2]) : a[j];
            hi[j] = INTER && VEC > 1 ? (j % 2 ? b[(j + VEC) / 2] : a[(j + VEC) / 2]) : b[j];
        }
        store<VEC>(p + q.a, lo);
        if (VEC > 1 || q.has_b) store<VEC>(p + q.b, hi);
    }
    __device__ __forceinline__ void read_weights(const void* p, int32_t dtype, const Slot& q) {
        if (dtype == MGOPT_F32) read(static_cast<const float*>(p), q);
        else if (dtype == MGOPT_F16) read(static_cast<const _Float16*>(p), q);
        else read(static_cast<const __bf16*>(p), q);
    }
};

// cos and sin of a slot's pairs at a token's position: 1 and 0 past the rotated part, NaN outside the table.
template <int VEC>
__device__ __forceinline__ void angles(const Args& k, const Slot& q, uint32_t s, int64_t pos, float (&c)[VEC], float (&d)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) c[j] = 1.0f, d[j] = 0.0f;
    if (!q.rotated) return;
    if (pos < 0 || pos >= k.a.table_rows) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = d[j] = __builtin_nanf("");
        return;
    }
    const int64_t at = pos * (k.a.rotary / 2) + static_cast<int64_t>(s) * VEC;
    load<VEC>(c, k.a.cos_dev + at);
    load<VEC>(d, k.a.sin_dev + at);
}

struct Token {
    int64_t batch, at, pos;
};
__device__ __forceinline__ Token token_of(const Args& k, uint32_t n) {
    const uint32_t length = static_cast<uint32_t>(k.a.length), b = n / length, t = n - b * length;
    const int64_t pos = k.a.positions_dev == nullptr
                            ? t
                            : id_at(k.a.positions_dev, b * k.a.position_stride + t, k.a.position_bytes);
    return {b, t, pos};
}

__device__ __forceinline__ int64_t offset(const int64_t (&stride)[3], const Token& t, uint32_t head) {
    return t.batch * stride[0] + t.at * stride[1] + static_cast<int64_t>(head) * stride[2];
}

template <typename T, int VEC, int SLOTS, bool INTER>
__global__ __launch_bounds__(kRopeBlock) void qk_norm_rope_kernel(Args k) {
    const uint32_t group = blockIdx.x * (kRopeBlock >> k.shift) + (threadIdx.x >> k.shift);
    const uint32_t n = group / k.parts, part = group - n * k.parts;
    if (n >= k.tokens) return;  // whole groups of lanes
    const Token t = token_of(k, n);
    const uint32_t l = threadIdx.x & (k.lanes - 1);
    const float inv_dim = 1.0f / static_cast<float>(k.a.dim);
    Slot q[SLOTS];
    float c[SLOTS][VEC], d[SLOTS][VEC];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const uint32_t s = l + i * k.lanes;
        q[i] = slot_of<VEC, INTER>(s, k.a.dim, k.a.rotary);
        angles<VEC>(k, q[i], s, t.pos, c[i], d[i]);
    }
    auto heads = [&](const mgopt_heads& side, uint32_t h) {
        Pairs<VEC, INTER> w[SLOTS];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
            if (q[i].on) w[i].read_weights(side.weight_dev, k.a.weight_dtype, q[i]);
        for (; h < static_cast<uint32_t>(side.heads); h += k.parts) {
            const T* x = static_cast<const T*>(side.x_dev) + offset(side.x_stride, t, h);
            T* out = static_cast<T*>(side.out_dev) + offset(side.out_stride, t, h);
            Pairs<VEC, INTER> v[SLOTS];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (!q[i].on) continue;
                v[i].read(x, q[i]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum = fmaf(v[i].a[j], v[i].a[j], fmaf(v[i].b[j], v[i].b[j], sum));
            }
            const float r = 1.0f / sqrtf(fmaf(sum_group(sum, k.lanes), inv_dim, k.a.eps));
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (!q[i].on) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float a = v[i].a[j] * r * w[i].a[j], b = v[i].b[j] * r * w[i].b[j];
                    v[i].a[j] = fmaf(a, c[i][j], -b * d[i][j]);
                    v[i].b[j] = fmaf(b, c[i][j], a * d[i][j]);
                }
                v[i].write(out, q[i]);
            }
        }
        return h - static_cast<uint32_t>(side.heads);
    };
    // the groups count through the queries' heads and on through the keys'
    const uint32_t first_k = heads(k.a.q, part);
    heads(k.a.k, first_k);
}

// The first q_blocks work-groups take the queries' heads, the others the keys':
// one side's weights and sums are all that a lane holds, which leaves registers
// for four waves a SIMD (8,192 tokens of 32 + 8 heads of 128 in bf16: 50 us, with
// both sides' in one wave, 185 registers, 62).
template <typename T, int VEC, int SLOTS, bool INTER>
__global__ __launch_bounds__(kRopeBlock, 4) void qk_norm_rope_backward_kernel(Args k) {
    const bool on_q = blockIdx.x < k.q_blocks;
    const mgopt_heads& side = on_q ? k.a.q : k.a.k;
    const uint32_t block = on_q ? blockIdx.x : blockIdx.x - k.q_blocks, blocks = on_q ? k.q_blocks : gridDim.x - k.q_blocks;
    const uint32_t heads = static_cast<uint32_t>(side.heads);
    const uint32_t lane = threadIdx.x % 64, l = lane & (k.lanes - 1), groups = kRopeBlock >> k.shift;
    const uint32_t parts = on_q ? k.q_parts : k.k_parts;
    const float inv_dim = 1.0f / static_cast<float>(k.a.dim);
    Slot q[SLOTS];
    Pairs<VEC, INTER> w[SLOTS], sum_w[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        q[i] = slot_of<VEC, INTER>(l + i * k.lanes, k.a.dim, k.a.rotary);
        if (q[i].on) w[i].read_weights(side.weight_dev, k.a.weight_dtype, q[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum_w[i].a[j] = sum_w[i].b[j] = 0.0f;
    }
    const uint32_t tasks = k.tokens * parts;
    for (uint32_t task = block * groups + (threadIdx.x >> k.shift); task < tasks; task += blocks * groups) {
        const uint32_t n = task / parts, part = task - n * parts;
        const Token t = token_of(k, n);
        float c[SLOTS][VEC], d[SLOTS][VEC];
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) angles<VEC>(k, q[i], l + i * k.lanes, t.pos, c[i], d[i]);
        for (uint32_t h = part; h < heads; h += parts) {
            const T* x = static_cast<const T*>(side.x_dev) + offset(side.x_stride, t, h);
            const T* grad = static_cast<const T*>(side.grad_dev) + offset(side.grad_stride, t, h);
            T* dx = static_cast<T*>(side.d_x_dev) + offset(side.d_x_stride, t, h);
            Pairs<VEC, INTER> v[SLOTS], g[SLOTS];
            float sum = 0.0f, dot = 0.0f;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (!q[i].on) continue;
                v[i].read(x, q[i]);
                g[i].read(grad, q[i]);
            }
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (!q[i].on) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float a = g[i].a[j], b = g[i].b[j];
                    g[i].a[j] = fmaf(a, c[i][j], b * d[i][j]);
                    g[i].b[j] = fmaf(b, c[i][j], -a * d[i][j]);
                    sum = fmaf(v[i].a[j], v[i].a[j], fmaf(v[i].b[j], v[i].b[j], sum));
                    dot = fmaf(g[i].a[j] * w[i].a[j], v[i].a[j], fmaf(g[i].b[j] * w[i].b[j], v[i].b[j], dot));
                }
            }
            const float r = 1.0f / sqrtf(fmaf(sum_group(sum, k.lanes), inv_dim, k.a.eps));
            const float m = sum_group(dot, k.lanes) * r * inv_dim;  // mean(h * xhat)
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                if (!q[i].on) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xa = v[i].a[j] * r, xb = v[i].b[j] * r;
                    sum_w[i].a[j] = fmaf(g[i].a[j], xa, sum_w[i].a[j]);
                    sum_w[i].b[j] = fmaf(g[i].b[j], xb, sum_w[i].b[j]);
                    v[i].a[j] = r * fmaf(-xa, m, g[i].a[j] * w[i].a[j]);
                    v[i].b[j] = r * fmaf(-xb, m, g[i].b[j] * w[i].b[j]);
                }
                v[i].write(dx, q[i]);
            }
        }
    }
    // over the groups of a wave, then over the work-group's waves
    __shared__ float part[kWaves][kMaxDim];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            for (uint32_t off = k.lanes; off < 64; off <<= 1) {
                sum_w[i].a[j] += __shfl_xor(sum_w[i].a[j], off);
                sum_w[i].b[j] += __shfl_xor(sum_w[i].b[j], off);
            }
        if (lane < k.lanes && q[i].on) sum_w[i].write(&part[threadIdx.x / 64][0], q[i]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < k.a.dim; e += kRopeBlock) {
        float x = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) x += part[v][e];
        k.partials[static_cast<int64_t>(blockIdx.x) * k.a.dim + e] = x;
    }
}

// Sums the rows of partial weight gradients, the first q_rows of them the
// queries': work-group (c, s) takes kCols columns of side s, its threads rows in
// turn, joined in a fixed order.
constexpr int kCols = 16, kSumBlock = 1024;
__global__ __launch_bounds__(kSumBlock) void weight_grad_kernel(const float* partials, uint32_t q_rows, uint32_t k_rows,
                                                                int32_t dim, void* dq, void* dk, int32_t dtype) {
    __shared__ float part[kSumBlock / kCols][kCols + 1];
    const int col = threadIdx.x % kCols, row = threadIdx.x / kCols, e = blockIdx.x * kCols + col;
    const uint32_t rows = blockIdx.y == 0 ? q_rows : k_rows;
    const float* at = partials + (blockIdx.y == 0 ? 0 : static_cast<int64_t>(q_rows) * dim) + e;
    float x = 0.0f;
    if (e < dim) {
#pragma unroll 8
        for (uint32_t r = row; r < rows; r += kSumBlock / kCols) x += at[static_cast<int64_t>(r) * dim];
    }
    part[row][col] = x;
    __syncthreads();
    for (int half = kSumBlock / kCols / 2; half > 0; half /= 2) {
        if (row < half) part[row][col] += part[row + half][col];
        __syncthreads();
    }
    if (row != 0 || e >= dim) return;
    x = part[0][col];
    void* out = blockIdx.y == 0 ? dq : dk;
    if (dtype == MGOPT_F32) static_cast<float*>(out)[e] = x;
    else if (dtype == MGOPT_F16) static_cast<_Float16*>(out)[e] = static_cast<_Float16>(x);
    else static_cast<__bf16*>(out)[e] = static_cast<__bf16>(x);
}

int check(const mgopt_qk_args* a, const char* what) {
    const std::string w(what);
    if (!a) return set_error(MGOPT_E_INVALID, w + ": NULL arguments");
    if (!known_dtype(a->dtype) || !known_dtype(a->weight_dtype)) return set_error(MGOPT_E_INVALID, w + ": bad dtype");
    if (a->batch < 0 || a->length < 0 || a->q.heads < 1 || a->k.heads < 1)
        return set_error(MGOPT_E_INVALID, w + ": negative sizes, or no heads");
    if (a->dim < 1 || a->rotary < 0 || a->rotary > a->dim || a->rotary % 2 != 0)
        return set_error(MGOPT_E_INVALID, w + ": rotary must be even and at most dim");
    if (a->dim > kMaxDim) return set_error(MGOPT_E_LIMIT, w + ": heads of more than " + std::to_string(kMaxDim) + " elements");
    if (a->batch > 0 && a->length > (int64_t{1} << 28) / a->batch)
        return set_error(MGOPT_E_LIMIT, w + ": more than 2^28 tokens");
    if (a->q.heads > (1 << 20) || a->k.heads > (1 << 20)) return set_error(MGOPT_E_LIMIT, w + ": more than 2^20 heads");
    if (a->positions_dev && a->position_bytes != 4 && a->position_bytes != 8)
        return set_error(MGOPT_E_INVALID, w + ": positions have 4 or 8 bytes");
    if (!(a->eps >= 0.0f)) return set_error(MGOPT_E_INVALID, w + ": eps must not be negative");
    if (a->rotary > 0 && (!a->cos_dev || !a->sin_dev || a->table_rows < 0))
        return set_error(MGOPT_E_INVALID, w + ": no table of cosines and sines");
    if (!a->q.weight_dev || !a->k.weight_dev) return set_error(MGOPT_E_INVALID, w + ": NULL weight");
    return 0;
}

// The kernel's form for these sizes: 16 bytes (VEC elements) of each half of the pairs per lane where
// the head and its rotated part are made of such; else 4 elements; else single ones.  Interleaved pairs
// of 8 elements do not fit the backward pass's registers at four waves a SIMD (40 of them spill), 4 do.
template <bool BACKWARD, typename F>
int with_form(const mgopt_qk_args& a, Args& k, F&& f) {
    auto shape = [&](int vec, int slots) {
        const int pieces = (a.dim + 2 * vec - 1) / (2 * vec);
        k.shift = 0;
        while ((1 << k.shift) * slots < pieces) ++k.shift;
        k.lanes = 1u << k.shift;
        // groups that share a token's heads: four heads each, for the use of one token's cosines, or fewer while
        // that leaves the chip short of waves
        const int64_t groups = 64 / k.lanes;
        const auto share = [&](int64_t heads) {
            int64_t parts = (heads + 3) / 4;
            while (parts < heads && k.tokens * parts < 4096 * groups) ++parts;
            return static_cast<uint32_t>(parts);
        };
        k.parts = share(a.q.heads + a.k.heads);
        k.q_parts = share(a.q.heads), k.k_parts = share(a.k.heads);
    };
    return with_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        auto inter = [&](auto vec, auto slots) {
            constexpr int VEC = decltype(vec)::value, SLOTS = decltype(slots)::value;
            shape(VEC, SLOTS);
            if constexpr (!BACKWARD || VEC < 8)
                if (a.interleaved) return f(T{}, vec, slots, std::true_type{});
            return f(T{}, vec, slots, std::false_type{});
        };
        auto both = [&](int n) { return a.dim % (2 * n) == 0 && a.rotary % (2 * n) == 0; };
        using One = std::integral_constant<int, 1>;
        if constexpr (sizeof(T) == 2)
            if (both(8) && !(BACKWARD && a.interleaved)) return inter(std::integral_constant<int, 8>{}, One{});
        if (both(4)) return inter(std::integral_constant<int, 4>{}, One{});
        if (a.dim <= 128) return inter(One{}, One{});
        return inter(One{}, std::integral_constant<int, 4>{});
    });
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int mgopt_qk_norm_rope(const mgopt_qk_args* a, void* stream) {
    if (int rc = check(a, "qk_norm_rope")) return rc;
    if (a->batch == 0 || a->length == 0) return 0;
    for (const mgopt_heads* h : {&a->q, &a->k})
        if (!h->x_dev || !h->out_dev) return set_error(MGOPT_E_INVALID, "qk_norm_rope: NULL argument");
    Args k{};
    k.a = *a;
    k.tokens = static_cast<uint32_t>(a->batch * a->length);
    return with_form<false>(*a, k, [&](auto t, auto vec, auto slots, auto inter) {
        using T = decltype(t);
        const uint64_t groups = kRopeBlock / k.lanes, tasks = static_cast<uint64_t>(k.tokens) * k.parts;
        const uint64_t blocks = (tasks + groups - 1) / groups;
        if (tasks > kMaxTasks || blocks > max_blocks(kRopeBlock))
            return set_error(MGOPT_E_LIMIT, "qk_norm_rope: too many heads");
        hipLaunchKernelGGL((qk_norm_rope_kernel<T, decltype(vec)::value, decltype(slots)::value, decltype(inter)::value>),
                           dim3(static_cast<uint32_t>(blocks)), dim3(kRopeBlock), 0, static_cast<hipStream_t>(stream), k);
        return launched("qk_norm_rope_kernel");
    });
}

MGOPT_API int64_t mgopt_qk_norm_rope_workspace(int32_t dim) {
    return dim < 1 ? -1 : int64_t{kBackwardBlocks} * dim * static_cast<int64_t>(sizeof(float));
}

MGOPT_API int mgopt_qk_norm_rope_backward(const mgopt_qk_args* a, void* stream) {
    if (int rc = check(a, "qk_norm_rope_backward")) return rc;
    for (const mgopt_heads* h : {&a->q, &a->k}) {
        if (!h->d_weight_dev) return set_error(MGOPT_E_INVALID, "qk_norm_rope_backward: NULL argument");
        if (a->batch * a->length > 0 && (!h->x_dev || !h->grad_dev || !h->d_x_dev))
            return set_error(MGOPT_E_INVALID, "qk_norm_rope_backward: NULL argument");
    }
    if (!a->workspace_dev || reinterpret_cast<uintptr_t>(a->workspace_dev) % 4 != 0)
        return set_error(MGOPT_E_ALIGN, "qk_norm_rope_backward: the workspace must be 4-byte aligned");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Args k{};
    k.a = *a;
    k.tokens = static_cast<uint32_t>(a->batch * a->length);
    k.partials = static_cast<float*>(a->workspace_dev);
    uint32_t k_blocks = 0;
    if (k.tokens > 0) {
        const int rc = with_form<true>(*a, k, [&](auto t, auto vec, auto slots, auto inter) {
            using T = decltype(t);
            if (static_cast<uint64_t>(k.tokens) * std::max(k.q_parts, k.k_parts) > kMaxTasks)
                return set_error(MGOPT_E_LIMIT, "qk_norm_rope_backward: too many heads");
            // work-groups by the sides' shares of the heads, each no more than it has work for
            const auto blocks_for = [&](uint32_t parts, uint32_t share) {
                const uint64_t groups = kRopeBlock / k.lanes, tasks = static_cast<uint64_t>(k.tokens) * parts;
                return static_cast<uint32_t>(std::min<uint64_t>((tasks + groups - 1) / groups, share));
            };
            const uint32_t k_share = std::max<uint32_t>(
                1, static_cast<uint32_t>(static_cast<uint64_t>(kBackwardBlocks) * a->k.heads / (a->q.heads + a->k.heads)));
            k.q_blocks = blocks_for(k.q_parts, kBackwardBlocks - k_share);
            k_blocks = blocks_for(k.k_parts, k_share);
            hipLaunchKernelGGL((qk_norm_rope_backward_kernel<T, decltype(vec)::value, decltype(slots)::value, decltype(inter)::value>),
                               dim3(k.q_blocks + k_blocks), dim3(kRopeBlock), 0, s, k);
            return launched("qk_norm_rope_backward_kernel");
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(weight_grad_kernel, dim3((a->dim + kCols - 1) / kCols, 2), dim3(kSumBlock), 0, s, k.partials,
                       k.q_blocks, k_blocks, a->dim, a->q.d_weight_dev, a->k.d_weight_dev, a->weight_dtype);
    return launched("weight_grad_kernel");
}

}  // extern "C"
