// ops_embedding.hip -- token embedding: the lookup of scaled rows, and the
// weight's gradient.
//
//     out[t] = scale * W[id[t]]
//     dW[v] = (dW[v] if accumulating) + scale * sum of dY[t] over t with id[t] = v != padding
//
// An id outside [0, rows) gives a row of NaN and no gradient.  The sums run in
// 32 bits over the tokens in their order, split in ways the sizes alone fix, so
// the same inputs give the same bits.
//
// Bound by memory: the lookup writes a row per token and reads its rows; the
// gradient reads a row per token and writes V rows, or reads and writes the
// rows the tokens name when it accumulates.
#include "ops_common.h"

namespace mgopt {
namespace {

constexpr int kBlock = 256;

// ------------------------------------------------------------------ lookup

struct LookupArgs {
    const void *ids, *weight;
    void* out;
    int64_t n, rows, width, first;
    int32_t id_bytes;
    uint32_t shift;  // 1 << shift threads a token
    float scale;
};

template <typename TW, typename TO>
__global__ __launch_bounds__(kBlock) void lookup_kernel(LookupArgs a) {
    constexpr int N = 16 / (sizeof(TW) > sizeof(TO) ? sizeof(TW) : sizeof(TO));
    const int64_t t = a.first + static_cast<int64_t>(blockIdx.x) * (kBlock >> a.shift) + (threadIdx.x >> a.shift);
    if (t >= a.n) return;
    const int64_t id = id_at(a.ids, t, a.id_bytes);
    const bool known = id >= 0 && id < a.rows;
    const TW* w = static_cast<const TW*>(a.weight) + (known ? id : 0) * a.width;
    TO* out = static_cast<TO*>(a.out) + t * a.width;
    const int64_t step = int64_t{N} << a.shift;
    for (int64_t c = static_cast<int64_t>(threadIdx.x & ((1u << a.shift) - 1)) * N; c < a.width; c += step) {
        float v[N];
        if (known) {
            load_some<N>(v, w + c, a.width - c);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= a.scale;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __builtin_nanf("");
        }
        store_some<N>(out + c, v, a.width - c);
    }
}

// ---------------------------------------------------------------- gradient

struct GradArgs {
    const void *ids, *grad_out;
    void* grad;
    int64_t n, rows, width, first_row;
    int64_t padding;       // -1: none
    int32_t id_bytes, accumulate;
    uint32_t shift;        // 1 << shift threads a row of a column chunk
    uint32_t chunks;       // column chunks of kBlock vectors
    float scale;
};

// One work-group per weight row (and column chunk): it reads all ids, lists the
// tokens that name its row, in their order, and sums their rows.  Its threads
// split the list in 1 << (8 - shift) parts, joined in a fixed order.
constexpr int kScan = 4;  // ids per thread and round
template <typename TG, typename TW>
__global__ __launch_bounds__(kBlock) void grad_by_row_kernel(GradArgs a) {
    constexpr int N = 16 / (sizeof(TG) > sizeof(TW) ? sizeof(TG) : sizeof(TW));
    constexpr int kTile = kBlock * kScan, kWaves = kBlock / 64;
    __shared__ int64_t list[kTile];
    __shared__ uint32_t count[kScan][kWaves];
    __shared__ float joined[kBlock][N + 1];
    const uint32_t rb = blockIdx.x / a.chunks, cb = blockIdx.x - rb * a.chunks;
    const int64_t row = a.first_row + rb;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t parts = kBlock >> a.shift, part = threadIdx.x >> a.shift;
    const int64_t c = (static_cast<int64_t>(cb) * kBlock + (threadIdx.x & ((1u << a.shift) - 1))) * N, left = a.width - c;
    float sum[N] = {};
    bool any = false;
    if (row != a.padding) {
        for (int64_t t0 = 0; t0 < a.n; t0 += kTile) {
            bool mine[kScan];
            uint64_t votes[kScan];
#pragma unroll
            for (int k = 0; k < kScan; ++k) {
                const int64_t t = t0 + k * kBlock + threadIdx.x;
                mine[k] = t < a.n && id_at(a.ids, t, a.id_bytes) == row;
                votes[k] = __ballot(mine[k]);
                if (lane == 0) count[k][wave] = static_cast<uint32_t>(__popcll(votes[k]));
            }
            __syncthreads();
            uint32_t before = 0;
#pragma unroll
            for (int k = 0; k < kScan; ++k) {
                uint32_t at = before;
                for (uint32_t w = 0; w < kWaves; ++w) {
                    if (w < wave) at += count[k][w];
                    before += count[k][w];
                }
                if (mine[k]) list[at + __popcll(votes[k] & ((uint64_t{1} << lane) - 1))] = t0 + k * kBlock + threadIdx.x;
            }
            __syncthreads();
            any |= before > 0;
            if (left > 0) {
                for (uint32_t i = part; i < before; i += parts) {
                    float v[N];
                    load_some<N>(v, static_cast<const TG*>(a.grad_out) + list[i] * a.width + c, left);
#pragma unroll
                    for (int j = 0; j < N; ++j) sum[j] += v[j];
                }
            }
            __syncthreads();  // the list is written again
        }
    }
    if (!any && a.accumulate) return;
#pragma unroll
    for (int j = 0; j < N; ++j) joined[threadIdx.x][j] = sum[j];
    __syncthreads();
    if (part != 0 || left <= 0) return;
    for (uint32_t p = 1; p < parts; ++p)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += joined[threadIdx.x + (p << a.shift)][j];
    TW* out = static_cast<TW*>(a.grad) + row * a.width + c;
    float old[N] = {};
    if (a.accumulate) load_some<N>(old, out, left);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = fmaf(sum[j], a.scale, old[j]);
    store_some<N>(out, sum, left);
}

uint32_t shift_for(int64_t vecs) {
    uint32_t s = 0;
    while ((1 << s) < kBlock && (int64_t{1} << s) < vecs) ++s;
    return s;
}

int check(const char* what, int64_t n, int64_t rows, int64_t width, int32_t id_bytes, int32_t a, int32_t b, float scale) {
    const std::string w(what);
    if (!known_dtype(a) || !known_dtype(b)) return set_error(MGOPT_E_INVALID, w + ": bad dtype");
    if (n < 0 || rows < 1 || width < 1) return set_error(MGOPT_E_INVALID, w + ": need n >= 0, rows >= 1 and width >= 1");
    if (id_bytes != 4 && id_bytes != 8) return set_error(MGOPT_E_INVALID, w + ": ids have 4 or 8 bytes");
    if (!std::isfinite(scale)) return set_error(MGOPT_E_INVALID, w + ": the scale must be finite");
    return 0;
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int mgopt_embedding(const void* ids_dev, int32_t id_bytes, int64_t n, const void* weight_dev, int32_t weight_dtype,
                              int64_t rows, int64_t width, float scale, void* out_dev, int32_t out_dtype, void* stream) {
    if (int rc = check("embedding", n, rows, width, id_bytes, weight_dtype, out_dtype, scale)) return rc;
    if (n == 0) return 0;
    if (!ids_dev || !weight_dev || !out_dev) return set_error(MGOPT_E_INVALID, "embedding: NULL argument");
    LookupArgs a{ids_dev, weight_dev, out_dev, n, rows, width, 0, id_bytes, 0, scale};
    return with_dtype(weight_dtype, [&](auto w) {
        return with_dtype(out_dtype, [&](auto o) {
            using TW = decltype(w);
            using TO = decltype(o);
            constexpr int N = 16 / (sizeof(TW) > sizeof(TO) ? sizeof(TW) : sizeof(TO));
            a.shift = shift_for((width + N - 1) / N);
            const int64_t per_block = kBlock >> a.shift, most = max_blocks(kBlock) * per_block;
            for (a.first = 0; a.first < n; a.first += most) {
                const int64_t blocks = (std::min(n - a.first, most) + per_block - 1) / per_block;
                hipLaunchKernelGGL((lookup_kernel<TW, TO>), dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0,
                                   static_cast<hipStream_t>(stream), a);
                if (int rc = launched("lookup_kernel")) return rc;
            }
            return 0;
        });
    });
}

MGOPT_API int64_t mgopt_embedding_grad_workspace(int64_t n, int64_t rows, int64_t width) {
    return n < 0 || rows < 1 || width < 1 ? -1 : 16;
}

MGOPT_API int mgopt_embedding_grad(const void* ids_dev, int32_t id_bytes, int64_t n, const void* grad_out_dev,
                                   int32_t grad_out_dtype, void* grad_dev, int32_t grad_dtype, int64_t rows, int64_t width,
                                   float scale, int64_t padding_idx, int32_t accumulate, void* workspace_dev, void* stream) {
    if (int rc = check("embedding_grad", n, rows, width, id_bytes, grad_out_dtype, grad_dtype, scale)) return rc;
    if (padding_idx < -1 || padding_idx >= rows) return set_error(MGOPT_E_INVALID, "embedding_grad: bad padding index");
    if (!grad_dev || (n > 0 && (!ids_dev || !grad_out_dev))) return set_error(MGOPT_E_INVALID, "embedding_grad: NULL argument");
    if (!workspace_dev || reinterpret_cast<uintptr_t>(workspace_dev) % 16 != 0)
        return set_error(MGOPT_E_ALIGN, "embedding_grad: the workspace must be 16-byte aligned");
    if (n == 0 && accumulate) return 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    GradArgs a{ids_dev, grad_out_dev, grad_dev, n, rows, width, 0, padding_idx, id_bytes, accumulate, 0, 0, scale};
    return with_dtype(grad_out_dtype, [&](auto g) {
        return with_dtype(grad_dtype, [&](auto w) {
            using TG = decltype(g);
            using TW = decltype(w);
            constexpr int N = 16 / (sizeof(TG) > sizeof(TW) ? sizeof(TG) : sizeof(TW));
            const int64_t vecs = (width + N - 1) / N, chunks = (vecs + kBlock - 1) / kBlock;
            if (chunks > max_blocks(kBlock)) return set_error(MGOPT_E_LIMIT, "embedding_grad: rows too long");
            a.shift = shift_for(vecs);
            a.chunks = static_cast<uint32_t>(chunks);
            const int64_t most = max_blocks(kBlock) / chunks;
            for (a.first_row = 0; a.first_row < rows; a.first_row += most) {
                const int64_t blocks = std::min(rows - a.first_row, most) * chunks;
                hipLaunchKernelGGL((grad_by_row_kernel<TG, TW>), dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, a);
                if (int rc = launched("grad_by_row_kernel")) return rc;
            }
            return 0;
        });
    });
}

}  // extern "C"
