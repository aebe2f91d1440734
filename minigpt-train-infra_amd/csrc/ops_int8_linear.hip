// ops_int8_linear.hip -- products of 8-bit integers with a scale for each token
// and each output channel.
//
//     y[t][n] = (x_scales[t] * w_scales[n]) * sum_k x[t][k] * w[n][k]  (+ bias[n])
//
// The sum is exact in 32-bit integers (at most 131,071 products of magnitudes up to
// 2^14), so neither tiles nor parts of the contraction change a result; it is turned
// into a 32-bit float, scaled, added to the bias and rounded once.
//
// The matrix cores take the channels as rows and the tokens as columns, so that a
// lane holds four consecutive channels of one token in each group of registers.
#include "ops_common.h"

namespace mgopt {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct LinearArgs {
    const int8_t *x, *w;
    int64_t x_stride, w_stride;
    const float *x_scales, *w_scales;
    const void* bias;
    void* y;
    int64_t rows, width, channels;
    uint32_t row_tiles, channel_tiles;
    int32_t bias_dtype;
};

// 16 codes from p, those from n on 0.
__device__ __forceinline__ i32x4 load_codes(const int8_t* p, int64_t n) {
    typedef int unaligned __attribute__((ext_vector_type(4), aligned(1)));
    if (n >= 16) return *reinterpret_cast<const unaligned*>(p);
    i32x4 v{};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < n) v[i / 4] |= static_cast<int>((static_cast<uint32_t>(p[i]) & 0xFFu) << (8 * (i % 4)));
    return v;
}

__device__ __forceinline__ i32x16 mma(i32x4 a, i32x4 b, i32x16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float bias_at(const LinearArgs& a, int64_t n) {
    if (a.bias_dtype == MGOPT_F32) return static_cast<const float*>(a.bias)[n];
    if (a.bias_dtype == MGOPT_F16) return static_cast<float>(static_cast<const _Float16*>(a.bias)[n]);
    return static_cast<float>(static_cast<const __bf16*>(a.bias)[n]);
}

// Four channels from n on of token t.
template <typename T>
__device__ __forceinline__ void finish(const LinearArgs& a, int64_t t, int64_t n, const int (&sum)[4], float x_scale) {
    const int64_t left = a.channels - n;
    if (left <= 0) return;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t at = i < left ? n + i : n;
        y[i] = static_cast<float>(sum[i]) * (x_scale * a.w_scales[at]);
        if (a.bias != nullptr) y[i] += bias_at(a, at);
    }
    store_some<4>(static_cast<T*>(a.y) + t * a.channels + n, y, left);
}

// Tiles of WC * TC * 32 channels and WT * TT * 32 tokens, WC * WT waves with TC x TT blocks of 32 x 32 each.
// 128 codes of each row at a time lie in LDS, twice: the next ones are on their way while these are multiplied.
// Chunk c (16 codes) of row r lies at chunk c ^ (r / 2 % 8), so that a chunk of 16 rows falls on all banks.
template <typename T, int WC, int WT, int TC, int TT>
__global__ __launch_bounds__(WC* WT * 64, 2) void int8_linear_kernel(LinearArgs a) {
    constexpr int THREADS = WC * WT * 64, BC = WC * TC * 32, BT = WT * TT * 32, BK = 128, CHUNKS = BK / 16;
    constexpr int EACH = (BC + BT) * CHUNKS / THREADS;
    static_assert((BC + BT) * CHUNKS % THREADS == 0 && BC * CHUNKS % THREADS == 0);
    __shared__ i32x4 lds[2][(BC + BT) * CHUNKS];
    const uint32_t total = a.row_tiles * a.channel_tiles, share = (total + 7) / 8;
    // an XCD's work-groups (every eighth) take neighbouring tiles, eight tiles of tokens at a time
    const uint32_t place = blockIdx.x % 8 * share + blockIdx.x / 8;
    if (blockIdx.x / 8 >= share || place >= total) return;
    const uint32_t band = place / (8 * a.channel_tiles), in = place - band * 8 * a.channel_tiles;
    const uint32_t high = min(8u, a.row_tiles - band * 8);
    const int64_t t0 = static_cast<int64_t>(band * 8 + in % high) * BT, n0 = static_cast<int64_t>(in / high) * BC;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 32, h = lane / 32;
    const int wc = wave % WC * TC * 32, wt = wave / WC * TT * 32;

    // rows beyond the last are the last once more: their results are not stored
    const int8_t* from[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int v = e * THREADS + threadIdx.x, r = v / CHUNKS, c = v % CHUNKS;
        from[e] = (r < BC ? a.w + min(n0 + r, a.channels - 1) * a.w_stride : a.x + min(t0 + r - BC, a.rows - 1) * a.x_stride) + c * 16;
    }
    const int mine = threadIdx.x % CHUNKS * 16;  // all of a thread's chunks have one column
    i32x4 next[EACH];
    const auto fetch = [&](int64_t k) {
        if (k + BK <= a.width) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) next[e] = load_codes(from[e] + k, 16);
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) next[e] = load_codes(from[e] + k, a.width - k - mine);
        }
    };
    const auto put = [&](int to) {
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int v = e * THREADS + threadIdx.x, r = v / CHUNKS, c = v % CHUNKS;
            lds[to][r * CHUNKS + (c ^ (r / 2 % 8))] = next[e];
        }
    };
    i32x16 acc[TC][TT];
#pragma unroll
    for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = i32x16{};
    fetch(0);
    put(0);
    __syncthreads();
    int buf = 0;
    for (int64_t k = 0; k < a.width; k += BK, buf ^= 1) {
        const bool more = k + BK < a.width;
        if (more) fetch(k + BK);
#pragma unroll
        for (int s = 0; s < BK / 32; ++s) {
            i32x4 w[TC], x[TT];
#pragma unroll
            for (int i = 0; i < TC; ++i) {
                const int r = wc + 32 * i + col;
                w[i] = lds[buf][r * CHUNKS + ((2 * s + h) ^ (r / 2 % 8))];
            }
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const int r = BC + wt + 32 * j + col;
                x[j] = lds[buf][r * CHUNKS + ((2 * s + h) ^ (r / 2 % 8))];
            }
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = mma(w[i], x[j], acc[i][j]);
        }
        if (more) put(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        const int64_t t = t0 + wt + 32 * j + col;
        if (t >= a.rows) continue;
        const float x_scale = a.x_scales[t];
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int sum[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                finish<T>(a, t, n0 + wc + 32 * i + 8 * q + 4 * h, sum, x_scale);
            }
    }
}

// Few tokens (TT blocks of 32): a work-group takes 32 channels, its eight waves an eighth of the contraction
// each, straight from memory to the matrix cores; their sums meet in LDS, as integers in any order.
constexpr int kFewWaves = 8;
template <typename T, int TT>
__global__ __launch_bounds__(kFewWaves * 64) void int8_few_kernel(LinearArgs a) {
    __shared__ int sums[TT * 32][33];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 32, h = lane / 32;
    for (int i = threadIdx.x; i < TT * 32 * 33; i += kFewWaves * 64) sums[i / 33][i % 33] = 0;
    __syncthreads();
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 32;
    const int8_t* w = a.w + min(n0 + col, a.channels - 1) * a.w_stride;
    const int8_t* x[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) x[j] = a.x + min(static_cast<int64_t>(32 * j + col), a.rows - 1) * a.x_stride;
    i32x16 acc[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[j] = i32x16{};
    // 128 codes a turn: this half of the wave takes 64 consecutive ones of a row
    const int64_t turns = (a.width + 127) / 128;
    for (int64_t turn = wave; turn < turns; turn += kFewWaves) {
        const int64_t k = turn * 128 + 64 * h;
        if (turn * 128 + 128 <= a.width) {
            i32x4 f[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) f[s] = load_codes(w + k + 16 * s, 16);
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                i32x4 g[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) g[s] = load_codes(x[j] + k + 16 * s, 16);
#pragma unroll
                for (int s = 0; s < 4; ++s) acc[j] = mma(f[s], g[s], acc[j]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int64_t left = a.width - k - 16 * s;
                const i32x4 f = load_codes(w + k + 16 * s, left);
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[j] = mma(f, load_codes(x[j] + k + 16 * s, left), acc[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) atomicAdd(&sums[32 * j + col][8 * (e / 4) + 4 * h + e % 4], acc[j][e]);
    __syncthreads();
    for (int i = threadIdx.x; i < TT * 32 * 8; i += kFewWaves * 64) {
        const int64_t t = i / 8;
        const int c = i % 8 * 4;
        if (t >= a.rows) continue;
        const int sum[4] = {sums[t][c], sums[t][c + 1], sums[t][c + 2], sums[t][c + 3]};
        finish<T>(a, t, n0 + c, sum, a.x_scales[t]);
    }
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int mgopt_int8_linear(const int8_t* x_dev, int64_t x_stride, const float* x_scales_dev, const int8_t* w_dev,
                                int64_t w_stride, const float* w_scales_dev, const void* bias_dev, int32_t bias_dtype,
                                int64_t rows, int64_t width, int64_t channels, void* y_dev, int32_t dtype, void* stream) {
    if (!known_dtype(dtype) || (bias_dev && !known_dtype(bias_dtype))) return set_error(MGOPT_E_INVALID, "int8_linear: bad dtype");
    if (rows < 0 || width < 1 || channels < 0) return set_error(MGOPT_E_INVALID, "int8_linear: need rows and channels >= 0 and width >= 1");
    if (width > MGOPT_MAX_INT8_WIDTH)
        return set_error(MGOPT_E_LIMIT, "int8_linear: rows of more than " + std::to_string(MGOPT_MAX_INT8_WIDTH) + " codes, whose sums pass 32 bits");
    if (rows == 0 || channels == 0) return 0;
    if (!x_dev || !x_scales_dev || !w_dev || !w_scales_dev || !y_dev) return set_error(MGOPT_E_INVALID, "int8_linear: NULL argument");
    LinearArgs a{};
    a.x = x_dev, a.w = w_dev, a.x_stride = x_stride, a.w_stride = w_stride, a.x_scales = x_scales_dev, a.w_scales = w_scales_dev;
    a.bias = bias_dev, a.bias_dtype = bias_dtype, a.y = y_dev, a.rows = rows, a.width = width, a.channels = channels;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (rows <= 64) {
            const int64_t blocks = (channels + 31) / 32;
            if (blocks > max_blocks(kFewWaves * 64)) return set_error(MGOPT_E_LIMIT, "int8_linear: too many channels");
            const dim3 grid(static_cast<uint32_t>(blocks)), block(kFewWaves * 64);
            if (rows <= 32) hipLaunchKernelGGL((int8_few_kernel<T, 1>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((int8_few_kernel<T, 2>), grid, block, 0, s, a);
            return launched("int8_linear");
        }
        const auto tiles = [&](int64_t bt, int64_t bc, int threads) -> int64_t {
            const int64_t r = (rows + bt - 1) / bt, c = (channels + bc - 1) / bc;
            if (r > int64_t{max_blocks(threads)} / 16 / c) return -1;
            a.row_tiles = static_cast<uint32_t>(r), a.channel_tiles = static_cast<uint32_t>(c);
            return (r * c + 7) / 8 * 8;
        };
        if ((rows + 255) / 256 * ((channels + 255) / 256) >= 256) {
            const int64_t grid = tiles(256, 256, 512);
            if (grid < 0) return set_error(MGOPT_E_LIMIT, "int8_linear: too many tiles");
            hipLaunchKernelGGL((int8_linear_kernel<T, 4, 2, 2, 4>), dim3(static_cast<uint32_t>(grid)), dim3(512), 0, s, a);
        } else {
            const int64_t grid = tiles(64, 64, 256);
            if (grid < 0) return set_error(MGOPT_E_LIMIT, "int8_linear: too many tiles");
            hipLaunchKernelGGL((int8_linear_kernel<T, 2, 2, 1, 1>), dim3(static_cast<uint32_t>(grid)), dim3(256), 0, s, a);
        }
        return launched("int8_linear");
    });
}

}  // extern "C"
