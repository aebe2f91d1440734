// ops_int8_linear.hip -- products of 8-bit integers with a scale for each token
// and each output channel.
//
//     y[t][n] = (x_scales[t] * w_scales[n]) * sum_k x[t][k] * w[n][k]  (+ bias[n])
//
// The sum is exact in 32-bit integers (at most 131,071 products of magnitudes up to
// 2^14), so neither tiles nor parts of the contraction change a result; it is turned
// into a 32-bit float, scaled, added to the bias and rounded once.
//
// Many tokens are bound by the matrix cores' chain of loads from LDS and products: 8,192 x
// 4,096 x 12,288 in bf16 426 to 479 us (1.7 to 1.9 POP/s; the same loop without its
// loads reaches 2.9).  Few tokens are bound by the weights' way from memory:
// 12,288 x 4,096 codes 10 us for one token (5.0 TB/s), 17 for 64.
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

// 16 codes at an address of any alignment.
__device__ __forceinline__ i32x4 load_codes(const int8_t* p) {
    typedef int unaligned __attribute__((ext_vector_type(4), aligned(1)));
    return *reinterpret_cast<const unaligned*>(p);
}
// 16 codes from code `at` of a row of `width`, those behind the row 0: the last 16 of the row, moved down.
__device__ __forceinline__ i32x4 load_codes(const int8_t* p, int64_t at, int64_t width) {
    const int64_t n = width - at;
    if (n >= 16) return load_codes(p);
    i32x4 v{};
    if (n <= 0) return v;
    if (width < 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) v[i / 4] |= static_cast<int>((static_cast<uint32_t>(p[i]) & 0xFFu) << (8 * (i % 4)));
        return v;
    }
    typedef uint64_t two __attribute__((ext_vector_type(2)));
    const two x = __builtin_bit_cast(two, load_codes(p + n - 16));
    const uint32_t bits = static_cast<uint32_t>(16 - n) * 8;  // 8 .. 120
    two y;
    y[0] = bits < 64 ? x[0] >> bits | x[1] << (64 - bits) : x[1] >> (bits - 64);
    y[1] = bits < 64 ? x[1] >> bits : 0;
    return __builtin_bit_cast(i32x4, y);
}

__device__ __forceinline__ i32x16 mma(i32x4 a, i32x4 b, i32x16 c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float bias_at(const LinearArgs& a, int64_t n) {
    if (a.bias_dtype == MGOPT_F32) return static_cast<const float*>(a.bias)[n];
    if (a.bias_dtype == MGOPT_F16) return static_cast<float>(static_cast<const _Float16*>(a.bias)[n]);
    return static_cast<float>(static_cast<const __bf16*>(a.bias)[n]);
}

// Four channels from n on of a token of scale x_scale; those behind the last are the last's.
__device__ __forceinline__ void scaled(float (&y)[4], const LinearArgs& a, int64_t n, const int (&sum)[4], float x_scale) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t at = min(n + i, a.channels - 1);
        y[i] = static_cast<float>(sum[i]) * (x_scale * a.w_scales[at]);
        if (a.bias != nullptr) y[i] += bias_at(a, at);
    }
}

// Where chunk c (16 codes) of row r of a tile lies in LDS: chunk c ^ turn(r) of the row, so that a chunk of 16
// rows falls on all banks.
template <int CHUNKS>
__device__ __forceinline__ int turn(int r) { return r / (16 / CHUNKS) % CHUNKS; }

// A wave's load of 64 chunks, each lane's from an address of its own, to LDS behind each other.  The compiler does not
// count it: waiting is the caller's.
__device__ __forceinline__ void load_direct(i32x4* lds, const int8_t* from) {
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) i32x4*)lds));
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(from) : "memory", "m0");
}
template <int LEFT>
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(%0)" ::"i"(LEFT) : "memory"); }

// Tiles of WC * TC * 32 channels and WT * TT * 32 tokens, WC * WT waves with TC x TT blocks of 32 x 32 each, BK codes of
// the contraction at a time.  ALIGNED (rows start on 16 bytes): codes go to LDS directly, AHEAD stages before they are
// multiplied.  Otherwise they are AHEAD stages ahead in registers and one in LDS.
template <typename T, int WC, int WT, int TC, int TT, int BK, int AHEAD, bool ALIGNED>
__global__ __launch_bounds__(WC* WT * 64, 2) void int8_linear_kernel(LinearArgs a) {
    constexpr int THREADS = WC * WT * 64, BC = WC * TC * 32, BT = WT * TT * 32, CHUNKS = BK / 16, SIZE = (BC + BT) * CHUNKS;
    constexpr int EACH = SIZE / THREADS, STEP = THREADS / CHUNKS;  // STEP: rows from a thread's chunk to its next
    constexpr int BUFFERS = ALIGNED ? AHEAD + 1 : 2;
    static_assert(SIZE % THREADS == 0 && BC * CHUNKS % THREADS == 0 && STEP % 16 == 0);
    __shared__ i32x4 lds[BUFFERS][SIZE];
    const uint32_t total = a.row_tiles * a.channel_tiles, share = (total + 7) / 8;
    // an XCD's work-groups (every eighth) take neighbouring tiles, eight tiles of tokens at a time
    const uint32_t place = blockIdx.x % 8 * share + blockIdx.x / 8;
    if (blockIdx.x / 8 >= share || place >= total) return;
    const uint32_t band = place / (8 * a.channel_tiles), in = place - band * 8 * a.channel_tiles;
    const uint32_t high = min(8u, a.row_tiles - band * 8);
    const int64_t t0 = static_cast<int64_t>(band * 8 + in % high) * BT, n0 = static_cast<int64_t>(in / high) * BC;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, h = lane / 32;
    const int wc = wave % WC * TC * 32, wt = wave / WC * TT * 32;

    // A thread's chunks: places e * THREADS + threadIdx.x of LDS, one chunk of every STEP-th row.
    // Rows beyond the last are the last once more: their results are not stored.
    const int row = threadIdx.x / CHUNKS, mine = ((threadIdx.x % CHUNKS) ^ turn<CHUNKS>(row)) * 16;
    const int8_t* from[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        from[e] = (e * STEP < BC ? a.w + min(n0 + e * STEP + row, a.channels - 1) * a.w_stride
                                 : a.x + min(t0 + e * STEP + row - BC, a.rows - 1) * a.x_stride) + mine;
    const int32_t stages = static_cast<int32_t>((a.width + BK - 1) / BK), whole = static_cast<int32_t>(a.width / BK);
    i32x16 acc[TC][TT];
#pragma unroll
    for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = i32x16{};
    const auto multiply = [&](const i32x4* codes) {
#pragma unroll
        for (int s = 0; s < BK / 32; ++s) {
            i32x4 w[TC], x[TT];
#pragma unroll
            for (int i = 0; i < TC; ++i) {
                const int r = wc + 32 * i + col;
                w[i] = codes[r * CHUNKS + ((2 * s + h) ^ turn<CHUNKS>(r))];
            }
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const int r = BC + wt + 32 * j + col;
                x[j] = codes[r * CHUNKS + ((2 * s + h) ^ turn<CHUNKS>(r))];
            }
#pragma unroll
            for (int i = 0; i < TC; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = mma(w[i], x[j], acc[i][j]);
        }
    };
    if constexpr (ALIGNED) {
        const auto fetch = [&](int32_t stage, int to) {
            const int64_t k = static_cast<int64_t>(stage) * BK;
            if (stage < whole) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) load_direct(&lds[to][e * THREADS + wave * 64], from[e] + k);
            } else if (stage < stages) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) lds[to][e * THREADS + threadIdx.x] = load_codes(from[e] + k, k + mine, a.width);
            }
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) fetch(u, u);
        int buf = 0;
        for (int32_t stage = 0; stage < stages; ++stage) {
            // this stage's loads are done when only those of the AHEAD - 1 behind it are not
            if (stage + AHEAD - 1 < whole) landed<EACH*(AHEAD - 1)>();
            else landed<0>();
            __syncthreads();
            fetch(stage + AHEAD, buf == 0 ? AHEAD : buf - 1);  // where the stage before this one was: all waves have left it
            multiply(lds[buf]);
            buf = buf == AHEAD ? 0 : buf + 1;
        }
    } else {
        i32x4 next[AHEAD][EACH];
        const auto fetch = [&](int32_t stage, int set) {
            const int64_t k = static_cast<int64_t>(stage) * BK;
            if (stage < whole) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) next[set][e] = load_codes(from[e] + k);
            } else if (stage < stages) {
#pragma unroll
                for (int e = 0; e < EACH; ++e) next[set][e] = load_codes(from[e] + k, k + mine, a.width);
            }
        };
        const auto put = [&](int to, int set) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) lds[to][e * THREADS + threadIdx.x] = next[set][e];
        };
        fetch(0, 0);
        put(0, 0);
#pragma unroll
        for (int u = 1; u <= AHEAD; ++u) fetch(u, u % AHEAD);
        __syncthreads();
        int buf = 0;
        for (int32_t first = 0; first < stages; first += AHEAD)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int32_t stage = first + u;
                if (stage >= stages) break;
                multiply(lds[buf]);
                if (stage + 1 < stages) {
                    put(buf ^ 1, (u + 1) % AHEAD);
                    fetch(stage + 1 + AHEAD, (u + 1) % AHEAD);
                }
                __syncthreads();
                buf ^= 1;
            }
    }
    // A token's channels lie four by four in lanes that are rows of y apart: they pass through LDS, to be written in
    // rows.  8,192 x 4,096 x 12,288 in bf16: 479 us, 512 with 8 bytes a lane written as they lie.
    constexpr int PITCH = BC + 16 / static_cast<int>(sizeof(T)), PER = 16 / static_cast<int>(sizeof(T));
    static_assert(sizeof(lds) >= WT * 32 * PITCH * sizeof(T));
    T* const out = reinterpret_cast<T*>(&lds[0][0]);
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        const float x_scale = a.x_scales[min(t0 + wt + 32 * j + col, a.rows - 1)];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TC; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int sum[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                const int c = wc + 32 * i + 8 * q + 4 * h;
                float y[4];
                scaled(y, a, n0 + c, sum, x_scale);
                store<4>(out + (wave / WC * 32 + col) * PITCH + c, y);
            }
        __syncthreads();
        for (int v = threadIdx.x; v < WT * 32 * (BC / PER); v += THREADS) {
            const int r = v / (BC / PER), c = v % (BC / PER) * PER;
            const int64_t t = t0 + r / 32 * (TT * 32) + 32 * j + r % 32, n = n0 + c;
            if (t >= a.rows) continue;
            const T* const at = out + r * PITCH + c;
            T* const to = static_cast<T*>(a.y) + t * a.channels + n;
            if (n + PER <= a.channels) {
                *reinterpret_cast<vec_t<T, PER>*>(to) = *reinterpret_cast<const vec_t<T, PER>*>(at);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (n + e < a.channels) to[e] = at[e];
            }
        }
    }
}

// Few tokens (TT blocks of 32): a work-group takes 32 channels, its eight waves an eighth of each 256 codes of the
// contraction; their sums meet in LDS, as integers in any order.  Three stages of codes are in LDS or on
// their way.  With one block of tokens a CU holds three work-groups (53,376 bytes of LDS each) and has up to 96 KB in flight,
// which is what the weights' stream needs: 12,288 x 4,096 codes at 5.0 TB/s.  With two it holds one (82,176 bytes; two
// work-groups are 512 too many), with 48 KB in flight: 2.8 TB/s for 64 tokens.
constexpr int kFewWaves = 8, kFewCodes = 32 * kFewWaves, kStages = 3;
template <typename T, int TT, bool ALIGNED>
__global__ __launch_bounds__(kFewWaves * 64) void int8_few_kernel(LinearArgs a) {
    constexpr int CHUNKS = kFewCodes / 16, ROWS = 32 + 32 * TT, THREADS = kFewWaves * 64, EACH = ROWS * CHUNKS / THREADS;
    static_assert(ROWS * CHUNKS % THREADS == 0 && THREADS / CHUNKS == 32);
    __shared__ i32x4 lds[kStages][ROWS * CHUNKS];
    __shared__ int sums[TT * 32][33];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), col = lane % 32, h = lane / 32;
    for (int i = threadIdx.x; i < TT * 32 * 33; i += THREADS) sums[i / 33][i % 33] = 0;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 32;
    // a thread's chunks: row threadIdx.x / CHUNKS of the weights and of each block of tokens; chunk c of row r lies at chunk
    // c ^ r % 16
    const int row = threadIdx.x / CHUNKS, mine = ((threadIdx.x % CHUNKS) ^ (row % 16)) * 16;
    const int8_t* from[EACH];
    from[0] = a.w + min(n0 + row, a.channels - 1) * a.w_stride + mine;
#pragma unroll
    for (int e = 1; e < EACH; ++e) from[e] = a.x + min(static_cast<int64_t>(32 * (e - 1) + row), a.rows - 1) * a.x_stride + mine;
    const int64_t stages = (a.width + kFewCodes - 1) / kFewCodes, direct = ALIGNED ? a.width / kFewCodes : 0;
    const auto fetch = [&](int64_t stage, int to) {
        const int64_t k = stage * kFewCodes;
        if (stage < direct) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) load_direct(&lds[to][e * THREADS + wave * 64], from[e] + k);
        } else if (stage < stages) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) lds[to][e * THREADS + threadIdx.x] = load_codes(from[e] + k, k + mine, a.width);
        }
    };
    i32x16 acc[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[j] = i32x16{};
    fetch(0, 0), fetch(1, 1);
    int buf = 0;
    for (int64_t stage = 0; stage < stages; ++stage) {
        // this stage's loads are done when only the next one's EACH are not
        if (stage + 1 < direct) landed<EACH>();
        else landed<0>();
        __syncthreads();
        fetch(stage + 2, buf == 0 ? 2 : buf - 1);  // where the stage before this one was: all waves have left it
        const int c = (2 * wave + h) ^ (col % 16);
        const i32x4 w = lds[buf][col * CHUNKS + c];
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[j] = mma(w, lds[buf][(32 + 32 * j + col) * CHUNKS + c], acc[j]);
        buf = buf == 2 ? 0 : buf + 1;
    }
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) atomicAdd(&sums[32 * j + col][8 * (e / 4) + 4 * h + e % 4], acc[j][e]);
    __syncthreads();
    for (int i = threadIdx.x; i < TT * 32 * 8; i += THREADS) {
        const int64_t t = i / 8;
        const int c = i % 8 * 4;
        if (t >= a.rows) continue;
        const int sum[4] = {sums[t][c], sums[t][c + 1], sums[t][c + 2], sums[t][c + 3]};
        float y[4];
        if (n0 + c >= a.channels) continue;
        scaled(y, a, n0 + c, sum, a.x_scales[t]);
        store_some<4>(static_cast<T*>(a.y) + t * a.channels + n0 + c, y, a.channels - n0 - c);
    }
}

template <int V>
using Int = std::integral_constant<int, V>;
constexpr int kBigCodes = 128, kBigAhead = 1, kMidAhead = 1, kSmallAhead = 2;

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
    const bool aligned = (reinterpret_cast<uintptr_t>(x_dev) | reinterpret_cast<uintptr_t>(w_dev) | static_cast<uint64_t>(x_stride | w_stride)) % 16 == 0;
    return with_dtype(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (rows <= 64) {
            const int64_t blocks = (channels + 31) / 32;
            if (blocks > max_blocks(kFewWaves * 64)) return set_error(MGOPT_E_LIMIT, "int8_linear: too many channels");
            const dim3 grid(static_cast<uint32_t>(blocks)), block(kFewWaves * 64);
            if (rows <= 32 && aligned) hipLaunchKernelGGL((int8_few_kernel<T, 1, true>), grid, block, 0, s, a);
            else if (rows <= 32) hipLaunchKernelGGL((int8_few_kernel<T, 1, false>), grid, block, 0, s, a);
            else if (aligned) hipLaunchKernelGGL((int8_few_kernel<T, 2, true>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((int8_few_kernel<T, 2, false>), grid, block, 0, s, a);
            return launched("int8_linear");
        }
        const auto tiles = [&](int64_t bt, int64_t bc, int threads) -> int64_t {
            const int64_t r = (rows + bt - 1) / bt, c = (channels + bc - 1) / bc;
            if (r > int64_t{max_blocks(threads)} / 16 / c) return -1;
            a.row_tiles = static_cast<uint32_t>(r), a.channel_tiles = static_cast<uint32_t>(c);
            return (r * c + 7) / 8 * 8;
        };
        const auto launch = [&](auto wc, auto wt, auto tc, auto tt, auto bk, auto ahead) -> int {
            constexpr int WC = decltype(wc)::value, WT = decltype(wt)::value, TC = decltype(tc)::value, TT = decltype(tt)::value;
            constexpr int BK = decltype(bk)::value, AHEAD = decltype(ahead)::value, THREADS = WC * WT * 64;
            const int64_t grid = tiles(WT * TT * 32, WC * TC * 32, THREADS);
            if (grid < 0) return set_error(MGOPT_E_LIMIT, "int8_linear: too many tiles");
            const dim3 blocks(static_cast<uint32_t>(grid)), threads(THREADS);
            if (aligned) hipLaunchKernelGGL((int8_linear_kernel<T, WC, WT, TC, TT, BK, AHEAD, true>), blocks, threads, 0, s, a);
            else hipLaunchKernelGGL((int8_linear_kernel<T, WC, WT, TC, TT, BK, (TC * TT > 4 ? 1 : 2), false>), blocks, threads, 0, s, a);
            return launched("int8_linear");
        };
        const auto count = [&](int64_t side) { return (rows + side - 1) / side * ((channels + side - 1) / side); };
        // tiles of 256 where they fill the chip, of 128 where those do, of 64 otherwise: 1,024 x 12,288 x 4,096 84 us with
        // tiles of 128, 130 of 64; 512 x 4,096 x 4,096 20 us with tiles of 64, 30 of 128; 8,192 x 12,288 x 4,096 479 us
        // with tiles of 256, 587 of 128
        if (count(256) >= 256) return launch(Int<4>{}, Int<2>{}, Int<2>{}, Int<4>{}, Int<kBigCodes>{}, Int<kBigAhead>{});
        if (count(128) >= 256) return launch(Int<2>{}, Int<2>{}, Int<2>{}, Int<2>{}, Int<128>{}, Int<kMidAhead>{});
        return launch(Int<2>{}, Int<2>{}, Int<1>{}, Int<1>{}, Int<128>{}, Int<kSmallAhead>{});
    });
}

}  // extern "C"
