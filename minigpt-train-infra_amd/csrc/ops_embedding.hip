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
// rows the tokens name when it accumulates.  16,384 tokens of 4,096 bf16, 151,936
// rows, ids whose frequency falls as one over their rank (7,100 distinct): lookup
// 38 us (134 MB written, 5 TB/s with what it reads); accumulated gradient: sort
// 24 us in four launches, bound by their latency, sums 58 us (4.6 TB/s), joining 10.
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

// N elements as they came; those past `left` are zeros.  NT: streamed.
template <typename T, int N, bool NT = false>
__device__ __forceinline__ vec_t<T, N> load_raw(const T* p, int64_t left) {
    if (left >= N) {
        if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const vec_t<T, N>*>(p));
        else return *reinterpret_cast<const vec_t<T, N>*>(p);
    }
    vec_t<T, N> v = {};
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < left) v[i] = p[i];
    return v;
}

// K tokens a thread, kBlock >> shift apart: the ids and then the rows of all of
// them are on their way before the first is written.
template <typename TW, typename TO, int K>
__global__ __launch_bounds__(kBlock) void lookup_kernel(LookupArgs a) {
    constexpr int N = 16 / (sizeof(TW) > sizeof(TO) ? sizeof(TW) : sizeof(TO));
    const int64_t per = kBlock >> a.shift;
    const int64_t t0 = a.first + static_cast<int64_t>(blockIdx.x) * (per * K) + (threadIdx.x >> a.shift);
    int64_t id[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int64_t t = t0 + k * per;
        id[k] = t < a.n ? id_at(a.ids, t, a.id_bytes) : -1;
    }
    const int64_t step = int64_t{N} << a.shift;
    for (int64_t c = static_cast<int64_t>(threadIdx.x & ((1u << a.shift) - 1)) * N; c < a.width; c += step) {
        vec_t<TW, N> w[K];
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (id[k] >= 0 && id[k] < a.rows) w[k] = load_raw<TW, N>(static_cast<const TW*>(a.weight) + id[k] * a.width + c, a.width - c);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t t = t0 + k * per;
            if (t >= a.n) break;
            const bool known = id[k] >= 0 && id[k] < a.rows;
            float v[N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = known ? static_cast<float>(w[k][i]) * a.scale : __builtin_nanf("");
            store_some<N>(static_cast<TO*>(a.out) + t * a.width + c, v, a.width - c);
        }
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

// Everything else sorts: the tokens by id, stably, so that a row's tokens are
// neighbours in their order; then the sorted list is cut in pieces of equal
// length, whatever rows they touch, and the pieces' sums are joined.
//
// The sort is a radix sort, at most kDigitBits a pass, from the low digit up.  A pass
// counts every tile's digits (and, of many tiles, scans the counts), and then
// places each token behind the tokens of smaller digits, those of its digit in
// earlier tiles, and those before it in its tile.  Ids that name no row, and the padding's, become the key `rows`
// and end up last.

constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;  // at most
constexpr int kSortBlock = 512, kSortItems = 4, kTile = kSortBlock * kSortItems, kSortWaves = kSortBlock / 64;
static_assert(kSortBlock == kDigits, "a thread a digit");

struct SortArgs {
    const void* ids;           // first pass
    const uint32_t *keys, *tokens;
    uint32_t *keys_out, *tokens_out;
    uint32_t* counts;          // [tiles + 1][kDigits]
    int64_t rows, padding;
    uint32_t n, tiles;
    int32_t id_bytes, shift;   // the digit's lowest bit
    int32_t scanned;           // counts hold what scan_kernel makes of them
    char* zeros;               // what the work-groups past the tiles clear: a multiple of 16 bytes but in the last launch
    int64_t zero_bytes;
};

__device__ __forceinline__ uint32_t key_at(const SortArgs& a, uint32_t t) {
    if (a.keys != nullptr) return a.keys[t];
    const int64_t id = id_at(a.ids, t, a.id_bytes);
    return static_cast<uint32_t>(id < 0 || id >= a.rows || id == a.padding ? a.rows : id);
}

// Clears a.zeros with the work-groups from `first` on.
__device__ __forceinline__ void clear(const SortArgs& a, uint32_t first) {
    const int64_t vecs = a.zero_bytes / 16, step = static_cast<int64_t>(gridDim.x - first) * blockDim.x;
    const vec_t<uint16_t, 8> zero = {};
    int64_t i = static_cast<int64_t>(blockIdx.x - first) * blockDim.x + threadIdx.x;
    if (i < a.zero_bytes % 16 / 2) reinterpret_cast<uint16_t*>(a.zeros)[vecs * 8 + i] = 0;
    for (; i < vecs; i += step) reinterpret_cast<vec_t<uint16_t, 8>*>(a.zeros)[i] = zero;
}

template <int BITS>
__global__ __launch_bounds__(kSortBlock) void count_kernel(SortArgs a) {
    if (blockIdx.x >= a.tiles) return clear(a, a.tiles);
    __shared__ uint32_t count[kDigits];
    count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t t = blockIdx.x * kTile + k * kSortBlock + threadIdx.x;
        if (t < a.n) atomicAdd(&count[key_at(a, t) >> a.shift & ((1u << BITS) - 1)], 1u);
    }
    __syncthreads();
    a.counts[static_cast<int64_t>(blockIdx.x) * kDigits + threadIdx.x] = count[threadIdx.x];
}

// Each tile's counts become the numbers in the tiles before it, digit by digit,
// and the row past the tiles the totals.  A work-group takes kScanDigits digits,
// its threads equal ranges of the tiles.
constexpr int kScanDigits = 16, kScanBlock = 1024, kScanParts = kScanBlock / kScanDigits;
__global__ __launch_bounds__(kScanBlock) void scan_kernel(uint32_t* counts, uint32_t tiles) {
    __shared__ uint32_t sums[kScanParts][kScanDigits];
    const uint32_t d = threadIdx.x % kScanDigits, part = threadIdx.x / kScanDigits;
    const uint32_t per = (tiles + kScanParts - 1) / kScanParts;
    const uint32_t begin = min(part * per, tiles), end = min(begin + per, tiles);
    uint32_t* const at = counts + blockIdx.x * kScanDigits + d;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t b = begin; b < end; ++b) sum += at[static_cast<int64_t>(b) * kDigits];
    sums[part][d] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (uint32_t p = 0; p < kScanParts; ++p) {
        if (p < part) before += sums[p][d];
        all += sums[p][d];
    }
    constexpr uint32_t kAhead = 8;
    for (uint32_t b = begin; b < end; b += kAhead) {
        uint32_t x[kAhead];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) x[u] = b + u < end ? at[static_cast<int64_t>(b + u) * kDigits] : 0;
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
            if (b + u < end) at[static_cast<int64_t>(b + u) * kDigits] = before;
            before += x[u];
        }
    }
    if (part == 0) at[static_cast<int64_t>(tiles) * kDigits] = all;
}

// The exclusive sum of x over the work-group's WAVES waves.
template <int WAVES>
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* wave_sums) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    uint32_t run = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y = __shfl_up(run, off);
        if (lane >= static_cast<uint32_t>(off)) run += y;
    }
    if (lane == 63) wave_sums[wave] = run;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < wave; ++w) base += wave_sums[w];
    __syncthreads();  // before the next use
    return base + run - x;
}

// The places within their digits of a tile's elements: element k of a thread
// is the tile's wave * 64 * ITEMS + k * 64 + lane.  rank counts those of its
// digit before it in its wave, used[w][d] becomes the number of digit d in the
// waves before w, and thread d's return value the number in the tile.  The
// lanes of one digit are found by a vote per bit.
template <int BITS, int WAVES, int ITEMS>
__device__ __forceinline__ uint32_t rank_tile(const uint32_t (&digit)[ITEMS], const bool (&on)[ITEMS],
                                              uint16_t (&used)[WAVES][kDigits], uint32_t (&rank)[ITEMS]) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    for (uint32_t i = threadIdx.x; i < WAVES * kDigits / 2; i += WAVES * 64) reinterpret_cast<uint32_t*>(used)[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        uint64_t same = __ballot(on[k]);
#pragma unroll
        for (int bit = 0; bit < BITS; ++bit) {
            const bool b = digit[k] >> bit & 1u;
            const uint64_t vote = __ballot(b);
            same &= b ? vote : ~vote;
        }
        const uint32_t before = static_cast<uint32_t>(__popcll(same & ((uint64_t{1} << lane) - 1)));
        // the wave's lanes read the counter, then the first of each digit moves it on
        volatile uint16_t* counter = &used[wave][digit[k]];
        const uint32_t old = *counter;
        __builtin_amdgcn_wave_barrier();
        if (on[k] && before == 0) *counter = static_cast<uint16_t>(old + static_cast<uint32_t>(__popcll(same)));
        __builtin_amdgcn_wave_barrier();
        rank[k] = old + before;
    }
    __syncthreads();
    uint32_t sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const uint32_t x = used[w][threadIdx.x];
            used[w][threadIdx.x] = static_cast<uint16_t>(sum);
            sum += x;
        }
    }
    __syncthreads();
    return sum;
}

template <int BITS>
__global__ __launch_bounds__(kSortBlock) void place_kernel(SortArgs a) {
    if (blockIdx.x >= a.tiles) return clear(a, a.tiles);
    __shared__ uint16_t used[kSortWaves][kDigits];
    __shared__ uint32_t base[kDigits], wave_sums[kSortWaves];
    const uint32_t d = threadIdx.x, lane = d % 64, wave = d / 64, begin = blockIdx.x * kTile;
    uint32_t earlier = 0, all = 0;  // elements of digit d
    if (a.scanned) {
        earlier = a.counts[static_cast<int64_t>(blockIdx.x) * kDigits + d];
        all = a.counts[static_cast<int64_t>(a.tiles) * kDigits + d];
    } else {
#pragma unroll 8
        for (uint32_t b = 0; b < a.tiles; ++b) {
            const uint32_t x = a.counts[static_cast<int64_t>(b) * kDigits + d];
            all += x;
            earlier += b < blockIdx.x ? x : 0;
        }
    }
    uint32_t key[kSortItems], token[kSortItems], digit[kSortItems];
    bool on[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const uint32_t t = begin + wave * (64 * kSortItems) + k * 64 + lane;
        on[k] = t < a.n;
        key[k] = on[k] ? key_at(a, t) : 0;
        token[k] = on[k] && a.tokens != nullptr ? a.tokens[t] : t;
        digit[k] = key[k] >> a.shift & ((1u << BITS) - 1);
    }
    uint32_t rank[kSortItems];
    rank_tile<BITS>(digit, on, used, rank);
    base[d] = sum_before<kSortWaves>(all, wave_sums) + earlier;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        if (!on[k]) continue;
        const uint32_t at = base[digit[k]] + used[wave][digit[k]] + rank[k];
        a.keys_out[at] = key[k];
        a.tokens_out[at] = token[k];
    }
}

// All passes over a list of at most WAVES * 64 * ITEMS tokens by one
// work-group, in LDS.  A key and its token share 32 bits: random accesses to the
// LDS are what bounds it.
constexpr int kWholeKeyBits = 19;
template <int BITS, int WAVES, int ITEMS>
__global__ __launch_bounds__(WAVES * 64) void sort_whole_kernel(SortArgs a, int32_t bits) {
    constexpr int kMost = WAVES * 64 * ITEMS;
    static_assert(kMost <= 1 << (32 - kWholeKeyBits) && WAVES * 64 >= kDigits, "a token's bits, a thread a digit");
    if (blockIdx.x >= 1) return clear(a, 1);
    __shared__ uint32_t list[kMost], wave_sums[WAVES];
    __shared__ uint16_t used[WAVES][kDigits];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, begin = wave * (64 * ITEMS) + lane;
    uint32_t item[ITEMS], digit[ITEMS], rank[ITEMS];
    bool on[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const uint32_t t = begin + k * 64;
        on[k] = t < a.n;
        item[k] = (on[k] ? key_at(a, t) : 0) | t << kWholeKeyBits;
    }
    for (int32_t shift = 0; shift < bits; shift += BITS) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            digit[k] = (item[k] & ((1u << kWholeKeyBits) - 1)) >> shift & ((1u << BITS) - 1);
        }
        const uint32_t sum = rank_tile<BITS>(digit, on, used, rank);
        const uint32_t before = sum_before<WAVES>(sum, wave_sums);
        if (threadIdx.x < kDigits) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) used[w][threadIdx.x] += static_cast<uint16_t>(before);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (on[k]) list[used[wave][digit[k]] + rank[k]] = item[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (on[k]) item[k] = list[begin + k * 64];
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if (!on[k]) continue;
        a.keys_out[begin + k * 64] = item[k] & ((1u << kWholeKeyBits) - 1);
        a.tokens_out[begin + k * 64] = item[k] >> kWholeKeyBits;
    }
}

struct SumArgs {
    const uint32_t *keys, *tokens;  // sorted
    const void* grad_out;
    void* grad;
    float* partials;                // [pieces][2][width]
    int64_t rows, width;
    uint32_t n, piece, pieces;
    uint32_t shift, chunks;         // as GradArgs
    int32_t accumulate;
    float scale;
};

// A group of 1 << shift threads sums the rows of one piece of the sorted list
// over its columns.  A run of one key that lies inside the piece is written to
// its row; one that began before it goes to the piece's first partial row, one
// that began in it and goes on after it to the second.  The rows of kAhead
// tokens, and what the weight rows that end among them hold, are on their way
// at once.  WIDE: a wave has one piece, so that its keys are scalars.
template <typename TG, typename TW, bool WIDE>
__global__ __launch_bounds__(kBlock) void sum_pieces_kernel(SumArgs a) {
    constexpr int N = 16 / (sizeof(TG) > sizeof(TW) ? sizeof(TG) : sizeof(TW)), kAhead = 4;
    const uint32_t pb = blockIdx.x / a.chunks, cb = blockIdx.x - pb * a.chunks;
    uint32_t piece = pb * (kBlock >> a.shift) + (threadIdx.x >> a.shift);
    if constexpr (WIDE) piece = __builtin_amdgcn_readfirstlane(piece);
    const int64_t c = (static_cast<int64_t>(cb) * kBlock + (threadIdx.x & ((1u << a.shift) - 1))) * N, left = a.width - c;
    if (piece >= a.pieces || left <= 0) return;
    const uint32_t none = static_cast<uint32_t>(a.rows), first = piece * a.piece;
    const uint32_t last = a.n - first < a.piece ? a.n : first + a.piece;
    // The keys and tokens of a batch come together, and the next batch's while its
    // rows are on their way.  The lists are longer than n by kAhead, so that no
    // load waits for a comparison; keys from n on count as none.
    uint32_t key[kAhead + 1], token[kAhead];
    const auto fetch = [&](uint32_t i) {
#pragma unroll
        for (int u = 0; u <= kAhead; ++u) key[u] = a.keys[i + u];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) token[u] = a.tokens[i + u];
#pragma unroll
        for (int u = 0; u <= kAhead; ++u) key[u] = i + u < a.n ? key[u] : none;
    };
    const uint32_t before = first > 0 ? a.keys[first - 1] : none;
    fetch(first);
    bool head = before == key[0];  // the piece's first run began before it
    bool open = false;             // the run at hand goes on
    float sum[N] = {};
    for (uint32_t i = first; i < last && key[0] != none; i += kAhead) {  // the ids that name no row come last
        uint32_t row[kAhead + 1];
#pragma unroll
        for (int u = 0; u <= kAhead; ++u) row[u] = key[u];
        vec_t<TG, N> v[kAhead];
        vec_t<TW, N> old[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u >= last || row[u] == none) continue;
            v[u] = load_raw<TG, N, true>(static_cast<const TG*>(a.grad_out) + static_cast<int64_t>(token[u]) * a.width + c, left);
            if (a.accumulate && row[u + 1] != row[u])
                old[u] = load_raw<TW, N>(static_cast<const TW*>(a.grad) + static_cast<int64_t>(row[u]) * a.width + c, left);
        }
        if (i + kAhead < last) fetch(i + kAhead);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u >= last || row[u] == none) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += static_cast<float>(v[u][j]);
            open = row[u + 1] == row[u];
            if (open) continue;
            if (head) {
                store_some<N>(a.partials + static_cast<int64_t>(piece) * 2 * a.width + c, sum, left);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] = a.accumulate ? fmaf(sum[j], a.scale, static_cast<float>(old[u][j])) : sum[j] * a.scale;
                store_some<N>(static_cast<TW*>(a.grad) + static_cast<int64_t>(row[u]) * a.width + c, sum, left);
            }
            head = false;
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] = 0.0f;
        }
    }
    if (open) store_some<N>(a.partials + (static_cast<int64_t>(piece) * 2 + (head ? 0 : 1)) * a.width + c, sum, left);
}

// Joins the runs that cross pieces.  The work-group of the piece in which a run
// began adds the partial rows of the pieces that it goes on through: 64 lanes
// over the columns, its waves over the pieces in turn, joined in a fixed order.
template <int N, typename TW>
__global__ __launch_bounds__(kBlock) void join_pieces_kernel(SumArgs a) {
    constexpr uint32_t kWaves = kBlock / 64;
    __shared__ float part[kWaves][64][N + 1];
    const uint32_t piece = blockIdx.x / a.chunks, cb = blockIdx.x - piece * a.chunks;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    if (piece + 1 >= a.pieces) return;
    const uint32_t first = piece * a.piece, next = first + a.piece, row = a.keys[next];
    if (row >= a.rows || a.keys[next - 1] != row) return;                       // nothing crosses this piece's end
    if (a.keys[first] == row && first > 0 && a.keys[first - 1] == row) return;  // it began before this piece
    // the pieces it goes on through: those whose first key is its
    uint32_t more = 0;
    for (uint32_t q = piece + 1;; q += kBlock) {
        const uint32_t here = q + threadIdx.x;
        const int n = __syncthreads_count(here < a.pieces && a.keys[here * a.piece] == row);
        more += static_cast<uint32_t>(n);
        if (n < kBlock) break;
    }
    const int64_t c = (static_cast<int64_t>(cb) * 64 + lane) * N, left = a.width - c;
    float sum[N] = {};
    if (left > 0) {
        const float* at = a.partials + static_cast<int64_t>(piece + 1) * 2 * a.width + c;
        if (wave == 0) load_some<N>(sum, at - a.width, left);
        constexpr uint32_t kAhead = 8;
        uint32_t q = wave;
        for (; left >= N && q + (kAhead - 1) * kWaves < more; q += kAhead * kWaves) {
            float v[kAhead][N];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) load<N>(v[u], at + static_cast<int64_t>(q + u * kWaves) * 2 * a.width);
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] += v[u][j];
        }
        for (; q < more; q += kWaves) {
            float v[N];
            load_some<N>(v, at + static_cast<int64_t>(q) * 2 * a.width, left);
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) part[wave][lane][j] = sum[j];
    __syncthreads();
    if (wave != 0 || left <= 0) return;
    for (uint32_t w = 1; w < kWaves; ++w)
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += part[w][lane][j];
    TW* out = static_cast<TW*>(a.grad) + static_cast<int64_t>(row) * a.width + c;
    float old[N] = {};
    if (a.accumulate) load_some<N>(old, out, left);
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = fmaf(sum[j], a.scale, old[j]);
    store_some<N>(out, sum, left);
}

// Which form: a work-group per row, or the sort.  A whole call in us, by row /
// sorted, bf16, ids whose frequency falls as one over their rank and all the same:
//                          accumulated                   written whole
//   tokens  rows    width  by rank       the same        by rank        the same
//   256     96      128    5.0 / 15.3    6.5 / 13.7      4.6 / 14.1     6.5 / 13.5
//   1,024   96      128    5.6 / 16.2    17.7 / 16.7     5.6 / 15.1     17.4 / 16.5
//   1,024   1,000   256    6.0 / 18.9    30.9 / 20.7     5.9 / 18.2     30.8 / 20.6
//   64      8,192   768    7.3 / 15.8    11.5 / 14.1     9.9 / 16.5     13.2 / 15.1
//   10      50,304  768    32.7 / 12.9   32.4 / 13.2     43.3 / 18.3    43.4 / 19.0
//   3       151,936 4,096  187 / 11.7    186 / 11.4      245 / 285      245 / 286
// and beyond the bounds:
//   256     1,000   4,096  7.3 / 17.0    59.0 / 17.2     8.0 / 17.6     60.2 / 17.9
//   1,024   96      768    19.4 / 15.0   117 / 17.0      19.2 / 14.7    117 / 16.8
//   64      16,000  4,096  22.7 / 16.2   25.2 / 14.8     31.3 / 27.6    39.3 / 26.7
//   16      50,304  768    32.5 / 13.1   32.4 / 13.2     43.2 / 18.6    43.4 / 19.0
// rows * tokens is what all rows read, tokens * width what a row that has all
// tokens sums alone.  The rows by themselves are not bounded, and a work-group each
// costs 0.6 to 1.6 ns: the few tokens (10 of 50,304 rows, 3 of 151,936) that still
// take the by-row form there would mostly be faster sorted.
constexpr int64_t kByRowWork = int64_t{1} << 19;   // rows * tokens
constexpr int64_t kByRowTerms = int64_t{1} << 17;  // tokens * width
bool by_row(int64_t n, int64_t rows, int64_t width) {
    return n == 0 || (rows <= kByRowWork / n && width <= kByRowTerms / n);
}

// Up to here one work-group sorts the whole list: at 8,183 tokens that takes
// 23 us, beside the clearing, where the two launches of each of two passes take
// 29; at 16,384, with 16 elements a thread, 44 us against 29.
constexpr int64_t kSortWhole = 8192;

// Up to here each tile of the sort adds up all tiles' counts itself, which costs
// tiles^2 reads of 2 KB a pass; beyond, a kernel of its own does it once.  A whole
// call in us, two passes, direct / scanned, by tiles of 2,048 tokens:
//   8: 32 / 38    64: 60 / 61    96: 88 / 87    128: 96 / 93    512: 215 / 182
//   2,048: 953 / 387    8,192: 10,149 / 1,318
constexpr uint32_t kDirectTiles = 96;

// Sorted positions per piece, a power of two from 8 to 64: about 8,192 waves'
// pieces, all that fit the chip at once.  Short pieces give the sums more waves,
// long ones the joining less to do; sums and joining, traced, in us, by the
// tokens of a piece:        4            8            16           32           64
//   8,183 tokens of 768     10.0 + 12.7  13.2 + 7.7   14.2 + 5.3
//   16,384 tokens of 4,096                            56.7 + 13.6  67.8 + 8.9   98.2 + 6.6
uint32_t piece_for(int64_t n, int64_t width) {
    const int64_t most = n * ((width + 511) / 512) / 8192;
    uint32_t p = 8;
    while (p < 64 && p < most) p *= 2;
    return p;
}

struct Work {
    int64_t counts, keys[2], tokens[2], partials, bytes;
};
Work work_of(int64_t n, int64_t width) {
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    Work w{};
    const int64_t tiles = (n + kTile - 1) / kTile, list = up(4 * (n + 16));  // sum_pieces_kernel reads a little past n
    w.keys[0] = up(4 * (tiles + 1) * kDigits);
    w.tokens[0] = w.keys[0] + list, w.keys[1] = w.tokens[0] + list, w.tokens[1] = w.keys[1] + list;
    w.partials = w.tokens[1] + list;
    const int64_t piece = piece_for(n, width);
    w.bytes = w.partials + (n + piece - 1) / piece * 2 * width * 4;
    return w;
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
            const int64_t per_block = kBlock >> a.shift;
            // four tokens a thread where that leaves work-groups enough for the chip
            const bool four = n >= 4 * 1024 * per_block;
            const int64_t tokens = per_block * (four ? 4 : 1), most = max_blocks(kBlock) * tokens;
            for (a.first = 0; a.first < n; a.first += most) {
                const dim3 grid(static_cast<uint32_t>((std::min(n - a.first, most) + tokens - 1) / tokens));
                if (four) hipLaunchKernelGGL((lookup_kernel<TW, TO, 4>), grid, dim3(kBlock), 0, static_cast<hipStream_t>(stream), a);
                else hipLaunchKernelGGL((lookup_kernel<TW, TO, 1>), grid, dim3(kBlock), 0, static_cast<hipStream_t>(stream), a);
                if (int rc = launched("lookup_kernel")) return rc;
            }
            return 0;
        });
    });
}

MGOPT_API int64_t mgopt_embedding_grad_workspace(int64_t n, int64_t rows, int64_t width) {
    if (n < 0 || rows < 1 || width < 1) return -1;
    return by_row(n, rows, width) ? 16 : work_of(n, width).bytes;
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
            const uint32_t shift = shift_for(vecs);
            if (by_row(n, rows, width)) {
                a.shift = shift;
                a.chunks = static_cast<uint32_t>(chunks);
                const int64_t most = max_blocks(kBlock) / chunks;
                for (a.first_row = 0; a.first_row < rows; a.first_row += most) {
                    const int64_t blocks = std::min(rows - a.first_row, most) * chunks;
                    hipLaunchKernelGGL((grad_by_row_kernel<TG, TW>), dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, a);
                    if (int rc = launched("grad_by_row_kernel")) return rc;
                }
                return 0;
            }
            if (n >= (int64_t{1} << 30) || rows >= (int64_t{1} << 31))
                return set_error(MGOPT_E_LIMIT, "embedding_grad: more than 2^30 tokens or 2^31 rows");
            const int64_t pieces = (n + piece_for(n, width) - 1) / piece_for(n, width), per_block = kBlock >> shift;
            const int64_t blocks = (pieces + per_block - 1) / per_block * chunks, join_chunks = (vecs + 63) / 64;
            if (blocks > max_blocks(kBlock) || join_chunks > max_blocks(kBlock) / pieces)
                return set_error(MGOPT_E_LIMIT, "embedding_grad: too many tokens of long rows");
            const Work work = work_of(n, width);
            char* const at = static_cast<char*>(workspace_dev);
            const auto list = [&](int64_t offset) { return reinterpret_cast<uint32_t*>(at + offset); };
            const uint32_t tiles = static_cast<uint32_t>((n + kTile - 1) / kTile);
            SortArgs o{ids_dev, nullptr, nullptr, nullptr, nullptr, list(work.counts), rows, padding_idx, static_cast<uint32_t>(n),
                       tiles, id_bytes, 0, tiles > kDirectTiles, nullptr, 0};
            int32_t bits = 1;
            while (rows >> bits) ++bits;  // of the largest key, `rows`
            const int passes = (bits + kDigitBits - 1) / kDigitBits;
            const bool eight = bits <= 8 * passes;  // bits a pass: 8 where that takes no more of them, else 9
            const bool whole = n <= kSortWhole && bits <= kWholeKeyBits;
            const int launches = whole ? 1 : 2 * passes;
            // a gradient that is written whole is cleared beside the sort, which leaves most of the chip idle: a share
            // with each launch, by the work-groups past the tiles
            int64_t dirty = accumulate ? 0 : rows * width * static_cast<int64_t>(sizeof(TW));
            const int64_t share = (dirty / launches + 15) / 16 * 16;
            const auto clearing = [&](bool rest) {
                if (o.zeros != nullptr) o.zeros += o.zero_bytes;
                else o.zeros = static_cast<char*>(grad_dev);
                o.zero_bytes = rest ? dirty : std::min(share, dirty);
                dirty -= o.zero_bytes;
                return static_cast<uint32_t>(std::min<int64_t>((o.zero_bytes + 16 * kSortBlock - 1) / (16 * kSortBlock), 2048));
            };
            int side = 0;
            if (whole) {
                o.keys_out = list(work.keys[0]), o.tokens_out = list(work.tokens[0]);
                const dim3 grid(1 + clearing(true));
                const auto sort = [&](auto digit) {
                    constexpr int BITS = decltype(digit)::value;
                    if (n <= 2048) hipLaunchKernelGGL((sort_whole_kernel<BITS, 8, 4>), grid, dim3(512), 0, s, o, bits);
                    else if (n <= 4096) hipLaunchKernelGGL((sort_whole_kernel<BITS, 16, 4>), grid, dim3(1024), 0, s, o, bits);
                    else hipLaunchKernelGGL((sort_whole_kernel<BITS, 16, 8>), grid, dim3(1024), 0, s, o, bits);
                };
                if (eight) sort(std::integral_constant<int, 8>{});
                else sort(std::integral_constant<int, 9>{});
                if (int rc = launched("sort_whole_kernel")) return rc;
                side = 1;
            } else {
                for (o.shift = 0; o.shift < bits; o.shift += eight ? 8 : 9, side ^= 1) {
                    o.keys_out = list(work.keys[side]), o.tokens_out = list(work.tokens[side]);
                    const dim3 counters(tiles + clearing(false));
                    if (eight) hipLaunchKernelGGL(count_kernel<8>, counters, dim3(kSortBlock), 0, s, o);
                    else hipLaunchKernelGGL(count_kernel<9>, counters, dim3(kSortBlock), 0, s, o);
                    if (int rc = launched("count_kernel")) return rc;
                    if (o.scanned) {
                        hipLaunchKernelGGL(scan_kernel, dim3(kDigits / kScanDigits), dim3(kScanBlock), 0, s, o.counts, tiles);
                        if (int rc = launched("scan_kernel")) return rc;
                    }
                    const dim3 grid(tiles + clearing(o.shift + (eight ? 8 : 9) >= bits));
                    if (eight) hipLaunchKernelGGL(place_kernel<8>, grid, dim3(kSortBlock), 0, s, o);
                    else hipLaunchKernelGGL(place_kernel<9>, grid, dim3(kSortBlock), 0, s, o);
                    if (int rc = launched("place_kernel")) return rc;
                    o.keys = o.keys_out, o.tokens = o.tokens_out;
                }
            }
            SumArgs m{list(work.keys[side ^ 1]), list(work.tokens[side ^ 1]), grad_out_dev, grad_dev,
                      reinterpret_cast<float*>(at + work.partials), rows, width, static_cast<uint32_t>(n), piece_for(n, width), 0, shift,
                      static_cast<uint32_t>(chunks), accumulate, scale};
            m.pieces = static_cast<uint32_t>(pieces);
            if (shift >= 6)
                hipLaunchKernelGGL((sum_pieces_kernel<TG, TW, true>), dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, m);
            else
                hipLaunchKernelGGL((sum_pieces_kernel<TG, TW, false>), dim3(static_cast<uint32_t>(blocks)), dim3(kBlock), 0, s, m);
            if (int rc = launched("sum_pieces_kernel")) return rc;
            m.chunks = static_cast<uint32_t>(join_chunks);
            hipLaunchKernelGGL((join_pieces_kernel<N, TW>), dim3(m.pieces * m.chunks), dim3(kBlock), 0, s, m);
            if (int rc = launched("join_pieces_kernel")) return rc;
            return 0;
        });
    });
}

}  // extern "C"
