// ops_attention.hip -- attention of grouped heads over batches, packed sequences
// and caches, and its backward pass.
//
// For a sequence of n queries and m keys, query i and key j of a head, x_ij =
// scale * q_i . k_j where j is seen (j <= i + m - n if causal, so that the last
// query sees the last key):
//
//     lse_i = log sum_j exp(x_ij)      p_ij = exp(x_ij - lse_i)      out_i = sum_j p_ij v_j
//
// and with g the gradient of out, delta_i = g_i . out_i:
//
//     ds_ij = p_ij (g_i . v_j - delta_i)    dq_i = scale sum_j ds_ij k_j
//     dv_j = sum_i p_ij g_i                 dk_j = scale sum_i ds_ij q_i
//
// A query that sees no key has out 0, lse -inf and no gradient; one whose largest
// score passes 32 bits is NaN.
//
// The query heads that share a key head are rows of one matrix: row r of a
// sequence is query r / group, head r % group of the group, so that keys and
// values are read once for all of them and few queries of many heads fill a tile.
//
// All products run on the matrix cores in blocks of 32 x 32.  The block's C layout
// leaves in a lane one column and, in its 16 registers, rows 8 (e/4) + 4 (lane/32) +
// e%4.  Scores are formed transposed (forward, dq: a column a query; dk and dv: a
// column a key), so that softmax statistics are one lane's and its partner's, and the
// probabilities are already the B operand of the product that follows, for that order
// of the contraction; the A operand is read from LDS transposed, in the same order.
//
// dq and dk, dv are kernels of their own, without atomics: scores and g v^T are
// formed twice, 7 products instead of 5, and the sums' order is fixed.
//
// Probabilities and ds are rounded to the inputs' type for the products that follow
// them: a result has up to 1.5 times the error of its own rounding.  dq of rows of few
// keys (one tile of them, 64 or where waves share rows 128), which hold much of its norm,
// also takes what that rounding leaves.
//
// What bounds it.  2 x 4,096 tokens of 32 + 8 heads of 128 in bf16: 304 us forward (904
// TFLOP/s), 398 for dq (1,036, of its three products), 804 for dk and dv (684, four
// products).  The matrix cores are busy for 34 to 46 % of the cycles; a wave waits for
// its own chain of products, exponentials and products for the rest, of which two
// waves a SIMD, as many as the registers hold, hide a part.  An operand read from LDS
// feeds one product, so that LDS would bound the matrix cores next.  Few tokens
// over a cache are bound by memory: 64 caches of 2,048 to 4,096 tokens 172 us (4.85 TB/s).
//
// fp32: 2 x 4,096 tokens as above 2,536 us forward (108 TFLOP/s of a library product's
// 154) and 8,430 backward (114); heads of 128, dq of 96 and dk and dv of 64 too, have
// one wave a SIMD.  A token over 64 caches of 4,096 of them takes 1,310 us (1.6 TB/s): its
// four rows are one wave's, whose 128 products of 32 x 32 x 2 a tile of 32 keys, 64
// cycles each, are 870 us in two turns of one work-group a CU.
#include "ops_common.h"

namespace mgopt {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;  // rows (queries x group), or keys, of a work-group: 32 a wave
constexpr int kShared = 32; // rows of one whose waves share them, and the keys out among them
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Eight elements of a lane along the contraction: k = 16 c + 8 (lane/32) + 0..7 of chunk c.
template <typename T>
using Frag = T __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mma(Frag<__bf16> a, Frag<__bf16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(Frag<_Float16> a, Frag<_Float16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(Frag<float> a, Frag<float> b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// Probabilities in fp16 are kept times 2^15 (at most 2^15): those of long rows would be subnormal.
template <typename T>
constexpr float kShift = std::is_same_v<T, _Float16> ? 15.0f : 0.0f;

// A tile of rows of DP elements in LDS, kPitch elements apart: a lane's place plus a constant is every address, and
// neither 8 rows' reads of a chunk (16 bytes) nor 4 rows' transposed reads of two fall on a bank twice: the
// pitch is 3, 7, 9 or 13 chunks more than a multiple of 16 (4-byte types: an odd number).
template <typename T, int DP>
struct Tile {
    static constexpr int kPer = 16 / sizeof(T);          // elements of a chunk
    static constexpr int kChunks = DP / kPer;            // of a row
    static constexpr int kPitch = (sizeof(T) == 4 ? kChunks + 1 : kChunks == 4 ? 7 : kChunks == 16 ? 19 : kChunks + 1) * kPer;
    static __device__ __forceinline__ int at(int r, int chunk) { return r * kPitch + chunk * kPer; }

    // chunk c of row r of the A operand
    static __device__ __forceinline__ Frag<T> rows(const T* lds, int r, int c, int h) {
        if constexpr (sizeof(T) == 2) {
            return *reinterpret_cast<const Frag<T>*>(lds + at(r, 2 * c + h));
        } else {
            typedef T four __attribute__((ext_vector_type(4)));
            const four x = *reinterpret_cast<const four*>(lds + at(r, 4 * c + 2 * h));
            const four y = *reinterpret_cast<const four*>(lds + at(r, 4 * c + 2 * h + 1));
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    // Transposed: row 32 db + lane%32 of the A operand, its contraction over the tile's rows 16 c .. 16 c + 15 in
    // the order of the C layout: element e is row 16 c + 8 (e/4) + 4 h + e%4.
    static __device__ __forceinline__ Frag<T> columns(const T* lds, int db, int c, int lane) {
        const int h = lane / 32;
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            // of 16 lanes, lane i names 4 elements of row i/4 and takes column i of the 4 rows
            const int d = 32 * db + 16 * (lane / 16 % 2) + 4 * (lane % 4);
            s16x4 part[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 16 * c + 8 * j + 4 * h + lane % 16 / 4;
                part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4*)(lds + at(r, d / kPer) + d % kPer));
            }
            f = __builtin_bit_cast(Frag<T>, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int d = 32 * db + lane % 32;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = lds[at(16 * c + 8 * (e / 4) + 4 * h + e % 4, d / kPer) + d % kPer];
        }
        return f;
    }
};

// N elements from p, those from n on 0.
template <typename T, int N>
__device__ __forceinline__ vec_t<T, N> load_part(const T* p, int n) {
    if (n >= N) return *reinterpret_cast<const vec_t<T, N>*>(p);
    vec_t<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? p[i] : static_cast<T>(0.0f);
    return v;
}

// A value that all lanes hold alike, in a scalar register.
__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const uint32_t low = static_cast<uint32_t>(uniform(static_cast<int32_t>(x)));
    return static_cast<int64_t>(uniform(static_cast<int32_t>(x >> 32))) << 32 | low;
}

// A tile's way from memory to LDS.  Rows whose chunks are aligned to 16 bytes go there without passing through
// registers: a wave's load puts its 64 chunks behind each other in LDS, those between a row's end and the
// pitch as well.  Chunks behind `dim` are copies of the row's first: the operand that meets them is 0 there.
template <typename T, int DP, int ROWS>
struct Stage {
    using L = Tile<T, DP>;
    static constexpr int kRowChunks = L::kPitch / L::kPer;
    static constexpr int kLoads = (ROWS * kRowChunks + 63) / 64, kEach = (kLoads + kThreads / 64 - 1) / (kThreads / 64);
    static constexpr int kSize = kLoads * 64 * L::kPer;  // elements of LDS
    uint32_t off[kEach];

    static __device__ __forceinline__ void load(T* lds, int i, const T* base, uint32_t bytes) {
        const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) T*)lds)) + i * 1024;
        // not counted by the compiler: landed() waits for it
        asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(bytes), "s"(base) : "memory", "m0");
    }
    static __device__ __forceinline__ uint32_t chunk_bytes(int v, int dim) {
        const int c = v % kRowChunks;
        return c * L::kPer < dim ? c * 16 : 0;
    }
    // For whole(): row r of a tile lies at r / group * stride + r % group * inner from its base.
    __device__ __forceinline__ void plan(int wave, uint32_t group, int64_t stride, int64_t inner, int dim) {
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
            const int v = (x * (kThreads / 64) + wave) * 64 + static_cast<int>(threadIdx.x % 64);
            const uint32_t r = min(v / kRowChunks, ROWS - 1), i = r / group;
            off[x] = (i * static_cast<uint32_t>(stride) + (r - i * group) * static_cast<uint32_t>(inner)) * static_cast<uint32_t>(sizeof(T)) +
                     chunk_bytes(v, dim);
        }
    }
    __device__ __forceinline__ void whole(T* lds, int wave, const T* base) const {
#pragma unroll
        for (int x = 0; x < kEach; ++x)
            if (const int i = x * (kThreads / 64) + wave; i < kLoads) load(lds, i, base, off[x]);
    }
    // `rows` rows (one at least) of one stride; the last one stands for those behind it.
    __device__ __forceinline__ void some(T* lds, int wave, const T* base, int64_t stride, int rows, int dim) const {
#pragma unroll
        for (int x = 0; x < kEach; ++x)
            if (const int i = x * (kThreads / 64) + wave; i < kLoads) {
                const int v = i * 64 + static_cast<int>(threadIdx.x % 64);
                const uint32_t row = min(v / kRowChunks, min(rows, ROWS) - 1);
                load(lds, i, base, row * static_cast<uint32_t>(stride) * static_cast<uint32_t>(sizeof(T)) + chunk_bytes(v, dim));
            }
    }
    // Rows anywhere; at(r): where row r lies.
    template <typename F>
    static __device__ __forceinline__ void scattered(T* lds, int wave, int dim, F&& at) {
        int lane = threadIdx.x % 64;
        asm volatile("" : "+v"(lane));  // nothing of this way is worth a register between the tiles
#pragma unroll 1
        for (int x = 0; x < kEach; ++x)
            if (const int i = x * (kThreads / 64) + wave; i < kLoads) {
                const int v = i * 64 + lane;
                const char* from = reinterpret_cast<const char*>(at(min(v / kRowChunks, ROWS - 1))) + chunk_bytes(v, dim);
                const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) T*)lds)) + i * 1024;
                asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
            }
    }
    // The same through registers, for rows of any alignment.
    template <typename F>
    static __device__ __forceinline__ void copy(T* lds, int dim, F&& at) {
        typedef T chunk_t __attribute__((ext_vector_type(L::kPer)));
        int v = threadIdx.x;
        asm volatile("" : "+v"(v));
        for (; v < ROWS * L::kChunks; v += kThreads) {
            const int r = v / L::kChunks, c = v % L::kChunks;
            *reinterpret_cast<chunk_t*>(lds + L::at(r, c)) = load_part<T, L::kPer>(at(r) + c * L::kPer, dim - c * L::kPer);
        }
    }
    __device__ __forceinline__ void fetch(T* lds, int wave, bool aligned, const T* base, int64_t stride, int rows, int dim) const {
        if (!aligned) copy(lds, dim, [&](int r) { return base + min(r, rows - 1) * stride; });
        else if (rows >= ROWS) whole(lds, wave, base);
        else some(lds, wave, base, stride, rows, dim);
    }
};
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// 4 bytes from each lane's address to LDS, 256 bytes a wave.
__device__ __forceinline__ void load_word(void* lds, const void* at) {
    const uint32_t to = uniform(static_cast<int32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds)));
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(at) : "memory", "m0");
}

struct AttArgs {
    mgopt_attention_args a;
    uint32_t group;      // query heads of a key head
    uint32_t magic, shift;  // x / group = (x * magic >> 32) >> shift for x < 2^31, but for a group of 1
    uint32_t tiles;      // of a batch's row (padded batches)
    uint32_t splits;
    float scale2;        // scale * log2(e)
    bool aligned_keys;   // keys' and values' chunks are aligned to 16 bytes
    bool aligned_rows;   // queries' and gradients' too
    bool even_rows;      // and their tiles have (query, head) alike, and 32 bits reach over them
    float* stats;        // backward: [2][batch][q_heads][queries], lse * log2(e) - kShift (inf: sees no key), and delta
    float* part_out;     // [splits][rows][dim]
    float* part_ml;      // [splits][rows][2]
};

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t low, int64_t high) { return x < low ? low : x > high ? high : x; }

// The sequence of a work-group, and its tile's first row in it.
struct Part {
    int64_t batch;       // its row of the batch
    int64_t q0, k0;      // its first query and key there
    int32_t n, m;        // its queries and keys
    int32_t total;       // queries (keys) of its place in memory: those from n (m) on are padding
    int64_t first;       // of the tile, in rows
};

// Tile `slot` of the queries (`per` rows each), or of the keys with KEYS.  Packed sequences, with what lies before the
// first and behind the last as two more that hold nothing, have places of their own for floor(rows / TILE) + 1
// tiles each; `first` is beyond `total` where a place stays empty.  Offsets are clamped to the tokens.
template <bool KEYS, int TILE>
__device__ Part find_part(const AttArgs& p, uint32_t slot, uint32_t per) {
    const mgopt_attention_args& a = p.a;
    Part s{};
    const int64_t tokens = KEYS ? a.keys : a.queries;
    if (a.q_offsets_dev == nullptr) {
        s.batch = slot / p.tiles;
        s.first = static_cast<int64_t>(slot % p.tiles) * TILE;
        s.total = static_cast<int32_t>(tokens);
        s.n = static_cast<int32_t>(a.q_lengths_dev ? clamp64(id_at(a.q_lengths_dev, s.batch, a.offset_bytes), 0, a.queries) : a.queries);
        s.m = static_cast<int32_t>(a.k_lengths_dev ? clamp64(id_at(a.k_lengths_dev, s.batch, a.offset_bytes), 0, a.keys) : a.keys);
        return s;
    }
    const void* offsets = KEYS ? a.k_offsets_dev : a.q_offsets_dev;
    const int32_t count = static_cast<int32_t>(a.sequences) + 2;
    const auto edge = [&](int32_t j) {
        return j <= 0 ? 0 : j >= count ? tokens : clamp64(id_at(offsets, j - 1, a.offset_bytes), 0, tokens);
    };
    const auto base = [&](int32_t j) { return edge(j) * per / TILE + j; };
    // the last part whose places begin at `slot` or before, 64 of them looked at at once
    int32_t low = 0, left = count;
    while (left > 1) {
        const int32_t step = (left + 63) / 64, at = low + static_cast<int32_t>(threadIdx.x % 64) * step;
        const uint64_t hit = __ballot(at < low + left && base(at) <= static_cast<int64_t>(slot));
        const int32_t k = max(1, __popcll(hit)) - 1;
        left = min(step, left - k * step);
        low += k * step;
    }
    const int64_t from = edge(low), to = edge(low + 1);
    s.first = (static_cast<int64_t>(slot) - base(low)) * TILE;
    s.total = static_cast<int32_t>(to > from ? to - from : 0);
    if (s.first < 0) s.first = 0, s.total = 0;
    s.q0 = s.k0 = from;
    if (low >= 1 && low + 1 < count) {
        const void* others = KEYS ? a.q_offsets_dev : a.k_offsets_dev;
        const int64_t all = KEYS ? a.queries : a.keys;
        const int64_t x = clamp64(id_at(others, low - 1, a.offset_bytes), 0, all), y = clamp64(id_at(others, low, a.offset_bytes), 0, all);
        const int32_t len = static_cast<int32_t>(y > x ? y - x : 0);
        (KEYS ? s.q0 : s.k0) = x;
        s.n = KEYS ? len : s.total, s.m = KEYS ? s.total : len;
    }
    return s;
}

template <bool KEYS, int TILE = kTile>
__device__ __forceinline__ Part find(const AttArgs& p, uint32_t slot, uint32_t per) {
    const Part s = find_part<KEYS, TILE>(p, slot, per);
    return {uniform(s.batch), uniform(s.q0), uniform(s.k0), uniform(s.n), uniform(s.m), uniform(s.total), uniform(s.first)};
}

// How many keys, from the first, query i of the sequence sees.
__device__ __forceinline__ int32_t seen(const AttArgs& p, const Part& s, int32_t i) {
    if (i >= s.n) return 0;
    return p.a.causal ? max(0, min(s.m, (i + 1 - s.n) + s.m)) : s.m;
}

// f of a lane and of the lane 32 away.
template <typename Op>
__device__ __forceinline__ float with_partner(float x, Op op) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }

// One row's elements as the B operand: chunk c's 8 elements of this half of the wave.
template <typename T, int DP>
__device__ __forceinline__ void load_row(Frag<T> (&f)[DP / 16], const T* row, int dim, int h) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
        f[c] = Frag<T>{};
        if (row != nullptr) {
            const int d = 16 * c + 8 * h;
            const vec_t<T, 8> v = load_part<T, 8>(row + d, dim - d);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[c][e] = v[e];
        }
    }
}

// Chunk c (of two) of a block of scores as the B operand.
template <typename T>
__device__ __forceinline__ Frag<T> as_operand(const f32x16& s, int c) {
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<T>(s[8 * c + e]);
    return f;
}

// A column of the accumulators (rows are the elements of a head) times `by`.
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DP / 32], float by, int dim, int h) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int d = 32 * b + 8 * q + 4 * h;
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = acc[b][4 * q + e] * by;
            store_some<4>(row + d, f, dim - d);
        }
}

// Row r's place: query r / group, head r % group of the group.
struct Place {
    int32_t query, head;
};
__device__ __forceinline__ Place place_of(const AttArgs& p, int64_t r) {
    const uint32_t x = static_cast<uint32_t>(r), i = p.group == 1 ? x : __umulhi(x, p.magic) >> p.shift;
    return {static_cast<int32_t>(i), static_cast<int32_t>(x - i * p.group)};
}

template <typename T>
__device__ __forceinline__ T* row_of(const void* base, const int64_t (&stride)[3], int64_t batch, int64_t token, int64_t head) {
    return const_cast<T*>(static_cast<const T*>(base)) + batch * stride[0] + token * stride[1] + head * stride[2];
}

// Which (slot, key head) a work-group has: key heads next to each other, so that with 8 of them each XCD keeps
// the keys and values of one; with last_first, for causal batches' queries, the last tiles, which see most keys, first.
struct Unit {
    uint32_t slot, head;
};
__device__ __forceinline__ Unit unit_of(const AttArgs& p, bool last_first) {
    const uint32_t heads = static_cast<uint32_t>(p.a.k_heads);
    uint32_t place = blockIdx.x;
    if (p.tiles == 1 && gridDim.x % 8 == 0) place = place % 8 * (gridDim.x / 8) + place / 8;
    uint32_t slot = place / heads;
    const uint32_t head = place - slot * heads;
    if (p.a.q_offsets_dev != nullptr && last_first) slot = gridDim.x / heads - 1 - slot;
    if (p.a.q_offsets_dev == nullptr) {
        // tiles outermost, the batch's rows within
        const uint32_t rows = static_cast<uint32_t>(p.a.batch);
        uint32_t t = slot / rows;
        const uint32_t b = slot - t * rows;
        if (last_first) t = p.tiles - 1 - t;
        slot = b * p.tiles + t;
    }
    return {slot, head};
}

// What any of `rows` rows from r on sees at most; later queries see no fewer keys than earlier ones.
__device__ __forceinline__ int32_t most_seen(const AttArgs& p, const Part& s, int64_t r, int rows) {
    return place_of(p, r).query < s.n ? seen(p, s, min(place_of(p, r + rows - 1).query, s.n - 1)) : 0;
}

// ------------------------------------------------------------------- forward

template <typename T, int DP>
constexpr int kKeys = sizeof(T) == 4 ? 32 : 64;  // keys of a tile in LDS
template <typename T, int DP>
constexpr int kMinWaves = sizeof(T) == 4 ? 1 : 2;  // a SIMD

// Where the sums of the waves that share rows or keys meet, a column's elements behind each other, and the thread's
// part of them in the join: row r, EACH elements from d0 on.
template <int DP>
struct Join {
    static constexpr int kPitch = DP + 4, kEach = DP / 8, kBytes = 4 * 32 * kPitch * 4;
    float (*sums)[32][kPitch];
    int r = threadIdx.x / 8, d0 = threadIdx.x % 8 * kEach;
    __device__ __forceinline__ explicit Join(void* lds) : sums(static_cast<float (*)[32][kPitch]>(lds)) {}
    __device__ __forceinline__ void put(int wave, int col, const f32x16 (&acc)[DP / 32], float by, int h) {
        store_row<float, DP>(sums[wave][col], acc, by, DP, h);
    }
    // y += by * wave w's elements
    __device__ __forceinline__ void get(float (&y)[kEach], int w, float by) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e) y[e] = fmaf(by, sums[w][r][d0 + e], y[e]);
    }
};

// SPLIT: a work-group takes one of `splits` parts of the keys and leaves its sums for join_kernel.  SHARED: its waves
// take the same 32 rows and a quarter of each 128 keys, and join their sums in LDS, for rows so few that 128 of them
// fill no work-group, or the work-groups do not fill the chip: 8 x 128 tokens of 4 heads of 32 in fp32 6.1 us, 10.8 with
// rows of its own for each wave; 2,048 tokens of 8 heads of 64 in fp16 21 and 39; but 8 x 1,024 of 12 heads 54 and 30.
template <typename T, int DP, bool SPLIT, bool SHARED>
__global__ __launch_bounds__(kThreads, (kMinWaves<T, DP>)) void attention_kernel(AttArgs p) {
    constexpr int TILE = SHARED ? kShared : kTile, BN = SHARED ? 128 : kKeys<T, DP>, BLOCKS = SHARED ? 1 : BN / 32;
    using L = Tile<T, DP>;
    using Keys = Stage<T, DP, BN>;
    // two work-groups a CU where their tiles leave room for it
    constexpr int BUFFERS = SHARED && Keys::kSize * sizeof(T) > 20 * 1024 ? 1 : 2;
    __shared__ alignas(16) T tiles[2][BUFFERS][Keys::kSize];
    const mgopt_attention_args& a = p.a;
    const Unit u = unit_of(p, a.causal);
    const Part s = find<false, TILE>(p, u.slot, p.group);
    if (s.first >= static_cast<int64_t>(s.total) * p.group) return;
    const int lane = threadIdx.x % 64, wave = uniform(static_cast<int32_t>(threadIdx.x / 64)), col = lane % 32, h = lane / 32;
    const int64_t first = SHARED ? s.first : s.first + wave * 32;  // of the wave's rows
    const int block0 = SHARED ? wave : 0;                          // of its keys in a tile
    const Place at = place_of(p, first + col);
    const int64_t head = static_cast<int64_t>(u.head) * p.group + at.head;
    const bool inside = at.query < s.total;
    const int32_t mine = seen(p, s, at.query);
    Frag<T> q[DP / 16];
    load_row<T, DP>(q, mine > 0 ? row_of<T>(a.q_dev, a.q_stride, s.batch, s.q0 + at.query, head) : nullptr, a.dim, h);
    // what the work-group's rows, and the wave's, see at most, and the wave's at least
    const int32_t most = most_seen(p, s, s.first, TILE);
    const int32_t wave_most = most_seen(p, s, first, 32);
    const int32_t wave_least = seen(p, s, place_of(p, first).query);
    int32_t from = 0, to = most;
    if constexpr (SPLIT) {
        const int32_t share = (most + BN * static_cast<int32_t>(p.splits) - 1) / (BN * static_cast<int32_t>(p.splits)) * BN;
        from = static_cast<int32_t>(min(static_cast<int64_t>(blockIdx.y) * share, static_cast<int64_t>(most)));
        to = min(from + share, most);
    }
    Keys stage_k, stage_v;
    const T* const kp = row_of<T>(a.k_dev, a.k_stride, s.batch, s.k0, u.head);
    const T* const vp = row_of<T>(a.v_dev, a.v_stride, s.batch, s.k0, u.head);
    stage_k.plan(wave, 1, a.k_stride[1], 0, a.dim), stage_v.plan(wave, 1, a.v_stride[1], 0, a.dim);
    const auto fetch = [&](int32_t k0, int buf) {
        stage_k.fetch(tiles[0][buf], wave, p.aligned_keys, kp + k0 * a.k_stride[1], a.k_stride[1], to - k0, a.dim);
        stage_v.fetch(tiles[1][buf], wave, p.aligned_keys, vp + k0 * a.v_stride[1], a.v_stride[1], to - k0, a.dim);
    };
    f32x16 o[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) o[b] = f32x16{};
    float top = -INFINITY, sum = 0.0f;
    if (from < to) fetch(from, 0);
    landed();
    __syncthreads();
    int buf = 0;
    for (int32_t k0 = from; k0 < to; k0 += BN) {
        if (BUFFERS == 2 && k0 + BN < to) fetch(k0 + BN, buf ^ 1);
        const T *const keys = tiles[0][buf], *const values = tiles[1][buf];
        if (k0 + 32 * block0 < wave_most) {
            f32x16 x[BLOCKS];
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) x[b] = f32x16{};
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) x[b] = mma(L::rows(keys, 32 * (block0 + b) + col, c, h), q[c], x[b]);
            if (k0 + 32 * (block0 + BLOCKS) > min(wave_least, to)) {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (k0 + 32 * (block0 + b) + 8 * (e / 4) + 4 * h + e % 4 >= min(mine, to)) x[b][e] = -INFINITY;
            }
            float big = x[0][0];
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) big = fmaxf(big, x[b][e]);
            big = with_partner(big, [](float y, float z) { return fmaxf(y, z); });
            const float next = fmaxf(top, big);
            const float ref = next == -INFINITY ? 0.0f : next;
            if (__any(next > top)) {
                const float alpha = exp2_hw((top - ref) * p.scale2);
                sum *= alpha;
#pragma unroll
                for (int b = 0; b < DP / 32; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[b][e] *= alpha;
                top = next;
            }
            const float off = fmaf(ref, p.scale2, -kShift<T>);
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    x[b][e] = exp2_hw(fmaf(x[b][e], p.scale2, -off));
                    sum += x[b][e];
                }
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> w = as_operand<T>(x[b], c);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) o[d] = mma(L::columns(values, d, 2 * (block0 + b) + c, lane), w, o[d]);
                }
        }
        if constexpr (BUFFERS == 2) {
            buf ^= 1;
        } else {
            __syncthreads();
            if (k0 + BN < to) fetch(k0 + BN, 0);
        }
        landed();
        __syncthreads();
    }
    sum = with_partner(sum, add);
    // a score beyond 32 bits took all others' probabilities, and its own, to 0: what inf - inf is, and not a row without keys
    if (top * p.scale2 == INFINITY) sum = NAN;
    if (mine == 0) {  // padding, or no key to see: what its column holds is of a query of zeros without a mask
        top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) o[b] = f32x16{};
    }
    const int64_t rows = a.batch * a.queries * a.q_heads;  // of parts: in the order (batch, query, head)
    const auto part = [&](const Place& x) {
        return blockIdx.y * rows + (s.batch * a.queries + s.q0 + x.query) * a.q_heads + static_cast<int64_t>(u.head) * p.group + x.head;
    };
    const auto write_lse = [&](const Place& x, float m, float l) {
        if (a.lse_dev != nullptr)
            a.lse_dev[(s.batch * a.q_heads + static_cast<int64_t>(u.head) * p.group + x.head) * a.queries + s.q0 + x.query] =
                l == 0.0f ? -INFINITY : static_cast<float>(kLn2) * (m * p.scale2 - kShift<T> + log2f(l));
    };
    if constexpr (SHARED) {
        constexpr int EACH = Join<DP>::kEach;
        static_assert(sizeof(tiles) >= Join<DP>::kBytes);
        __shared__ float stats[2][4][32];
        Join<DP> join(&tiles[0][0][0]);
        join.put(wave, col, o, 1.0f, h);
        if (h == 0) stats[0][wave][col] = top, stats[1][wave][col] = sum;
        __syncthreads();
        const int r = join.r, d0 = join.d0;
        const Place x = place_of(p, first + r);
        if (x.query >= s.total) return;
        const float m = fmaxf(fmaxf(stats[0][0][r], stats[0][1][r]), fmaxf(stats[0][2][r], stats[0][3][r]));
        float l = 0.0f, y[EACH] = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float by = exp2_hw((stats[0][w][r] - (m == -INFINITY ? 0.0f : m)) * p.scale2);
            l = fmaf(by, stats[1][w][r], l);
            join.get(y, w, by);
        }
        if constexpr (SPLIT) {
            store_some<EACH>(p.part_out + part(x) * a.dim + d0, y, a.dim - d0);
            if (d0 == 0) p.part_ml[2 * part(x)] = m, p.part_ml[2 * part(x) + 1] = l;
        } else {
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < EACH; ++e) y[e] *= by;
            store_some<EACH>(row_of<T>(a.out_dev, a.out_stride, s.batch, s.q0 + x.query, static_cast<int64_t>(u.head) * p.group + x.head) + d0, y,
                             a.dim - d0);
            if (d0 == 0) write_lse(x, m, l);
        }
    } else {
        if (!inside) return;
        if constexpr (SPLIT) {
            store_row<float, DP>(p.part_out + part(at) * a.dim, o, 1.0f, a.dim, h);
            if (h == 0) p.part_ml[2 * part(at)] = top, p.part_ml[2 * part(at) + 1] = sum;
        } else {
            T* const out = row_of<T>(a.out_dev, a.out_stride, s.batch, s.q0 + at.query, head);
            store_row<T, DP>(out, o, sum == 0.0f ? 0.0f : 1.0f / sum, a.dim, h);
            if (h == 0) write_lse(at, top, sum);
        }
    }
}

// Joins the parts of a row, which a work-group's waves share.
constexpr uint32_t kMostSplits = kThreads;
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(AttArgs p) {
    __shared__ float weight[kMostSplits], tops[kThreads / 64], sums[kThreads / 64], part[kThreads / 64][128];
    const mgopt_attention_args& a = p.a;
    const int64_t rows = a.batch * a.queries * a.q_heads, row = blockIdx.x;
    const int64_t head = row % a.q_heads, t = row / a.q_heads, query = t % a.queries, batch = t / a.queries;
    const uint32_t i = threadIdx.x, wave = i / 64, lane = i % 64;
    const bool mine = i < p.splits;
    float top = mine ? p.part_ml[2 * (i * rows + row)] : -INFINITY;
    const float kept = top, len = mine ? p.part_ml[2 * (i * rows + row) + 1] : 0.0f;
    top = reduce_lanes<64>(top, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float w = exp2_hw((kept - (top == -INFINITY ? 0.0f : top)) * p.scale2);
    if (mine) weight[i] = w;
    float sum = reduce_lanes<64>(w * len, add);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    float acc[2] = {};  // elements lane and lane + 64
#pragma unroll 8
    for (uint32_t k = wave; k < p.splits; k += kThreads / 64) {
        const float* o = p.part_out + (k * rows + row) * a.dim;
        const float by = weight[k];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int d = lane + 64 * j;
            if (d < a.dim) acc[j] = fmaf(by, o[d], acc[j]);
        }
    }
    part[wave][lane] = acc[0], part[wave][lane + 64] = acc[1];
    __syncthreads();
    const int d = threadIdx.x;
    if (d < a.dim) {
        const float x = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
        row_of<T>(a.out_dev, a.out_stride, batch, query, head)[d] = static_cast<T>(x * (sum == 0.0f ? 0.0f : 1.0f / sum));
    }
    if (threadIdx.x == 0 && a.lse_dev != nullptr)
        a.lse_dev[(batch * a.q_heads + head) * a.queries + query] =
            sum == 0.0f ? -INFINITY : static_cast<float>(kLn2) * (top * p.scale2 - kShift<T> + log2f(sum));
}

// ------------------------------------------------------------------ backward

// The score gradients of fp16 heads are rounded to fp16 times a power of two of each column's own, lowered
// with the accumulators when a value would pass 2^15: without it those of long rows, a probability times a
// small gradient, are subnormal or 0.
template <typename T>
struct Range {
    template <int B>
    __device__ __forceinline__ void fit(f32x16&, f32x16 (&)[B]) {}
    __device__ __forceinline__ float back() const { return 1.0f; }
};
template <>
struct Range<_Float16> {
    float by = 0x1p100f;
    template <int B>
    __device__ __forceinline__ void fit(f32x16& ds, f32x16 (&acc)[B]) {
        float big = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) big = fmaxf(big, fabsf(ds[e]));
        big = with_partner(big, [](float y, float z) { return fmaxf(y, z); });
        if (__any(big * by > 32768.0f)) {
            // the power of two that takes big to [2^13, 2^14); an inf or a NaN is not fitted
            const bool lower = big * by > 32768.0f && big < INFINITY;
            const float next = lower ? __uint_as_float((267u - (__float_as_uint(big) >> 23)) << 23) : by;
            const float change = next / by;
            by = next;
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[b][e] *= change;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[e] *= by;
    }
    __device__ __forceinline__ float back() const { return 1.0f / by; }
};

// dq, and delta for the kernel that follows.  SHARED: as in the forward pass.
template <typename T, int DP, bool SHARED>
__global__ __launch_bounds__(kThreads, (kMinWaves<T, DP>)) void attention_dq_kernel(AttArgs p) {
    constexpr int TILE = SHARED ? kShared : kTile, BN = SHARED ? 128 : kKeys<T, DP>, BLOCKS = SHARED ? 1 : BN / 32;
    using L = Tile<T, DP>;
    using Keys = Stage<T, DP, BN>;
    constexpr int BUFFERS = SHARED && Keys::kSize * sizeof(T) > 20 * 1024 ? 1 : 2;
    __shared__ alignas(16) T tiles[2][BUFFERS][Keys::kSize];
    __shared__ float deltas[SHARED ? 4 : 1][32];
    const mgopt_attention_args& a = p.a;
    const Unit u = unit_of(p, a.causal);
    const Part s = find<false, TILE>(p, u.slot, p.group);
    if (s.first >= static_cast<int64_t>(s.total) * p.group) return;
    const int lane = threadIdx.x % 64, wave = uniform(static_cast<int32_t>(threadIdx.x / 64)), col = lane % 32, h = lane / 32;
    const int64_t first = SHARED ? s.first : s.first + wave * 32;  // of the wave's rows
    const int block0 = SHARED ? wave : 0;                          // of its keys in a tile
    const Place at = place_of(p, first + col);
    const int64_t head = static_cast<int64_t>(u.head) * p.group + at.head;
    const bool inside = at.query < s.total;
    const int32_t mine = seen(p, s, at.query);
    Frag<T> q[DP / 16], g[DP / 16];
    load_row<T, DP>(q, mine > 0 ? row_of<T>(a.q_dev, a.q_stride, s.batch, s.q0 + at.query, head) : nullptr, a.dim, h);
    load_row<T, DP>(g, mine > 0 ? row_of<T>(a.grad_out_dev, a.grad_out_stride, s.batch, s.q0 + at.query, head) : nullptr, a.dim, h);
    const int32_t to = most_seen(p, s, s.first, TILE);
    const int32_t wave_most = most_seen(p, s, first, 32);
    const int32_t wave_least = seen(p, s, place_of(p, first).query);
    const int64_t stat = (s.batch * a.q_heads + head) * a.queries + s.q0 + at.query;
    // Rows whose keys are one tile take delta from it, as sum_j p_ij g_i . v_j: of few keys, what is left of
    // g_i . v_j - delta_i can be less than the rounding of out.
    const bool one_tile = wave_most <= BN;
    float delta = 0.0f, lse = mine > 0 ? a.lse_dev[stat] * static_cast<float>(kLog2e) : INFINITY;
    if (!one_tile) {
        Frag<T> o[DP / 16];
        load_row<T, DP>(o, mine > 0 ? row_of<T>(a.out_dev, a.out_stride, s.batch, s.q0 + at.query, head) : nullptr, a.dim, h);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(static_cast<float>(g[c][e]), static_cast<float>(o[c][e]), delta);
        delta = with_partner(delta, add);
    }
    Keys stage_k, stage_v;
    const T* const kp = row_of<T>(a.k_dev, a.k_stride, s.batch, s.k0, u.head);
    const T* const vp = row_of<T>(a.v_dev, a.v_stride, s.batch, s.k0, u.head);
    stage_k.plan(wave, 1, a.k_stride[1], 0, a.dim), stage_v.plan(wave, 1, a.v_stride[1], 0, a.dim);
    const auto fetch = [&](int32_t k0, int buf) {
        stage_k.fetch(tiles[0][buf], wave, p.aligned_keys, kp + k0 * a.k_stride[1], a.k_stride[1], to - k0, a.dim);
        stage_v.fetch(tiles[1][buf], wave, p.aligned_keys, vp + k0 * a.v_stride[1], a.v_stride[1], to - k0, a.dim);
    };
    int buf = 0;
    // p_ij and g_i . v_j of block b of the keys from k0 on
    const auto scores = [&](int b, f32x16& x, f32x16& dp) {
        x = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            x = mma(L::rows(tiles[0][buf], 32 * b + col, c, h), q[c], x);
            dp = mma(L::rows(tiles[1][buf], 32 * b + col, c, h), g[c], dp);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = exp2_hw(fmaf(x[e], p.scale2, -lse));
    };
    const auto hide = [&](int32_t k, f32x16& x, f32x16& dp) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool out = k + 8 * (e / 4) + 4 * h + e % 4 >= mine;
            x[e] = out ? 0.0f : x[e], dp[e] = out ? 0.0f : dp[e];
        }
    };
    f32x16 acc[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) acc[b] = f32x16{};
    Range<T> range;
    if (to > 0) fetch(0, 0);
    landed();
    __syncthreads();
    if (one_tile) {
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
            if (32 * (block0 + b) < wave_most) {
                f32x16 x, dp;
                scores(block0 + b, x, dp);
                hide(32 * (block0 + b), x, dp);
#pragma unroll
                for (int e = 0; e < 16; ++e) delta = fmaf(x[e], dp[e], delta);
            }
        delta = with_partner(delta, add);
        if constexpr (SHARED) {  // wave_most is the work-group's: all waves are here
            if (h == 0) deltas[wave][col] = delta;
            __syncthreads();
            delta = (deltas[0][col] + deltas[1][col]) + (deltas[2][col] + deltas[3][col]);
        }
    }
    for (int32_t k0 = 0; k0 < to; k0 += BN) {
        if (BUFFERS == 2 && k0 + BN < to) fetch(k0 + BN, buf ^ 1);
        if (k0 + 32 * block0 < wave_most) {
            const bool edge = k0 + 32 * (block0 + BLOCKS) > wave_least;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                f32x16 x, ds;
                scores(block0 + b, x, ds);
                if (edge) hide(k0 + 32 * (block0 + b), x, ds);
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] = x[e] * (ds[e] - delta);
                range.fit(ds, acc);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> w = as_operand<T>(ds, c);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) acc[d] = mma(L::columns(tiles[0][buf], d, 2 * (block0 + b) + c, lane), w, acc[d]);
                    // and what the rounding left, where keys are few and dq large: 4,608 causal rows of 8 heads of 32 in fp16
                    // are off by 3.0e-4 of dq's norm, without it by 3.2e-4; 22 sequences of 48 to 1,417 56 us, 54
                    if constexpr (sizeof(T) < 4) {
                        if (one_tile) {
                            Frag<T> rest;
#pragma unroll
                            for (int e = 0; e < 8; ++e) rest[e] = static_cast<T>(ds[8 * c + e] - static_cast<float>(w[e]));
#pragma unroll
                            for (int d = 0; d < DP / 32; ++d)
                                acc[d] = mma(L::columns(tiles[0][buf], d, 2 * (block0 + b) + c, lane), rest, acc[d]);
                        }
                    }
                }
            }
        }
        if constexpr (BUFFERS == 2) {
            buf ^= 1;
        } else {
            __syncthreads();
            if (k0 + BN < to) fetch(k0 + BN, 0);
        }
        landed();
        __syncthreads();
    }
    if (inside && h == 0 && (!SHARED || wave == 0))
        p.stats[stat] = lse - kShift<T>, p.stats[a.batch * a.q_heads * a.queries + stat] = mine > 0 ? delta : 0.0f;
    if (mine == 0) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) acc[b] = f32x16{};
    }
    const float by = static_cast<float>(a.scale) * range.back();
    if constexpr (SHARED) {
        static_assert(sizeof(tiles) >= Join<DP>::kBytes);
        Join<DP> join(&tiles[0][0][0]);
        join.put(wave, col, acc, by, h);
        __syncthreads();
        const Place x = place_of(p, first + join.r);
        if (x.query >= s.total) return;
        float y[Join<DP>::kEach] = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) join.get(y, w, 1.0f);
        store_some<Join<DP>::kEach>(
            row_of<T>(a.d_q_dev, a.d_q_stride, s.batch, s.q0 + x.query, static_cast<int64_t>(u.head) * p.group + x.head) + join.d0, y,
            a.dim - join.d0);
    } else if (inside) {
        store_row<T, DP>(row_of<T>(a.d_q_dev, a.d_q_stride, s.batch, s.q0 + at.query, head), acc, by, a.dim, h);
    }
}

template <typename T, int DP>
constexpr int kRows = sizeof(T) == 4 || DP > 64 ? 32 : 64;  // rows of a tile in LDS, for dk and dv

// Whether the values stay in LDS: with the keys and both sums they pass the registers of two waves a SIMD.
template <typename T, int DP>
constexpr bool kValuesInLds = sizeof(T) == 2 && DP > 64;

// dk and dv of 128 keys over all rows that see them.  SHARED: of 32 keys, and the waves take a quarter each of 128 rows at
// a time, and join their sums in LDS.
template <typename T, int DP, bool SHARED>
__global__ __launch_bounds__(kThreads, (kMinWaves<T, DP>)) void attention_dkv_kernel(AttArgs p) {
    constexpr int BM = SHARED ? 128 : kRows<T, DP>, TILE = SHARED ? kShared : kTile, BLOCKS = SHARED ? 1 : BM / 32;
    constexpr bool LDS_V = !SHARED && kValuesInLds<T, DP>;
    using L = Tile<T, DP>;
    using Rows = Stage<T, DP, BM>;
    constexpr int BUFFERS = SHARED && Rows::kSize * sizeof(T) > 20 * 1024 ? 1 : 2;
    __shared__ alignas(16) T tiles[2][BUFFERS][Rows::kSize];
    __shared__ alignas(16) T values[LDS_V ? Stage<T, DP, kTile>::kSize : 8];
    __shared__ alignas(16) float lses[BUFFERS][SHARED ? 128 : 64], deltas[BUFFERS][SHARED ? 128 : 64];
    const mgopt_attention_args& a = p.a;
    const Unit u = unit_of(p, false);
    const Part s = find<true, TILE>(p, u.slot, 1);
    if (s.first >= s.total) return;
    const int lane = threadIdx.x % 64, wave = uniform(static_cast<int32_t>(threadIdx.x / 64)), col = lane % 32, h = lane / 32;
    const int32_t tile0 = static_cast<int32_t>(s.first), key0 = tile0 + (SHARED ? 0 : wave * 32), key = key0 + col;
    const int block0 = SHARED ? wave : 0;  // of the wave's rows in a tile
    const bool live = key < s.m;
    Frag<T> k[DP / 16], v[LDS_V ? 1 : DP / 16];
    load_row<T, DP>(k, live ? row_of<T>(a.k_dev, a.k_stride, s.batch, s.k0 + key, u.head) : nullptr, a.dim, h);
    if constexpr (!LDS_V) load_row<T, DP>(v, live ? row_of<T>(a.v_dev, a.v_stride, s.batch, s.k0 + key, u.head) : nullptr, a.dim, h);
    else if (tile0 < s.m)
        Stage<T, DP, kTile>::copy(values, a.dim, [&](int r) { return row_of<T>(a.v_dev, a.v_stride, s.batch, s.k0 + min(tile0 + r, s.m - 1), u.head); });
    // the first row that sees the tile's first key
    const int32_t group = static_cast<int32_t>(p.group), rows = s.n * group;
    int32_t from = 0;
    if (a.causal) from = min(max(0, tile0 - (s.m - s.n)), s.n) * group / BM * BM;
    if (tile0 >= s.m) from = rows;
    const int32_t blind = a.causal ? max(0, s.n - s.m) * group : 0;  // rows before this one see no key, and have no gradient
    Rows stage_q, stage_g;
    const int64_t head0 = static_cast<int64_t>(u.head) * group;
    const T* const qp = row_of<T>(a.q_dev, a.q_stride, s.batch, s.q0, head0);
    const T* const gp = row_of<T>(a.grad_out_dev, a.grad_out_stride, s.batch, s.q0, head0);
    stage_q.plan(wave, p.group, a.q_stride[1], a.q_stride[2], a.dim);
    stage_g.plan(wave, p.group, a.grad_out_stride[1], a.grad_out_stride[2], a.dim);
    const float* const stats = p.stats + (s.batch * a.q_heads + head0) * a.queries + s.q0;
    const int64_t all = a.batch * a.q_heads * a.queries;
    const auto q_row = [&](const Place& x) { return qp + x.query * a.q_stride[1] + x.head * a.q_stride[2]; };
    const auto g_row = [&](const Place& x) { return gp + x.query * a.grad_out_stride[1] + x.head * a.grad_out_stride[2]; };
    // rows that are not there, or see no key, are others here: their probabilities are 0
    const auto at = [&](int32_t r) { return place_of(p, min(max(r, blind), rows - 1)); };
    const auto fetch = [&](int32_t r0, int buf) {
        if (p.even_rows && r0 + BM <= rows && r0 >= blind) {
            const int64_t first = place_of(p, r0).query;
            stage_q.whole(tiles[0][buf], wave, qp + first * a.q_stride[1]);
            stage_g.whole(tiles[1][buf], wave, gp + first * a.grad_out_stride[1]);
        } else {
            const auto q_at = [&](int r) { return q_row(at(r0 + r)); };
            const auto g_at = [&](int r) { return g_row(at(r0 + r)); };
            if (p.aligned_rows) Rows::scattered(tiles[0][buf], wave, a.dim, q_at), Rows::scattered(tiles[1][buf], wave, a.dim, g_at);
            else Rows::copy(tiles[0][buf], a.dim, q_at), Rows::copy(tiles[1][buf], a.dim, g_at);
        }
        // waves 0 and 1 (of 128 rows 0 to 3) bring 64 rows' statistics each
        if (wave < (BM > 64 ? 4 : 2)) {
            const int half = wave / 2 * 64;
            const Place x = at(r0 + min(half + lane, BM - 1));
            load_word((wave % 2 == 0 ? lses[buf] : deltas[buf]) + half, stats + (wave % 2 == 0 ? 0 : all) + x.head * a.queries + x.query);
        }
    };
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dk[b] = f32x16{}, dv[b] = f32x16{};
    Range<T> range;
    // from the last rows, which all key tiles have, to the first, so that the tiles of a head read the same rows at
    // about the same time
    const int32_t last = (rows - 1) / BM * BM;
    if (from < rows) fetch(last, 0);
    landed();
    __syncthreads();
    int buf = 0;
    for (int32_t r0 = last; r0 >= from && from < rows; r0 -= BM) {
        if (BUFFERS == 2 && r0 > from) fetch(r0 - BM, buf ^ 1);
        const T *const queries = tiles[0][buf], *const grads = tiles[1][buf];
        // the tile's rows see no fewer keys than its first and no more than its last
        const int32_t r1 = r0 + 32 * block0, r2 = r1 + 32 * BLOCKS;
        if (r1 < rows && seen(p, s, place_of(p, min(r2, rows) - 1).query) > key0) {
            const bool edge = r2 > rows || seen(p, s, place_of(p, r1).query) < min(key0 + 32, s.m);
#pragma unroll
            for (int b = block0; b < block0 + BLOCKS; ++b) {
                f32x16 x{}, ds{};
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) {
                    x = mma(L::rows(queries, 32 * b + col, c, h), k[c], x);
                    if constexpr (LDS_V) ds = mma(L::rows(grads, 32 * b + col, c, h), L::rows(values, wave * 32 + col, c, h), ds);
                    else ds = mma(L::rows(grads, 32 * b + col, c, h), v[c], ds);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = 32 * b + 8 * (e / 4) + 4 * h + e % 4;
                    x[e] = exp2_hw(fmaf(x[e], p.scale2, -lses[buf][r]));
                    ds[e] = x[e] * (ds[e] - deltas[buf][r]);
                }
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool out = key >= seen(p, s, place_of(p, r0 + 32 * b + 8 * (e / 4) + 4 * h + e % 4).query);
                        x[e] = out ? 0.0f : x[e], ds[e] = out ? 0.0f : ds[e];
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> w = as_operand<T>(x, c);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dv[d] = mma(L::columns(grads, d, 2 * b + c, lane), w, dv[d]);
                }
                range.fit(ds, dk);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> w = as_operand<T>(ds, c);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) dk[d] = mma(L::columns(queries, d, 2 * b + c, lane), w, dk[d]);
                }
            }
        }
        if constexpr (BUFFERS == 2) {
            buf ^= 1;
        } else {
            __syncthreads();
            if (r0 > from) fetch(r0 - BM, 0);
        }
        landed();
        __syncthreads();
    }
    // a key that is not there: its column holds exp(0 - lse) of the rows, where they see all keys that are, which may
    // have passed the type's range
    if (!live) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) dk[b] = dv[b] = f32x16{};
    }
    const float by_v = exp2_hw(-kShift<T>), by_k = static_cast<float>(a.scale) * range.back() * by_v;
    if constexpr (SHARED) {
        static_assert(sizeof(tiles) >= Join<DP>::kBytes);
        Join<DP> join(&tiles[0][0][0]);
        const int32_t row = tile0 + join.r;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            join.put(wave, col, side == 0 ? dk : dv, side == 0 ? by_k : by_v, h);
            __syncthreads();
            if (row < s.total) {
                float y[Join<DP>::kEach] = {};
#pragma unroll
                for (int w = 0; w < 4; ++w) join.get(y, w, 1.0f);
                T* const to = side == 0 ? row_of<T>(a.d_k_dev, a.d_k_stride, s.batch, s.k0 + row, u.head)
                                        : row_of<T>(a.d_v_dev, a.d_v_stride, s.batch, s.k0 + row, u.head);
                store_some<Join<DP>::kEach>(to + join.d0, y, a.dim - join.d0);
            }
            __syncthreads();
        }
    } else if (key < s.total) {
        store_row<T, DP>(row_of<T>(a.d_k_dev, a.d_k_stride, s.batch, s.k0 + key, u.head), dk, by_k, a.dim, h);
        store_row<T, DP>(row_of<T>(a.d_v_dev, a.d_v_stride, s.batch, s.k0 + key, u.head), dv, by_v, a.dim, h);
    }
}

// ---------------------------------------------------------------------- host

constexpr int64_t kNear = int64_t{1} << 30;  // elements that a lane's offset of 32 bits, in bytes, reaches over

// Whether heads' chunks of 16 bytes are whole and aligned.
bool aligned(const void* at, const int64_t* stride, int bytes, int32_t dim) {
    return reinterpret_cast<uintptr_t>(at) % 16 == 0 && dim * bytes % 16 == 0 && stride[0] * bytes % 16 == 0 &&
           stride[1] * bytes % 16 == 0 && stride[2] * bytes % 16 == 0;
}

int check(const mgopt_attention_args* a, const char* what) {
    const std::string w(what);
    if (!a) return set_error(MGOPT_E_INVALID, w + ": NULL arguments");
    if (!known_dtype(a->dtype)) return set_error(MGOPT_E_INVALID, w + ": bad dtype");
    if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->sequences < 0)
        return set_error(MGOPT_E_INVALID, w + ": negative sizes");
    if (a->q_heads < 1 || a->k_heads < 1 || a->q_heads % a->k_heads != 0)
        return set_error(MGOPT_E_INVALID, w + ": the query heads must be a multiple of the key heads");
    if (a->dim < 1) return set_error(MGOPT_E_INVALID, w + ": heads need at least one element");
    if (a->dim > MGOPT_MAX_ATTENTION_DIM)
        return set_error(MGOPT_E_LIMIT, w + ": heads of more than " + std::to_string(MGOPT_MAX_ATTENTION_DIM) + " elements");
    // far smaller ones are 0 in fp32, and 0 times a masked score's -inf a NaN
    if (!(a->scale >= 0x1p-100) || !(a->scale < 0x1p100))
        return set_error(MGOPT_E_INVALID, w + ": the scale must be at least 2^-100 and below 2^100");
    if ((a->q_offsets_dev == nullptr) != (a->k_offsets_dev == nullptr))
        return set_error(MGOPT_E_INVALID, w + ": offsets of both sides, or of none");
    if (a->q_offsets_dev && (a->batch != 1 || a->q_lengths_dev || a->k_lengths_dev))
        return set_error(MGOPT_E_INVALID, w + ": packed sequences are a batch of 1 and have no lengths");
    if ((a->q_offsets_dev || a->q_lengths_dev || a->k_lengths_dev) && a->offset_bytes != 4 && a->offset_bytes != 8)
        return set_error(MGOPT_E_INVALID, w + ": offsets and lengths have 4 or 8 bytes");
    for (const int64_t* stride : {a->q_stride, a->k_stride, a->v_stride, a->out_stride, a->grad_out_stride, a->d_q_stride,
                                  a->d_k_stride, a->d_v_stride})
        if (stride[0] < 0 || stride[1] < 0 || stride[2] < 0) return set_error(MGOPT_E_INVALID, w + ": negative strides");
    // offsets over a tile of 128 of them have 32 bits; one alone has no next
    if (a->keys > 1 && (a->k_stride[1] >= kNear / 128 || a->v_stride[1] >= kNear / 128))
        return set_error(MGOPT_E_LIMIT, w + ": keys or values 2^23 elements apart or more");
    const int64_t most = int64_t{1} << 30;
    if (a->keys > most || a->queries > most / a->q_heads || a->sequences > most || a->q_heads > (1 << 20))
        return set_error(MGOPT_E_LIMIT, w + ": more than 2^30 keys, sequences or queries times heads");
    if (a->batch > max_blocks(kThreads)) return set_error(MGOPT_E_LIMIT, w + ": more rows of the batch than work-groups");
    return 0;
}

// Work-groups of `tile` rows, `per` a token, on one side.
int places(const mgopt_attention_args& a, int64_t tokens, int64_t per, int tile, const char* what, uint32_t& tiles, uint32_t& blocks) {
    const int64_t each = (tokens * per + tile - 1) / tile;
    const int64_t slots = a.q_offsets_dev ? tokens * per / tile + a.sequences + 2 : each;
    tiles = static_cast<uint32_t>(each);
    const int64_t most = max_blocks(kThreads);
    if (a.q_offsets_dev ? slots > most / a.k_heads : a.batch > 0 && each > most / a.k_heads / a.batch)
        return set_error(MGOPT_E_LIMIT, std::string(what) + ": too many work-groups");
    blocks = static_cast<uint32_t>(slots * (a.q_offsets_dev ? 1 : a.batch) * a.k_heads);
    return 0;
}

// How the forward pass takes its rows: whether the waves of a work-group share 32 of them, and in how many parts the
// keys of each row are cut where the rows alone leave the chip short of work.
struct Form {
    bool shared;
    uint32_t splits;
};
constexpr int64_t kMinShare = 256;   // keys of a part at least
constexpr int64_t kFill = 512;       // work-groups that fill the chip: two a CU
constexpr int64_t kFew = 128, kFewF32 = 512;  // fewer than this in the backward pass, and waves share rows, or keys
// (8 x 128 tokens of 4 heads of 32 in fp32 16 us, not shared 32; 2 x 1,024 of 12 heads of 64 in fp32 166, not shared 282;
// 2 x 1,024 of 32 + 8 heads of 128 in bf16, 128 work-groups, 249, not shared 229),
// but for 2-byte heads of more than 64 and keys of more rows: 2 x 2,000 queries of 6 + 2 heads of 128 391 us, shared 438;
// 2,048 of 4 + 4 160 us, shared 100
constexpr int64_t kFewRows = 4096;
int64_t groups_of(const mgopt_attention_args& a, int64_t tokens, int64_t per, int tile) {
    return a.k_heads * (a.q_offsets_dev ? tokens * per / tile + a.sequences : (tokens * per + tile - 1) / tile * a.batch);
}
Form form_of(const mgopt_attention_args& a) {
    const int64_t per = a.q_heads / a.k_heads;
    Form f;
    f.shared = groups_of(a, a.queries, per, kTile) < kFill;
    const int64_t work = std::max<int64_t>(1, groups_of(a, a.queries, per, f.shared ? kShared : kTile));
    const int64_t keys = a.q_offsets_dev ? a.keys / std::max<int64_t>(1, a.sequences) : a.keys;
    const int64_t s = std::min((kFill + work - 1) / work, keys / kMinShare);
    f.splits = static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(s, kMostSplits)));
    // few rows over long caches are bound by memory, and two tiles a work-group on their way matter more than its waves:
    // one row of 32 + 8 heads of 128 over 131,071 keys 106 us, shared 116; of 8 x 500 keys 17, shared 12
    if (a.queries * per <= kShared && a.dim > 64 && a.dtype != MGOPT_F32 && keys / f.splits >= 1024) f.shared = false;
    return f;
}

template <typename F>
int with_dim(int32_t dim, F&& f) {
    if (dim <= 32) return f(std::integral_constant<int, 32>{});
    if (dim <= 64) return f(std::integral_constant<int, 64>{});
    if (dim <= 96) return f(std::integral_constant<int, 96>{});
    return f(std::integral_constant<int, 128>{});
}

int64_t rows_of_all(const mgopt_attention_args& a) { return a.batch * a.queries * a.q_heads; }

AttArgs args_of(const mgopt_attention_args& a) {
    AttArgs p{};
    p.a = a;
    p.group = static_cast<uint32_t>(a.q_heads / a.k_heads);
    uint32_t bits = 0;
    while ((uint64_t{1} << bits) < p.group) ++bits;
    if (bits > 0) p.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + p.group - 1) / p.group), p.shift = bits - 1;
    p.scale2 = static_cast<float>(a.scale * kLog2e);
    p.aligned_keys = aligned(a.k_dev, a.k_stride, dtype_bytes(a.dtype), a.dim) && aligned(a.v_dev, a.v_stride, dtype_bytes(a.dtype), a.dim);
    return p;
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int64_t mgopt_attention_workspace(const mgopt_attention_args* a, int32_t backward) {
    if (check(a, "attention_workspace")) return -1;
    if (backward) return rows_of_all(*a) * 8;
    const int64_t splits = form_of(*a).splits;
    return splits > 1 ? splits * rows_of_all(*a) * (a->dim + 2) * 4 : 0;
}

MGOPT_API int mgopt_attention(const mgopt_attention_args* a, void* stream) {
    if (int rc = check(a, "attention")) return rc;
    if (rows_of_all(*a) == 0) return 0;
    if (!a->q_dev || !a->out_dev || (a->keys > 0 && (!a->k_dev || !a->v_dev)))
        return set_error(MGOPT_E_INVALID, "attention: NULL argument");
    AttArgs p = args_of(*a);
    const Form form = form_of(*a);
    p.splits = form.splits;
    if (p.splits > 1) {
        if (!a->workspace_dev || reinterpret_cast<uintptr_t>(a->workspace_dev) % 16 != 0)
            return set_error(MGOPT_E_ALIGN, "attention: the workspace must be 16-byte aligned and not NULL");
        p.part_out = static_cast<float*>(a->workspace_dev);
        p.part_ml = p.part_out + p.splits * rows_of_all(*a) * a->dim;
    }
    uint32_t blocks;
    if (int rc = places(*a, a->queries, p.group, form.shared ? kShared : kTile, "attention", p.tiles, blocks)) return rc;
    if (p.splits > 1 && rows_of_all(*a) > max_blocks(kThreads)) return set_error(MGOPT_E_LIMIT, "attention: too many rows");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_dim(a->dim, [&](auto d) {
            constexpr int DP = decltype(d)::value;
            const dim3 grid(blocks, p.splits), threads(kThreads);
            if (form.shared && p.splits > 1) hipLaunchKernelGGL((attention_kernel<T, DP, true, true>), grid, threads, 0, s, p);
            else if (form.shared) hipLaunchKernelGGL((attention_kernel<T, DP, false, true>), grid, threads, 0, s, p);
            else if (p.splits > 1) hipLaunchKernelGGL((attention_kernel<T, DP, true, false>), grid, threads, 0, s, p);
            else hipLaunchKernelGGL((attention_kernel<T, DP, false, false>), grid, threads, 0, s, p);
            if (int rc = launched("attention")) return rc;
            if (p.splits == 1) return 0;
            hipLaunchKernelGGL((join_kernel<T>), dim3(static_cast<uint32_t>(rows_of_all(*a))), dim3(kThreads), 0, s, p);
            return launched("attention");
        });
    });
}

MGOPT_API int mgopt_attention_backward(const mgopt_attention_args* a, void* stream) {
    if (int rc = check(a, "attention_backward")) return rc;
    const bool rows = rows_of_all(*a) > 0, keys = a->batch * a->keys > 0;
    if (rows && (!a->q_dev || !a->out_dev || !a->grad_out_dev || !a->lse_dev || !a->d_q_dev))
        return set_error(MGOPT_E_INVALID, "attention_backward: NULL argument");
    if (keys && (!a->k_dev || !a->v_dev || !a->d_k_dev || !a->d_v_dev))
        return set_error(MGOPT_E_INVALID, "attention_backward: NULL argument");
    if (rows && (!a->workspace_dev || reinterpret_cast<uintptr_t>(a->workspace_dev) % 16 != 0))
        return set_error(MGOPT_E_ALIGN, "attention_backward: the workspace must be 16-byte aligned and not NULL");
    AttArgs p = args_of(*a);
    p.stats = static_cast<float*>(a->workspace_dev);
    const int64_t few = a->dtype == MGOPT_F32 ? kFewF32 : kFew;
    const bool shared_rows = groups_of(*a, a->queries, p.group, kTile) < few, shared_keys = groups_of(*a, a->keys, 1, kTile) < few &&
        (a->dim <= 64 || a->dtype == MGOPT_F32 || a->queries * p.group <= kFewRows);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        return with_dim(a->dim, [&](auto d) -> int {
            constexpr int DP = decltype(d)::value;
            p.aligned_rows = aligned(a->q_dev, a->q_stride, sizeof(T), a->dim) && aligned(a->grad_out_dev, a->grad_out_stride, sizeof(T), a->dim);
            p.even_rows = p.aligned_rows && (shared_keys ? 128 : kRows<T, DP>) % p.group == 0;
            for (const int64_t* stride : {a->q_stride, a->grad_out_stride})
                p.even_rows = p.even_rows && stride[1] < kNear / 512 && stride[2] < kNear / 8 / p.group;
            uint32_t blocks;
            if (rows) {
                if (int rc = places(*a, a->queries, p.group, shared_rows ? kShared : kTile, "attention_backward", p.tiles, blocks)) return rc;
                if (shared_rows) hipLaunchKernelGGL((attention_dq_kernel<T, DP, true>), dim3(blocks), dim3(kThreads), 0, s, p);
                else hipLaunchKernelGGL((attention_dq_kernel<T, DP, false>), dim3(blocks), dim3(kThreads), 0, s, p);
                if (int rc = launched("attention_backward")) return rc;
            }
            if (!keys) return 0;
            if (int rc = places(*a, a->keys, 1, shared_keys ? kShared : kTile, "attention_backward", p.tiles, blocks)) return rc;
            if (shared_keys) hipLaunchKernelGGL((attention_dkv_kernel<T, DP, true>), dim3(blocks), dim3(kThreads), 0, s, p);
            else hipLaunchKernelGGL((attention_dkv_kernel<T, DP, false>), dim3(blocks), dim3(kThreads), 0, s, p);
            return launched("attention_backward");
        });
    });
}

}  // extern "C"
