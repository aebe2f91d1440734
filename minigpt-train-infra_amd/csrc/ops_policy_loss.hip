// ops_policy_loss.hip -- the clipped policy loss with a KL term over a batch's
// logits, its gradient, and the log-probabilities it is made of.
//
// For row n with logits x, target y, temperature T and weight w_n (the mask):
//
//     logp   = x_y / T - log sum_j exp(x_j / T)        ratio = exp(logp - old)
//     policy = -min(ratio * A, clip(ratio, lo, hi) * A)
//     kl     = exp(r) - r - 1,  r = ref - logp
//     loss   = sum_n w_n (policy + kl_coef * kl) / sum_n w_n
//
// and, with p the softmax and [.] one where it holds,
//
//     slope  = w_n / sum(w) * ((clipped ? 0 : -ratio * A) + kl_coef * (1 - exp(r)))
//     dx_j   = scale * slope / T * ([j = y] - p_j)
//
// A row is one work-group's: a pass over it keeps, per thread, the maximum m
// and a sum s of powers of two; the row's scalars are formed once, in 64 bits; a
// second pass writes the gradient.  Rows of weight 0 are not read.
//
// With c = log2(e) / T, s = sum 2^((x - m) c): the difference is formed first.
// One fused multiply-add of x c and a rounded m c is an instruction less (153 us
// for 157, vectors taken singly, in the first case below), but off by m c's
// rounding, which passes every exponent where m c passes 2^32: a row of -1e10, or
// a small temperature.
//
// A row is held in registers between the passes (cached_kernel), as it came, so
// that it is read once; what does not fit is read again.  Few long rows are cut
// in slices, a work-group each (slice_kernel), and joined by those that finish
// them (finish_kernel).
//
// Bound by memory: a row's logits once, its gradient once.  8,192 rows of 50,304
// bf16: log-probabilities 154 us (5.3 TB/s).  4,096 rows of 151,936 bf16, a quarter
// of weight 0: loss and gradient 421 us (5.2 TB/s); one such row fills a CU's
// registers, so that its read, its join and its write follow each other.  As two
// passes, for autograd: the loss 181 us (5.1 TB/s), the gradient from what it kept
// (grad_kernel) 422 (5.2).
#include "ops_common.h"

namespace mgopt {
namespace {

enum Mode { kLogp, kLoss, kLossGrad, kGrad };

// What a forward pass keeps of a row for a backward pass of its own.
struct RowStats {
    float m, s;
    double slope;  // by the row's log-probability, with neither weight nor scale
};

struct PolicyArgs {
    const void* logits;
    int64_t row_stride, rows, vocab, first_row;
    const void* targets;
    int32_t target_bytes, mask_kind;
    const float *old_logp, *ref_logp, *advantages;
    const void* mask;
    double low, high, kl_coef, inv_temp;
    float c;                     // log2(e) / T, a normal number
    const float* grad_scale;     // may be NULL
    const double* weight_sum;    // NULL: every row's weight is 1
    float* log_probs;
    RowStats* stats;             // of each row: written by kLoss, read by kGrad
    float4* terms;               // w * policy, w * kl, w * clipped: rounded to 32 bits, 2^-24 of a row's term, and summed in 64
    void* d_logits;
    int64_t d_stride;
    uint32_t slices = 1;         // of a row
    int64_t slice;               // elements of one
    float2* parts;               // m and s of each slice
    float* picked;               // the targets' logits: a gradient in place may overwrite them before another slice is done
};

__device__ __forceinline__ float weight_at(const void* mask, int32_t kind, int64_t n) {
    if (kind == MGOPT_MASK_NONE) return 1.0f;
    if (kind == MGOPT_MASK_BYTES) return static_cast<const uint8_t*>(mask)[n] != 0 ? 1.0f : 0.0f;
    return static_cast<const float*>(mask)[n];
}

// The maximum starts at the lowest finite value: -inf - -inf does not occur, -inf
// counts 0, and a row of nothing else has s = 0, whose log is -inf.  Powers below
// 2^-126 come out as 0: beside the largest element's 1 they are nothing, and a
// gradient's elements of such a p are 0.
struct Running {
    float m = -3.402823466e38f, s = 0.0f;
};
__device__ __forceinline__ Running join(Running a, Running b, float c) {
    const float m = fmaxf(a.m, b.m);
    return {m, a.s * exp2_hw((a.m - m) * c) + b.s * exp2_hw((b.m - m) * c)};
}
template <int N>
__device__ __forceinline__ void take(Running& r, const float (&x)[N], float c) {
    float m = r.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    r.s *= exp2_hw((r.m - m) * c);
    r.m = m;
#pragma unroll
    for (int i = 0; i < N; ++i) r.s += exp2_hw((x[i] - m) * c);
}

template <int NT>
__device__ __forceinline__ Running join_block(Running r, float c) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) r = join(r, Running{__shfl_xor(r.m, off), __shfl_xor(r.s, off)}, c);
    if constexpr (NT > 64) {
        __shared__ float part_m[NT / 64], part_s[NT / 64];
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) part_m[wave] = r.m, part_s[wave] = r.s;
        __syncthreads();
        r = {part_m[0], part_s[0]};
#pragma unroll 1
        for (int i = 1; i < NT / 64; ++i) r = join(r, Running{part_m[i], part_s[i]}, c);
    }
    return r;
}

// What the row's scalars are made of, read before the row so that nothing
// waits for them after it.
struct RowInputs {
    int64_t target;
    float x, old_logp, advantage, ref;  // x: the target's logit, NaN for a target outside the vocabulary
    float scale;                        // of the gradient, with the weights' sum
    double total;
};
__device__ __forceinline__ void gradient_inputs(const PolicyArgs& a, RowInputs& r) {
    r.scale = a.grad_scale != nullptr ? *a.grad_scale : 1.0f;
    r.total = a.weight_sum != nullptr ? *a.weight_sum : static_cast<double>(a.rows);
}
template <typename T, Mode MODE>
__device__ __forceinline__ RowInputs row_inputs(const PolicyArgs& a, int64_t n, bool pick = true) {
    RowInputs r{};
    r.target = id_at(a.targets, n, a.target_bytes);
    if (pick)
        r.x = r.target >= 0 && r.target < a.vocab
                  ? static_cast<float>(static_cast<const T*>(a.logits)[n * a.row_stride + r.target])
                  : __builtin_nanf("");
    if (MODE == kLogp) return r;
    r.old_logp = a.old_logp[n], r.advantage = a.advantages[n];
    if (a.ref_logp != nullptr) r.ref = a.ref_logp[n];
    gradient_inputs(a, r);
    return r;
}

struct RowResult {
    float slope, k;  // of the gradient: slope * [j = y] + k * 2^((x - m) c)
};

__device__ __forceinline__ RowResult row_gradient(const PolicyArgs& a, double slope, const RowInputs& in, float w, float s) {
    // where the weights' sum is 0 the loss is 0, and so is its gradient
    slope = in.total == 0.0 ? 0.0 : slope * (w / in.total * a.inv_temp * static_cast<double>(in.scale));
    return {static_cast<float>(slope), static_cast<float>(-slope / static_cast<double>(s))};
}

// What one row adds to the loss, and its slope, from m and s.  A backward pass of
// its own takes the slope from here: formed again from the rounded log-probability,
// it could hold a row at the clip's edge that the loss did not.
template <Mode MODE>
__device__ RowResult row_scalars(const PolicyArgs& a, int64_t n, const RowInputs& in, float w, float m, float s,
                                 bool write = true) {
    const double logp = (static_cast<double>(in.x) - static_cast<double>(m)) * a.inv_temp - log(static_cast<double>(s));
    if (write) a.log_probs[n] = static_cast<float>(logp);
    if constexpr (MODE == kLogp) return {};
    const double A = in.advantage, ratio = exp(logp - static_cast<double>(in.old_logp));
    const double s1 = ratio * A, s2 = fmin(fmax(ratio, a.low), a.high) * A;
    const bool held = s2 < s1;
    double slope = held ? 0.0 : -s1, kl = 0.0;
    if (a.ref_logp != nullptr) {
        const double r = static_cast<double>(in.ref) - logp, e = expm1(r);
        kl = e - r;
        slope -= a.kl_coef * e;
    }
    if (write)
        a.terms[n] = make_float4(static_cast<float>(w * -(held ? s2 : s1)), static_cast<float>(w * kl), held ? w : 0.0f, 0.0f);
    if constexpr (MODE == kLoss) {
        a.stats[n] = {m, s, slope};
        return {};
    }
    return row_gradient(a, slope, in, w, s);
}

template <typename T, int NT>
__device__ __forceinline__ void clear(T* dx, int64_t begin, int64_t end) {
    constexpr int N = 16 / sizeof(T);
    const float zero[N] = {};
    for (int64_t i = begin + static_cast<int64_t>(threadIdx.x) * N; i < end; i += int64_t{NT} * N)
        store_some<N>(dx + i, zero, end - i);
}

// A row of weight 0: its outputs are zeros.
template <typename T, int NT, Mode MODE>
__device__ __forceinline__ void skip_row(const PolicyArgs& a, int64_t n, T* dx) {
    if (threadIdx.x == 0) {
        a.log_probs[n] = 0.0f;
        if (MODE != kLogp) a.terms[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if constexpr (MODE == kLossGrad) clear<T, NT>(dx, 0, a.vocab);
}

// One vector of the gradient, from column i on.
template <int N>
__device__ __forceinline__ void to_gradient(float (&v)[N], const RowResult& q, float m, float c, int64_t y, int64_t i) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = q.k * exp2_hw((v[j] - m) * c);
    if (y >= i && y < i + N) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (y == i + j) v[j] += q.slope;
    }
}

// The gradient of columns begin to end, from their logits.
template <typename T, int NT>
__device__ __forceinline__ void write_gradient(const T* x, T* dx, int64_t begin, int64_t end, const RowResult& q,
                                               float m, float c, int64_t y) {
    constexpr int N = 16 / sizeof(T);
    for (int64_t i = begin + static_cast<int64_t>(threadIdx.x) * N; i < end; i += int64_t{NT} * N) {
        float v[N];
        load_some<N>(v, x + i, end - i);
        to_gradient<N>(v, q, m, c, y, i);
        store_some<N>(dx + i, v, end - i);
    }
}

// 16 bytes of a row as they came, and their values.
typedef uint32_t Raw __attribute__((ext_vector_type(4)));
template <typename T, int N>
__device__ __forceinline__ void widen(float (&v)[N], const Raw& raw) {
    const vec_t<T, N> q = __builtin_bit_cast(vec_t<T, N>, raw);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = static_cast<float>(q[j]);
}

// The forward forms.  Each thread holds NV vectors of its row, so that rows of at
// most NT * NV of them (and a tail of less than one) are read once; LONG: what
// lies beyond is read again for the gradient.  All of a row's first loads are
// issued before one is used; vectors past its end repeat its last one and are
// not counted.  Vectors are taken in pairs, for one rescaling of two (log-
// probabilities of 8,192 rows of 50,304 bf16: 154 us for 157).
template <typename T, int NT, int NV, Mode MODE, bool LONG>
__global__ __launch_bounds__(NT) void cached_kernel(PolicyArgs a) {
    constexpr int N = 16 / sizeof(T);
    const int64_t n = a.first_row + blockIdx.x;
    const float w = weight_at(a.mask, a.mask_kind, n);
    const T* x = static_cast<const T*>(a.logits) + n * a.row_stride;
    T* dx = static_cast<T*>(a.d_logits) + n * a.d_stride;
    if (w == 0.0f) return skip_row<T, NT, MODE>(a, n, dx);
    // vectors of the row; LONG ones have more than 32 bits count
    using Index = std::conditional_t<LONG, int64_t, int>;
    const Index V = static_cast<Index>(a.vocab), full = V / N, tail = V - full * N;
    const int t = threadIdx.x;
    Raw raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Index v = i * NT + t;
        raw[i] = full > 0 ? __builtin_bit_cast(Raw, __builtin_nontemporal_load(reinterpret_cast<const vec_t<T, N>*>(x) +
                                                                              (v < full ? v : full - 1)))
                          : Raw{};
    }
    float last[1] = {t < tail ? static_cast<float>(x[full * N + t]) : -INFINITY};
    __shared__ RowInputs in;  // not in registers, which the row needs
    if (t == 0) in = row_inputs<T, MODE>(a, n);
    Running r;
    take<1>(r, last, a.c);
#pragma unroll
    for (int i = 0; i < NV; i += 2) {
        __builtin_amdgcn_sched_barrier(0);  // two vectors' values at a time: all of them widened do not fit
        float v[2][N];
        widen<T, N>(v[0], raw[i]);
        widen<T, N>(v[1], raw[i + 1]);
        if ((i + 1) * NT + t < full) take<2 * N>(r, reinterpret_cast<const float(&)[2 * N]>(v), a.c);
        else if (i * NT + t < full) take<N>(r, v[0], a.c);
        asm("" : "+v"(raw[i]), "+v"(raw[i + 1]));  // widened again below, not kept
    }
    if constexpr (LONG) {
#pragma unroll 4
        for (int64_t i = int64_t{NV} * NT + t; i < full; i += NT) {
            float v[N];
            load<N>(v, x + i * N);
            take<N>(r, v, a.c);
        }
    }
    r = join_block<NT>(r, a.c);
    __shared__ RowResult shared;
    if (t == 0) shared = row_scalars<MODE>(a, n, in, w, r.m, r.s);
    if constexpr (MODE != kLossGrad) return;
    __syncthreads();
    const RowResult q = shared;
    const int64_t y = id_at(a.targets, n, a.target_bytes);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Index at = i * NT + t;
        if (at >= full) continue;
        __builtin_amdgcn_sched_barrier(0);
        float v[N];
        widen<T, N>(v, raw[i]);
        to_gradient<N>(v, q, r.m, a.c, y, static_cast<int64_t>(at) * N);
        store_nt<N>(dx + static_cast<int64_t>(at) * N, v);
    }
    if constexpr (LONG) {
#pragma unroll 4
        for (int64_t i = int64_t{NV} * NT + t; i < full; i += NT) {
            float v[N];
            load<N>(v, x + i * N);
            to_gradient<N>(v, q, r.m, a.c, y, i * N);
            store_nt<N>(dx + i * N, v);
        }
    }
    if (t < tail) {
        to_gradient<1>(last, q, r.m, a.c, y, full * N + t);
        dx[full * N + t] = static_cast<T>(last[0]);
    }
}

template <int V>
using Int = std::integral_constant<int, V>;

// The gradient from what a forward pass kept, a slice of a row a work-group.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void grad_kernel(PolicyArgs a) {
    const uint32_t row = blockIdx.x / a.slices, part = blockIdx.x - row * a.slices;
    const int64_t n = a.first_row + row, begin = part * a.slice, end = begin + a.slice < a.vocab ? begin + a.slice : a.vocab;
    const float w = weight_at(a.mask, a.mask_kind, n);
    const T* x = static_cast<const T*>(a.logits) + n * a.row_stride;
    T* dx = static_cast<T*>(a.d_logits) + n * a.d_stride;
    if (w == 0.0f) return clear<T, NT>(dx, begin, end);
    const RowStats kept = a.stats[n];
    __shared__ RowResult shared;
    if (threadIdx.x == 0) {
        RowInputs in{};
        gradient_inputs(a, in);
        shared = row_gradient(a, kept.slope, in, w, kept.s);
    }
    __syncthreads();
    write_gradient<T, NT>(x, dx, begin, end, shared, kept.m, a.c, id_at(a.targets, n, a.target_bytes));
}

// m and s of one slice of a row.
constexpr int kSliceBlock = 256;
template <typename T>
__global__ __launch_bounds__(kSliceBlock) void slice_kernel(PolicyArgs a) {
    constexpr int N = 16 / sizeof(T);
    const uint32_t n = blockIdx.x / a.slices, part = blockIdx.x - n * a.slices, t = threadIdx.x;
    if (weight_at(a.mask, a.mask_kind, n) == 0.0f) return;
    const T* x = static_cast<const T*>(a.logits) + n * a.row_stride;
    const int64_t begin = part * a.slice, end = begin + a.slice < a.vocab ? begin + a.slice : a.vocab;
    const int64_t full = end > begin ? begin + (end - begin) / N * N : begin;
    if (part == 0 && t == 0) a.picked[n] = row_inputs<T, kLogp>(a, n).x;
    Running r;
    if (full + t < end) {
        const float v[1] = {static_cast<float>(x[full + t])};
        take<1>(r, v, a.c);
    }
#pragma unroll 4
    for (int64_t i = begin + static_cast<int64_t>(t) * N; i < full; i += kSliceBlock * N) {
        float v[N];
        load<N>(v, x + i);
        take<N>(r, v, a.c);
    }
    r = join_block<kSliceBlock>(r, a.c);
    if (t == 0) a.parts[blockIdx.x] = make_float2(r.m, r.s);
}

// Joins a row's slices in their order of lanes, and does what the mode asks: a
// work-group a row, or, for the gradient, a slice.
template <typename T, Mode MODE>
__global__ __launch_bounds__(kSliceBlock) void finish_kernel(PolicyArgs a) {
    constexpr bool kWithGrad = MODE == kLossGrad;
    const uint32_t n = kWithGrad ? blockIdx.x / a.slices : blockIdx.x, part = kWithGrad ? blockIdx.x - n * a.slices : 0;
    const float w = weight_at(a.mask, a.mask_kind, n);
    const int64_t begin = part * a.slice, end = begin + a.slice < a.vocab ? begin + a.slice : a.vocab;
    T* dx = static_cast<T*>(a.d_logits) + n * a.d_stride;
    if (w == 0.0f) {
        if (part == 0 && threadIdx.x == 0) {
            a.log_probs[n] = 0.0f;
            if (MODE != kLogp) a.terms[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        if constexpr (kWithGrad) clear<T, kSliceBlock>(dx, begin, end);
        return;
    }
    __shared__ RowResult shared;
    __shared__ float top;
    if (threadIdx.x < 64) {
        Running r;
        for (uint32_t i = threadIdx.x; i < a.slices; i += 64) {
            const float2 p = a.parts[n * a.slices + i];
            r = join(r, Running{p.x, p.y}, a.c);
        }
        r = join_block<64>(r, a.c);
        if (threadIdx.x == 0) {
            RowInputs in = row_inputs<T, MODE>(a, n, false);  // the target's logit may be overwritten
            in.x = a.picked[n];
            shared = row_scalars<MODE>(a, n, in, w, r.m, r.s, part == 0);
            top = r.m;
        }
    }
    if constexpr (kWithGrad) {
        __syncthreads();
        write_gradient<T, kSliceBlock>(static_cast<const T*>(a.logits) + n * a.row_stride, dx, begin, end, shared, top,
                                       a.c, id_at(a.targets, n, a.target_bytes));
    }
}

constexpr int kSumBlock = 1024;

template <typename X>
__device__ __forceinline__ X sum_block(X x) {
    __shared__ X part[kSumBlock / 64];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    __syncthreads();  // an earlier call's reads
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
    __syncthreads();
    x = part[0];
#pragma unroll
    for (int i = 1; i < kSumBlock / 64; ++i) x += part[i];
    return x;
}

__global__ __launch_bounds__(kSumBlock) void weight_sum_kernel(const void* mask, int32_t kind, int64_t rows, double* out) {
    double x = 0.0;
#pragma unroll 8
    for (int64_t n = threadIdx.x; n < rows; n += kSumBlock) x += weight_at(mask, kind, n);
    x = sum_block(x);
    if (threadIdx.x == 0) *out = x;
}

// loss, policy, kl, clipped share from the rows' terms.  Weights whose sum is 0
// make all four 0.
__global__ __launch_bounds__(kSumBlock) void policy_sum_kernel(const float4* terms, int64_t rows, const double* weight_sum,
                                                               double kl_coef, float* loss, float* parts) {
    double p = 0.0, k = 0.0, h = 0.0;
#pragma unroll 8
    for (int64_t n = threadIdx.x; n < rows; n += kSumBlock) {
        const float4 t = terms[n];
        p += t.x, k += t.y, h += t.z;
    }
    p = sum_block(p), k = sum_block(k), h = sum_block(h);
    if (threadIdx.x == 0) {
        const double total = weight_sum != nullptr ? *weight_sum : static_cast<double>(rows);
        const double inv = total == 0.0 ? 0.0 : 1.0 / total;
        *loss = static_cast<float>((p + kl_coef * k) * inv);
        parts[0] = static_cast<float>(p * inv);
        parts[1] = static_cast<float>(k * inv);
        parts[2] = static_cast<float>(h * inv);
    }
}

// Slices of a row: rows too few for the chip's 256 CUs are cut, in 1,024 slices
// together at most, where a row makes six slices of 8 vectors a thread or more; a
// shorter one is done by a work-group of its own in the time of the second launch.
// Kernels of loss and gradient in bf16, traced, in us, cut / whole: 4 rows of
// 151,936 12.7 / 19.6, 60 rows 19.5 / 22.1; 8 rows of 50,304 11.4 / 10.4.  Log-
// probabilities of one row of 151,936: 7.3 / 11.7.
constexpr int64_t kSplitRows = 128, kSplitSlices = 1024;
template <typename T>
void cut(PolicyArgs& a) {
    constexpr int64_t N = 16 / sizeof(T);
    const int64_t most = (a.vocab / N + 2047) / 2048;
    a.slices = 1, a.slice = a.vocab;
    if (a.rows >= kSplitRows || most < 6 || a.parts == nullptr) return;
    const int64_t slices = std::min(most, kSplitSlices / a.rows);
    if (slices < 2) return;
    a.slices = static_cast<uint32_t>(slices);
    a.slice = ((a.vocab + slices - 1) / slices + N - 1) / N * N;
}

// The kernel for rows of this length: threads enough to keep a row's loads in
// flight, few enough that short rows do not idle.
template <typename T, Mode MODE>
int launch_rows(PolicyArgs a, hipStream_t s) {
    constexpr int N = 16 / sizeof(T);
    const int64_t most = max_blocks(1024), vecs = a.vocab / N;
    cut<T>(a);
    if (a.slices > 1) {
        const dim3 every(static_cast<uint32_t>(a.rows * a.slices)), block(kSliceBlock);
        if constexpr (MODE == kGrad) {
            hipLaunchKernelGGL((grad_kernel<T, kSliceBlock>), every, block, 0, s, a);
        } else {
            hipLaunchKernelGGL((slice_kernel<T>), every, block, 0, s, a);
            if (int rc = launched("slice_kernel")) return rc;
            if (MODE == kLossGrad) hipLaunchKernelGGL((finish_kernel<T, MODE>), every, block, 0, s, a);
            else hipLaunchKernelGGL((finish_kernel<T, MODE>), dim3(static_cast<uint32_t>(a.rows)), dim3(64), 0, s, a);
        }
        return launched("policy_loss");
    }
    for (a.first_row = 0; a.first_row < a.rows; a.first_row += most) {
        const dim3 grid(static_cast<uint32_t>(a.rows - a.first_row < most ? a.rows - a.first_row : most));
        const auto cached = [&](auto threads, auto held) {
            constexpr int NT = decltype(threads)::value, NV = decltype(held)::value;
            if (vecs > NT * NV) return false;
            hipLaunchKernelGGL((cached_kernel<T, NT, NV, MODE, false>), grid, dim3(NT), 0, s, a);
            return true;
        };
        if constexpr (MODE == kGrad) {
            if (vecs <= 256) hipLaunchKernelGGL((grad_kernel<T, 64>), grid, dim3(64), 0, s, a);
            else if (vecs <= 2048) hipLaunchKernelGGL((grad_kernel<T, 256>), grid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((grad_kernel<T, 1024>), grid, dim3(1024), 0, s, a);
        } else if (!(cached(Int<64>{}, Int<4>{}) || cached(Int<256>{}, Int<8>{}) || cached(Int<1024>{}, Int<4>{}) ||
                     cached(Int<1024>{}, Int<8>{}) || cached(Int<1024>{}, Int<12>{}) || cached(Int<1024>{}, Int<16>{}) ||
                     cached(Int<1024>{}, Int<20>{}))) {
            hipLaunchKernelGGL((cached_kernel<T, 1024, 12, MODE, true>), grid, dim3(1024), 0, s, a);
        }
        if (int rc = launched("policy_loss")) return rc;
    }
    return 0;
}

int check(const mgopt_policy_args* p, const char* what) {
    const std::string w(what);
    if (!p) return set_error(MGOPT_E_INVALID, w + ": NULL arguments");
    if (!known_dtype(p->dtype)) return set_error(MGOPT_E_INVALID, w + ": bad dtype");
    if (p->rows < 0 || p->vocab < 1) return set_error(MGOPT_E_INVALID, w + ": need rows >= 0 and vocab >= 1");
    if (p->target_bytes != 4 && p->target_bytes != 8) return set_error(MGOPT_E_INVALID, w + ": targets have 4 or 8 bytes");
    if (p->mask_kind < MGOPT_MASK_NONE || p->mask_kind > MGOPT_MASK_F32) return set_error(MGOPT_E_INVALID, w + ": bad mask kind");
    if (!(p->temperature >= 0x1p-120 && p->temperature <= 0x1p120))  // log2(e) / T is a normal 32-bit number
        return set_error(MGOPT_E_INVALID, w + ": the temperature must lie between 2^-120 and 2^120");
    if (p->workspace_dev && reinterpret_cast<uintptr_t>(p->workspace_dev) % 16 != 0)
        return set_error(MGOPT_E_ALIGN, w + ": the workspace must be 16-byte aligned");
    if (p->rows > 0 && (!p->logits_dev || !p->targets_dev || !p->log_probs_dev))
        return set_error(MGOPT_E_INVALID, w + ": NULL argument");
    if ((p->mask_kind != MGOPT_MASK_NONE) != (p->mask_dev != nullptr) && p->rows > 0)
        return set_error(MGOPT_E_INVALID, w + ": mask and mask kind disagree");
    return 0;
}

// What the loss needs beyond the log-probabilities.
int check_loss(const mgopt_policy_args* p, const char* what) {
    if (int rc = check(p, what)) return rc;
    const std::string w(what);
    if (!(p->clip_low >= 0.0) || !(p->clip_high >= 0.0)) return set_error(MGOPT_E_INVALID, w + ": negative clip range");
    if (!p->workspace_dev) return set_error(MGOPT_E_ALIGN, w + ": no workspace");
    if (p->rows > 0 && (!p->old_logp_dev || !p->advantages_dev)) return set_error(MGOPT_E_INVALID, w + ": NULL argument");
    return 0;
}

PolicyArgs args_of(const mgopt_policy_args* p) {
    PolicyArgs a{};
    a.logits = p->logits_dev, a.row_stride = p->logits_stride, a.rows = p->rows, a.vocab = p->vocab;
    a.targets = p->targets_dev, a.target_bytes = p->target_bytes, a.mask_kind = p->mask_kind, a.mask = p->mask_dev;
    a.old_logp = p->old_logp_dev, a.ref_logp = p->ref_logp_dev, a.advantages = p->advantages_dev;
    a.low = 1.0 - p->clip_low, a.high = 1.0 + p->clip_high, a.kl_coef = p->kl_coef;
    a.inv_temp = 1.0 / p->temperature, a.c = static_cast<float>(1.4426950408889634 / p->temperature);
    a.grad_scale = p->grad_scale_dev, a.log_probs = p->log_probs_dev;
    a.d_logits = p->d_logits_dev, a.d_stride = p->d_logits_stride;
    // workspace: the sum of the weights, then the rows' terms, then what a backward pass needs of them, then the slices'
    // m and s and the targets' logits
    char* at = static_cast<char*>(p->workspace_dev);
    if (at != nullptr) {
        a.weight_sum = p->mask_kind == MGOPT_MASK_NONE ? nullptr : reinterpret_cast<const double*>(at);
        a.terms = reinterpret_cast<float4*>(at + 16);
        a.stats = reinterpret_cast<RowStats*>(at + 16 + 16 * p->rows);
        a.parts = reinterpret_cast<float2*>(at + 16 + 32 * p->rows);
        a.picked = reinterpret_cast<float*>(a.parts + kSplitSlices);
    }
    return a;
}

}  // namespace
}  // namespace mgopt

using namespace mgopt;

extern "C" {

MGOPT_API int64_t mgopt_policy_workspace(int64_t rows) {
    // as args_of lays it out; few rows may be cut in slices
    const int64_t cuts = rows < kSplitRows ? 8 * kSplitSlices + 4 * kSplitRows : 0;
    return rows < 0 ? -1 : 16 + 32 * rows + cuts;
}

MGOPT_API int mgopt_token_log_probs(const mgopt_policy_args* p, void* stream) {
    if (int rc = check(p, "token_log_probs")) return rc;
    if (p->rows == 0) return 0;
    return with_dtype(p->dtype, [&](auto t) {
        return launch_rows<decltype(t), kLogp>(args_of(p), static_cast<hipStream_t>(stream));
    });
}

MGOPT_API int mgopt_policy_loss(const mgopt_policy_args* p, float* loss_dev, float* parts_dev, void* stream) {
    if (int rc = check_loss(p, "policy_loss")) return rc;
    if (!loss_dev || !parts_dev) return set_error(MGOPT_E_INVALID, "policy_loss: NULL argument");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const PolicyArgs a = args_of(p);
    if (a.weight_sum != nullptr) {
        hipLaunchKernelGGL(weight_sum_kernel, dim3(1), dim3(kSumBlock), 0, s, a.mask, a.mask_kind, a.rows,
                           static_cast<double*>(p->workspace_dev));
        if (int rc = launched("weight_sum_kernel")) return rc;
    }
    if (p->rows > 0) {
        const int rc = with_dtype(p->dtype, [&](auto t) {
            using T = decltype(t);
            return a.d_logits != nullptr ? launch_rows<T, kLossGrad>(a, s) : launch_rows<T, kLoss>(a, s);
        });
        if (rc) return rc;
    }
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(kSumBlock), 0, s, a.terms, a.rows, a.weight_sum, a.kl_coef, loss_dev,
                       parts_dev);
    return launched("policy_sum_kernel");
}

MGOPT_API int mgopt_policy_loss_backward(const mgopt_policy_args* p, void* stream) {
    if (int rc = check_loss(p, "policy_loss_backward")) return rc;
    if (p->rows == 0) return 0;
    if (!p->d_logits_dev) return set_error(MGOPT_E_INVALID, "policy_loss_backward: NULL argument");
    return with_dtype(p->dtype, [&](auto t) {
        return launch_rows<decltype(t), kGrad>(args_of(p), static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
