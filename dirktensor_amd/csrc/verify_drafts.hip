// Drafted tokens verified against a model's probabilities, from given random numbers.
//
// For batch row b with n drafted tokens x_1 .. x_n, the model's probabilities p_i = softmax(logits_i / T) of the i-th next token
// (i = 1 .. n + 1) and those that the drafts were drawn from, q_i = softmax(draft_i / T) (or 1 at the draft, where there are no
// draft logits): draft i is accepted, if those before it were, while u_i q_i(x_i) < p_i(x_i). One more token follows the
// accepted ones, drawn with the random number u: the first j with sum_{k <= j} w_k > u sum_k w_k, where
//   w = max(p_i - q_i, 0)  behind a refused draft i (p_i itself, should that leave nothing), so that what is emitted is distributed as p
//   w = p_{n+1}            where all were accepted.
// At T = 0 a draft is accepted where it is the largest logit's token (the first of equals), and that token is the one that follows.
//
// A token is one side of a border or the other, and there are as many borders as tokens in the vocabulary: weights that are off by
// 2^-24 of their probability would give another token about once in a few hundred calls. So the weights and their sums are held in
// 64 bits, the terms to 10^-13. The rows' sums that decide on drafts (one border each) are of terms in 32 bits, summed in 64; the largest
// term is exact, so the log probability of a token that is almost certain is, too.
//
// Work: every row is read once for its sum (first kernel: a row in segments, as many as fill the CUs), and the one or two rows that the
// weights come from once more, mostly from the caches (second kernel: each workgroup works out from the first kernel's sums which draft
// was refused, and its waves take chunks of 512 values). The weights' difference needs the ratio of both rows' sums, which is known
// to 32 bits only: a chunk leaves sum (p' - ratio q') and sum q' over the values where that is above 0 (p', q': the powers, not divided
// by their sums), and sum p' and sum q' over all; the last workgroup of a batch row to be done has the ratio to 64 bits then and
// corrects the chunks' weights by it. What that leaves wrong are values whose sign the first ratio got wrong, each by the ratio's error
// times q' at most. These are among the values with |p' - ratio q'| < kClose p' (the ratio's error, 10^-8 as a rule, is compared with
// half of kClose), which are rare, and their q' are summed, too: where the ratio's error times that sum exceeds kSlack of the row's sum, as it
// does for rows that agree almost everywhere, that workgroup sums the weights again (90 us more at 100352 values, 200 for 64 such
// rows). So a border is off by 3 10^-12 of the row's sum at most, whatever the total of the weights. Last it finds the chunk that the
// border lies in, and in it the token.
//
// Measured at 100352 logits a row: 4 drafts of one sequence in fp32, 3.6 MB, 4.4 and 9.9 us in the two kernels: chains of one batch and of
// one chunk, with six trips to memory in the second (the partial sums, a chunk, its sums out, the count, the sums in, the border's chunk),
// of about 2.2, 2.5, 0.6, 1.1 and 1.5 us with what is done between them; without draft logits 3.9 and 8.5, at temperature 0 5.0 and 4.2. Up to 5
// drafts of 64 sequences in bf16, 72 MB, 21.2 and 20.4: the first is 3.4 TB/s (where all have 5, 141 MB, 29.4, 4.8 TB/s: half of the workgroups
// have nothing to do where drafts are ragged, and the others share the CUs unevenly), with 26 cycles a value and wave for the powers and
// sums beside the reads; the second has the 64 bits' arithmetic, 7 us a workgroup at the median and 12 where a CU's workgroups all
// have two rows, and the chain around it. (26 with powers by a longer polynomial in place of the table, the next chunk's loads not
// ahead, the counts in one cache line and 13 workgroups a batch row.)
// Without draft logits 18.8 and 15.0, without drafts 8.4 and 14.8, at temperature 0 22.8 and 4.0.

#include "dt_internal.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace dt {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kFewRows = 32;
constexpr int kMaxDrafts = 64;
constexpr int kMaxRows = 2 * kMaxDrafts + 1;  // of a batch row
constexpr int kMaxVocab = 1 << 24;
constexpr int kChunk = 512;                   // values that a wave of the second kernel takes at a time: 8 a lane
constexpr int kWhole = 4096;                  // of a batch of the first kernel, all threads
constexpr int kMinSegment = 2048;             // values of a segment of the first kernel at least
constexpr int kFill = 2048;                   // workgroups that the first kernel aims at, eight a CU
constexpr int kDrawFill = 1280;               // and the second: five a CU (64 sequences 21.4 us, 23.2 with 832, 22.5 with 1600)
constexpr int kCountStride = 64;              // a cache line and more: counts of one line wait for each other
constexpr double kClose = 0x1p-20, kSlack = 0x1p-40;
constexpr double kCloseUnit = 0x1p-38;        // of the sum of close values' q', which is 2^24 at most: whole units add up alike in any order
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kFar = -1100.0;              // (2^-1100 is none of 64 bits)
constexpr float kLowest = -3.402823466e38f;

template <int kRows>
struct VerifyArgs {
    const void* x;        // logits
    const void* y;        // draft logits, or NULL
    const void* drafts;   // [B, K]
    const float* u;       // [B, K + 1]
    int32_t* accepted;    // [B]
    int32_t* tokens;      // [B, K + 1]
    float* logprob;       // [B, K + 1]
    int32_t* count;       // [B], kCountStride apart: workgroups of the second kernel that are done; 8 bytes behind it the sum of close values' q'
    double2* part;        // [B][rows][segments]: the largest logit, and the sum of 2^(c (x - it))
    float2* best;         // [B][K + 1][segments] at T = 0: the largest logit, its index (as bits)
    float* picked;        // [B][rows]: the draft's logit
    double* sums;         // [B][chunks][4]: sum of p' - ratio q' and of q' where that is above 0, of p' and of q'
    int64_t ldb_x, ldt_x, ldb_y, ldt_y;
    double c;             // log2(e) / T
    float c_hi, c_lo;     // in two parts, both above 0 (a logit of -inf times either is -inf)
    int K, V, tok_bytes;
    int rows;             // of a batch row: K + 1, and K of the drafts
    int segments, segment;  // of the first kernel, values of one
    int chunks, runs;     // of the second, at most one a thread; a chunk has so many times kChunk values
    uint8_t n[kRows];     // drafts of each batch row
};

// 2^t to 1.1 10^-12 for t <= 1000, 0 for t <= kFar (and for NaN). (2^f on [-1/2, 1/2] as its interpolation in nine Chebyshev points.)
__device__ __forceinline__ double exp2_64(double t) {
    t = fmax(t, kFar);
    constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are the nearest whole number
    const double m = t + kMagic;
    const double f = t - (m - kMagic);
    double v = 0x1.63d136366db24p-20;
    v = fma(v, f, 0x1.00dc4a532fb8ep-16);
    v = fma(v, f, 0x1.4308ac85aa947p-13);
    v = fma(v, f, 0x1.5d8745a728441p-10);
    v = fma(v, f, 0x1.3b2ab7181b755p-7);
    v = fma(v, f, 0x1.c6b08dd6fd234p-5);
    v = fma(v, f, 0x1.ebfbdff823cedp-3);
    v = fma(v, f, 0x1.62e42fef84cf0p-1);
    v = fma(v, f, 1.0);
    return __builtin_amdgcn_ldexp(v, static_cast<int>(__double_as_longlong(m)));
}

// The same for many of them, 2^(t/32): 2^(j/32) from a table, and 2^(f/32) on [-1/2, 1/2] as its interpolation in five points, to 10^-13.
// The table lies in LDS, an entry in two of the 64 banks, so lanes read it without conflicts.
constexpr int kRoots = 32;
__device__ const double kRootsOfTwo[kRoots] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};
__device__ __forceinline__ double exp2_64(double t, const double* roots) {
    t = fmax(t, kRoots * kFar);
    constexpr double kMagic = 6755399441055744.0;
    const double m = t + kMagic;
    const double f = t - (m - kMagic);
    const int i = static_cast<int>(__double_as_longlong(m));
    double v = 0x1.3b2b1bee88b09p-27;
    v = fma(v, f, 0x1.c6b167e571135p-20);
    v = fma(v, f, 0x1.ebfbdff8131c3p-13);
    v = fma(v, f, 0x1.62e42fef6d01ap-6);
    v = fma(v, f, 1.0);
    return __builtin_amdgcn_ldexp(v * roots[i & (kRoots - 1)], i >> 5);
}

template <bool kBf16>
constexpr int kPer = kBf16 ? 8 : 4;  // values of a 16-byte piece

template <bool kBf16>
__device__ __forceinline__ float load_one(const void* row, int at) {
    if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[at]) << 16);
    else return static_cast<const float*>(row)[at];
}
// the values at..at+15 bytes of a row; with fewer than a whole piece left, one by one (and -inf behind the end)
template <bool kBf16>
__device__ __forceinline__ void load_piece(const void* row, int at, int end, float (&x)[kPer<kBf16>]) {
    if (at + kPer<kBf16> <= end) {
        if constexpr (kBf16) {
            const u32x4 w = *reinterpret_cast<const u32x4_at2*>(static_cast<const uint16_t*>(row) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const u32x4 w = *reinterpret_cast<const u32x4_at4*>(static_cast<const float*>(row) + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kPer<kBf16>; ++i) x[i] = -__builtin_huge_valf();
    if (at < end) {  // (all loads at once)
#pragma unroll
        for (int i = 0; i < kPer<kBf16>; ++i) {
            const float v = load_one<kBf16>(row, min(at + i, end - 1));
            if (at + i < end) x[i] = v;
        }
    }
}

// row r of a batch row: the model's (r <= K) or the drafts'
template <bool kBf16, int kRows>
__device__ __forceinline__ const void* row_of(const VerifyArgs<kRows>& a, int b, int r) {
    const int64_t at = r <= a.K ? b * a.ldb_x + r * a.ldt_x : b * a.ldb_y + (r - a.K - 1) * a.ldt_y;
    return static_cast<const char*>(r <= a.K ? a.x : a.y) + at * (kBf16 ? 2 : 4);
}

// Sums over a wave without LDS: within 16 lanes by data-parallel moves, across by permutes of halves.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double moved(double x) {  // (0 from lanes that are none, in rows that are masked)
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), kCtrl, kRowMask, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), kCtrl, kRowMask, 0xf, false);
    return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo));
}
__device__ __forceinline__ double sum16(double x) {
    x += moved<0xb1, 0xf>(x);   // the neighbour
    x += moved<0x4e, 0xf>(x);   // the other pair of four
    x += moved<0x141, 0xf>(x);  // mirrored within 8
    return x + moved<0x140, 0xf>(x);  // and within 16
}
template <int kCtrl>
__device__ __forceinline__ float moved32(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, static_cast<int>(__float_as_uint(x)), kCtrl, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float x) {
    x = fmaxf(x, moved32<0xb1>(x));
    x = fmaxf(x, moved32<0x4e>(x));
    x = fmaxf(x, moved32<0x141>(x));
    return fmaxf(x, moved32<0x140>(x));
}
template <bool k32>
__device__ __forceinline__ double sum_halves(double x) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
    const uint32_t l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
    const auto lo = k32 ? __builtin_amdgcn_permlane32_swap(l, l, false, false) : __builtin_amdgcn_permlane16_swap(l, l, false, false);
    const auto hi = k32 ? __builtin_amdgcn_permlane32_swap(h, h, false, false) : __builtin_amdgcn_permlane16_swap(h, h, false, false);
    const auto join = [](uint32_t a, uint32_t b) { return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(b) << 32 | a)); };
    return join(lo[0], hi[0]) + join(lo[1], hi[1]);
}
__device__ __forceinline__ double sum_wave(double x) { return sum_halves<true>(sum_halves<false>(sum16(x))); }
// Four sums at once, sum (lane & 1) * 2 + (lane >> 1 & 1) in each lane: two steps leave a lane one of four values, which the others then add up.
__device__ __forceinline__ double sum_four(double a, double b, double c, double d) {
    const int lane = threadIdx.x;
    const bool odd = lane & 1, upper = lane & 2;
    const double x = (odd ? c : a) + moved<0xb1, 0xf>(odd ? a : c), y = (odd ? d : b) + moved<0xb1, 0xf>(odd ? b : d);
    double s = (upper ? y : x) + moved<0x4e, 0xf>(upper ? x : y);
    s += moved<0x124, 0xf>(s);  // from 4 lanes away, of 16
    s += moved<0x128, 0xf>(s);  // and from 8
    return sum_halves<true>(sum_halves<false>(s));
}
// the sums of a lane's and all lower lanes' values
__device__ __forceinline__ double scan_wave(double x) {
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);  // the last lane of a row of 16 to the next, of 32 to the other half
    return x + moved<0x143, 0xc>(x);
}

// kPieces whole pieces of a thread, and their values
template <bool kBf16, int kN>
__device__ __forceinline__ void load_batch(const void* row, int at, u32x4 (&w)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const int to = at + i * kThreads * kPer<kBf16>;
        if constexpr (kBf16) w[i] = *reinterpret_cast<const u32x4_at2*>(static_cast<const uint16_t*>(row) + to);
        else w[i] = *reinterpret_cast<const u32x4_at4*>(static_cast<const float*>(row) + to);
    }
}
template <bool kBf16, int kN>
__device__ __forceinline__ void open_batch(const u32x4 (&w)[kN], float (&x)[kN][kPer<kBf16>]) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kBf16) x[i][2 * j] = __uint_as_float(w[i][j] << 16), x[i][2 * j + 1] = __uint_as_float(w[i][j] & 0xffff0000u);
            else x[i][j] = __uint_as_float(w[i][j]);
        }
}

// 2^(c d) in 32 bits, for d <= 0
template <int kRows>
__device__ __forceinline__ float power(const VerifyArgs<kRows>& a, float d) {
    return __builtin_amdgcn_exp2f(fmaf(d, a.c_hi, d * a.c_lo));
}
template <int kRows>
__device__ __forceinline__ int draft_of(const VerifyArgs<kRows>& a, int b, int i) {
    const int64_t at = static_cast<int64_t>(b) * a.K + i;
    if (a.tok_bytes == 4) return static_cast<const int32_t*>(a.drafts)[at];
    const int64_t t = static_cast<const int64_t*>(a.drafts)[at];
    return t < 0 || t >= a.V ? -1 : static_cast<int>(t);
}

template <int kRows>
__device__ __forceinline__ unsigned long long* close_sum(const VerifyArgs<kRows>& a, int b) {
    return reinterpret_cast<unsigned long long*>(a.count + b * kCountStride + 2);
}

template <bool kBf16, bool kGreedy, int kRows>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs<kRows> a) {
    constexpr int P = kPer<kBf16>;
    constexpr int kPieces = kBf16 ? 2 : 4;  // under way at once
    __shared__ double red[kWaves];
    __shared__ float red_top[kWaves];
    __shared__ float2 red_best[kWaves];
    const int b = blockIdx.z, r = blockIdx.y, seg = blockIdx.x, n = a.n[b];
    if (seg == 0 && r == 0 && threadIdx.x == 0) a.count[b * kCountStride] = 0, *close_sum(a, b) = 0;
    if (r <= a.K ? r > n : r - a.K - 1 >= n) return;
    const void* row = row_of<kBf16>(a, b, r);
    // the draft's logit, for the second kernel (in the last segment, which may be the shortest)
    const int i = r <= a.K ? r : r - a.K - 1;
    if (seg == a.segments - 1 && threadIdx.x == kThreads - 1 && i < n) {
        const int draft = draft_of(a, b, i);
        a.picked[b * a.rows + r] = draft >= 0 && draft < a.V ? load_one<kBf16>(row, draft) : 0.0f;
    }
    const int from = seg * a.segment, end = min(a.V, from + a.segment);
    float top = kLowest, best = -__builtin_huge_valf();
    double sum = 0.0;
    int best_at = from;
    constexpr int kBatch = kPieces * kThreads * P;
    static_assert(kBatch == kWhole, "segments of whole batches");
    const auto take = [&](const float (&x)[kPieces][P], int at) {
        float most = top;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                most = fmaxf(most, x[i][j]);
                if (kGreedy && x[i][j] > best) best = x[i][j], best_at = at + i * kThreads * P + j;
            }
        sum *= exp2_64((static_cast<double>(top) - most) * a.c);
        top = most;
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) sum += static_cast<double>(power(a, x[i][j] - top));
    };
    // whole batches, two under way (the last ones are loaded twice, from the caches: a load under a condition would make every wait one
    // for all loads); then what is left
    int at = from + static_cast<int>(threadIdx.x) * P;
    const int whole = (end - from) / kBatch;
    if (whole > 0) {
        u32x4 w[2][kPieces];
        const auto load = [&](int i, u32x4 (&to)[kPieces]) { load_batch<kBf16>(row, at + min(i, whole - 1) * kBatch, to); };
        const auto use = [&](int i, u32x4 (&of)[kPieces]) {
            float x[kPieces][P];
            open_batch<kBf16>(of, x);
            take(x, at + i * kBatch);
        };
        load(0, w[0]);
        load(1, w[1]);
        int i = 0;
        for (; i + 1 < whole; i += 2) {
            use(i, w[0]);
            load(i + 2, w[0]);
            use(i + 1, w[1]);
            load(i + 3, w[1]);
        }
        if (i < whole) use(i, w[0]);
        at += whole * kBatch;
    }
    if (whole * kBatch < end - from) {
        float x[kPieces][P];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) load_piece<kBf16>(row, at + i * kThreads * P, end, x[i]);
        take(x, at);
    }
    // the threads' sums meet: brought to the largest logit of all, each by one factor
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float most = top;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        most = fmaxf(most, __shfl_xor(most, o, 64));
        if constexpr (kGreedy) {
            const float t2 = __shfl_xor(best, o, 64);
            const int a2 = __shfl_xor(best_at, o, 64);
            if (t2 > best || (t2 == best && a2 < best_at)) best = t2, best_at = a2;
        }
    }
    if (lane == 0) {
        red_top[wave] = most;
        if constexpr (kGreedy) red_best[wave] = make_float2(best, __int_as_float(best_at));
    }
    __syncthreads();
    most = fmaxf(fmaxf(red_top[0], red_top[1]), fmaxf(red_top[2], red_top[3]));
    sum = sum_wave(sum * exp2_64((static_cast<double>(top) - most) * a.c));
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    if (threadIdx.x != 0) return;
    sum = red[0] + red[1] + red[2] + red[3];
    a.part[(static_cast<int64_t>(b) * a.rows + r) * a.segments + seg] = make_double2(most, sum);
    if constexpr (kGreedy) {
#pragma unroll
        for (int i = 1; i < kWaves; ++i) {
            const float t2 = red_best[i].x;
            const int a2 = __float_as_int(red_best[i].y);
            if (t2 > best || (t2 == best && a2 < best_at)) best = t2, best_at = a2;
        }
        a.best[(static_cast<int64_t>(b) * (a.K + 1) + r) * a.segments + seg] = make_float2(best, __int_as_float(best_at));
    }
}

// sums before a thread's own of the workgroup's, in the threads' order, and of all
__device__ __forceinline__ double scan(double v, double (&red)[kWaves], double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double s = scan_wave(v);
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    double base = 0.0, sum = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i < wave) base += red[i];
        sum += red[i];
    }
    *all = sum;
    return base + (s - v);
}

__device__ __forceinline__ double sum_all(double v, double (&red)[kWaves]) {
    v = sum_wave(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) s += red[i];
    return s;
}

// log2 of a sum, at least 1: the instruction's, once corrected
__device__ __forceinline__ double log2_64(double s) {
    const double y = static_cast<double>(__builtin_amdgcn_logf(static_cast<float>(s)));
    return y + (s * exp2_64(-y) - 1.0) * kLog2e;
}

// 8 values of a row as they lie there, which the loop over them takes in four pairs: a kernel that runs once through its code waits for the
// code, too, so that loop is not unrolled.
template <bool kBf16>
struct Eight {
    static constexpr int kWords = kBf16 ? 4 : 8;
    uint32_t w[kWords];
    // whole: none of the wave's values lie behind the row's end (these are -inf). Nothing is done with a whole one's words here, so the
    // loads stay under way.
    __device__ __forceinline__ void load(const void* row, int at, int end, bool whole) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                u32x4 v;
                if constexpr (kBf16) v = *reinterpret_cast<const u32x4_at2*>(static_cast<const uint16_t*>(row) + at);
                else v = *reinterpret_cast<const u32x4_at4*>(static_cast<const float*>(row) + at + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const auto one = [&](int to) {
                const float v = load_one<kBf16>(row, min(to, end - 1));
                return to < end ? __float_as_uint(v) : 0xff800000u;
            };
            if constexpr (kBf16) w[i] = one(at + 2 * i) >> 16 | one(at + 2 * i + 1);
            else w[i] = one(at + i);
        }
    }
    __device__ __forceinline__ void hide(int i) {  // value i, if it is one of these, has no weight
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j == i) {
                if constexpr (kBf16) w[j >> 1] = j & 1 ? (w[j >> 1] & 0xffffu) | 0xff800000u : (w[j >> 1] & 0xffff0000u) | 0xff80u;
                else w[j] = 0xff800000u;
            }
    }
    __device__ __forceinline__ float lo() const { return __uint_as_float(kBf16 ? w[0] << 16 : w[0]); }
    __device__ __forceinline__ float hi() const { return __uint_as_float(kBf16 ? w[0] & 0xffff0000u : w[1]); }
    __device__ __forceinline__ void next() {
        constexpr int kBy = kBf16 ? 1 : 2;
#pragma unroll
        for (int i = 0; i + kBy < kWords; ++i) w[i] = w[i + kBy];
    }
};
// The two rows that the weights come from: p', and q', 0 where there is no such row.
struct Rows {
    const void *px, *qx;  // qx: or NULL
    const double* roots;
    double p_top, q_top, c;  // c: times kRoots
    __device__ __forceinline__ double p(float x) const { return exp2_64((static_cast<double>(x) - p_top) * c, roots); }
    __device__ __forceinline__ double q(float y) const { return exp2_64((static_cast<double>(y) - q_top) * c, roots); }
};

template <bool kBf16, bool kGreedy, int kRows>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs<kRows> a) {
    __shared__ double roots[kRoots];
    __shared__ float tops[kMaxRows];
    __shared__ double sums[kMaxRows];  // NaN of a row that has none
    __shared__ int best[kMaxDrafts + 1];
    __shared__ float draft_x[kMaxDrafts];
    __shared__ int drafts[kMaxDrafts];
    __shared__ double red[kWaves];
    __shared__ double sh_before;
    __shared__ int sh_over[kWaves], sh_some[kWaves];
    __shared__ int sh_accepted, sh_last, sh_token;
    __shared__ float sh_logit;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = a.n[b], K = a.K, V = a.V;

    // the drafts' logits, while the rows' sums are joined: 16 lanes a row
    int draft = -1;
    float x = 0.0f, y = 0.0f, u = 0.0f;
    if (tid < n) {
        draft = draft_of(a, b, tid);
        if (!kGreedy) u = a.u[static_cast<int64_t>(b) * (K + 1) + tid];
        x = a.picked[b * a.rows + tid];
        if (a.y) y = a.picked[b * a.rows + K + 1 + tid];
    }
    if (!kGreedy && tid >= kThreads - kRoots) roots[tid - (kThreads - kRoots)] = kRootsOfTwo[tid - (kThreads - kRoots)];
    const double last_u = kGreedy ? 0.0 : a.u[static_cast<int64_t>(b) * (K + 1) + K];
    const int own_rows = n + 1 + (a.y ? n : 0);
    for (int i = tid >> 4; i < own_rows; i += kThreads / 16) {
        const int r = i <= n ? i : K + 1 + (i - n - 1);
        const double2* p = a.part + (static_cast<int64_t>(b) * a.rows + r) * a.segments;
        // The largest logit first (four of a lane's segments at a time; rows of more are read twice), then the sum brought to it.
        float to = kLowest, most = -__builtin_huge_valf();
        double2 v[4];
        int most_at = 0;
        const auto load = [&](int first) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s = first + 16 * j + (tid & 15);
                v[j] = s < a.segments ? p[s] : make_double2(kLowest, 0.0);
            }
        };
        for (int first = 0; first < a.segments; first += 64) {
            load(first);
#pragma unroll
            for (int j = 0; j < 4; ++j) to = fmaxf(to, static_cast<float>(v[j].x));
            if constexpr (kGreedy) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int s = first + 16 * j + (tid & 15);
                    if (s >= a.segments) continue;
                    const float2 w = a.best[(static_cast<int64_t>(b) * (K + 1) + r) * a.segments + s];
                    if (w.x > most) most = w.x, most_at = __float_as_int(w.y);
                }
            }
        }
        to = max16(to);
        if constexpr (kGreedy) {
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) {
                const float t2 = __shfl_xor(most, o, 16);
                const int a2 = __shfl_xor(most_at, o, 16);
                if (t2 > most || (t2 == most && a2 < most_at)) most = t2, most_at = a2;
            }
        }
        double sum = 0.0;
#pragma unroll 1
        for (int first = 0; first < a.segments; first += 64) {
            if (a.segments > 64) load(first);
#pragma unroll 1
            for (int s = first; s < min(first + 64, a.segments); s += 16) {  // (not unrolled, as below)
                sum += v[0].y * exp2_64((v[0].x - to) * a.c);
                v[0] = v[1], v[1] = v[2], v[2] = v[3];
            }
        }
        sum = sum16(sum);
        if ((tid & 15) == 0) {
            tops[r] = to;
            sums[r] = sum > 0.0 ? sum : __builtin_nan("");
            if (kGreedy) best[i] = sum > 0.0 ? most_at : -1;
        }
    }
    __syncthreads();
    if (wave == 0) {
        bool ok = false;
        if (tid < n) {
            if (draft >= 0 && draft < V) {
                if (kGreedy) ok = draft == best[tid];
                else {
                    // u q < p, times both sums
                    const double p = exp2_64((static_cast<double>(x) - tops[tid]) * a.c);
                    double q = u * sums[tid];
                    if (a.y) q *= exp2_64((static_cast<double>(y) - tops[K + 1 + tid]) * a.c);
                    ok = q < (a.y ? p * sums[K + 1 + tid] : p);
                }
            }
            drafts[tid] = draft;
            draft_x[tid] = x;
        }
        const uint64_t yes = __ballot(ok);
        if (tid == 0) sh_accepted = yes == ~0ull ? 64 : __builtin_ctzll(~yes);
    }
    __syncthreads();
    const int acc = sh_accepted;
    int token = -1;    // the one that follows
    double sum = sums[acc];
    if constexpr (kGreedy) {
        token = best[acc];
    } else {
        const bool refused = acc < n;
        Rows rows{row_of<kBf16>(a, b, acc), refused && a.y ? row_of<kBf16>(a, b, K + 1 + acc) : nullptr, roots, tops[acc], 0.0, kRoots * a.c};
        const int skip = refused && !a.y ? drafts[acc] : -1;  // a draft that nothing was drawn for
        double near = 0.0;  // the ratio of the rows' sums, to 32 bits
        if (rows.qx) {
            rows.q_top = tops[K + 1 + acc];
            near = sums[acc] / sums[K + 1 + acc];
        }
        const bool none = !(sum > 0.0) || !(near >= 0.0);  // a row that is none (the same for all of the batch row's workgroups)
        if (none && blockIdx.x > 0) return;
        double* out = a.sums + static_cast<int64_t>(b) * a.chunks * 4;
        double h[4], p_sum = 0.0, ratio = 0.0, weight, before, all;
        int first = blockIdx.x * kWaves + wave, step = gridDim.x * kWaves;
        for (bool again = false; !none; again = true) {
            // Runs of kChunk values, the next one's under way while one is summed; behind a chunk's last its sums go out.
            Eight<kBf16> px{}, qx{};
            double pw = 0.0, qw = 0.0, pa = 0.0, qa = 0.0, close = 0.0;
            int chunk = first, run = 0, at = 0, of = 0;
            bool more = false, last = false;
#pragma clang loop unroll(disable)
            do {
                Eight<kBf16> x = px, y = qx;
                const bool some = more, ends = last;
                const int base = at, to = of;
                more = chunk < a.chunks;
                if (more) {
                    of = chunk;
                    at = (chunk * a.runs + run) * kChunk;
                    last = ++run == a.runs;
                    if (last) run = 0, chunk += step;
                    const bool whole = at + kChunk <= V;
                    px.load(rows.px, at + lane * 8, V, whole);
                    if (rows.qx) qx.load(rows.qx, at + lane * 8, V, whole);
                }
                if (some) {
                    if (static_cast<uint32_t>(skip - base) < kChunk) x.hide(skip - base - lane * 8);  // (the same for the whole wave)
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        if (rows.qx) {  // (both branches whole: the powers' chains then go side by side)
                            const double p[2] = {rows.p(x.lo()), rows.p(x.hi())}, q[2] = {rows.q(y.lo()), rows.q(y.hi())};
                            bool some_close = false;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const double w = fma(-near, q[j], p[j]);
                                pa += p[j];
                                qa += q[j];
                                pw += fmax(w, 0.0);
                                qw += w > 0.0 ? q[j] : 0.0;
                                some_close |= fabs(w) < kClose * p[j];
                            }
                            if (__builtin_expect(some_close, 0))
#pragma unroll
                                for (int j = 0; j < 2; ++j) close += fabs(fma(-near, q[j], p[j])) < kClose * p[j] ? q[j] : 0.0;
                            y.next();
                        } else {
                            const double p0 = rows.p(x.lo()), p1 = rows.p(x.hi());
                            pa += p0;
                            pa += p1;
                        }
                        x.next();
                    }
                    if (ends) {
                        const double s = sum_four(pw, qw, pa, qa);
                        if (lane < 4)  // through to the memory that all XCDs see
                            __hip_atomic_store(out + to * 4 + (lane & 1) * 2 + (lane >> 1), s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        pw = qw = pa = qa = 0.0;
                        if (!again && __any(close > 0.0)) {
                            const double c = ceil(sum_wave(close) / kCloseUnit);
                            if (lane == 0)
                                __hip_atomic_fetch_add(close_sum(a, b), static_cast<unsigned long long>(c), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                            close = 0.0;
                        }
                    }
                }
            } while (more);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // and complete before they are counted
            __syncthreads();
            if (!again) {
                if (tid == 0)
                    sh_last = __hip_atomic_fetch_add(a.count + b * kCountStride, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == static_cast<int>(gridDim.x) - 1;
                __syncthreads();
                if (!sh_last) return;
            }
            // the last workgroup: thread i has chunk i
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = tid < a.chunks ? __hip_atomic_load(out + tid * 4 + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
            if (!again) {
                p_sum = sum_all(h[2], red);
                if (rows.qx) ratio = p_sum / sum_all(h[3], red);
            }
            weight = rows.qx ? fmax(h[0] - (ratio - near) * h[1], 0.0) : h[2];
            before = scan(weight, red, &all);
            if (again || !rows.qx) break;  // (these are the same for the whole workgroup)
            const double off = fabs(ratio - near);
            const double close_q = static_cast<double>(__hip_atomic_load(close_sum(a, b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) * kCloseUnit;
            if (off <= 0.5 * kClose * near && off * close_q <= kSlack * p_sum) break;
            near = ratio;
            first = wave, step = kWaves;
        }
        if (!none && all == 0.0 && rows.qx) {  // nothing is left: p itself
            rows.qx = nullptr;
            ratio = 0.0;
            weight = h[2];
            before = scan(weight, red, &all);
        }
        if (skip < 0) sum = p_sum;
        if (!none && all > 0.0) {
            const double bound = last_u * all;
            // the first thread whose sum passes the border; where rounding leaves none, the last that has a weight (none: -1)
            bool passed = false;
            const auto first_over = [&](bool over, bool some) {
                const uint64_t o = __ballot(over), w = __ballot(some);
                if (lane == 0) {
                    sh_over[wave] = o ? wave * 64 + __builtin_ctzll(o) : kThreads;
                    sh_some[wave] = w ? wave * 64 + 63 - __builtin_clzll(w) : -1;
                }
                __syncthreads();
                const int f = min(min(sh_over[0], sh_over[1]), min(sh_over[2], sh_over[3]));
                passed = f < kThreads;
                return passed ? f : max(max(sh_some[0], sh_some[1]), max(sh_some[2], sh_some[3]));
            };
            const int chunk = first_over(weight > 0.0 && before + weight > bound, weight > 0.0);
            if (tid == chunk) sh_before = before;
            __syncthreads();
            before = sh_before;
            if (tid == 0) sh_token = -1;
            constexpr int kOwn = kChunk / kThreads;  // neighbouring values of a thread
#pragma unroll 1
            for (int run = 0; run < a.runs; ++run) {
                const int at = (chunk * a.runs + run) * kChunk + tid * kOwn;
                float x[kOwn], y[kOwn];
                double w[kOwn], mine = 0.0;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    x[i] = at + i < V ? load_one<kBf16>(rows.px, at + i) : -__builtin_huge_valf();
                    y[i] = rows.qx && at + i < V ? load_one<kBf16>(rows.qx, at + i) : -__builtin_huge_valf();
                    if (at + i == skip) x[i] = -__builtin_huge_valf();
                }
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    w[i] = rows.qx ? fmax(fma(-ratio, rows.q(y[i]), rows.p(x[i])), 0.0) : rows.p(x[i]);
                    mine += w[i];
                }
                double upto = before + scan(mine, red, &all);
                bool over = false, some = false;
                int mine_at = 0;
                float mine_x = 0.0f;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    if (!over && w[i] > 0.0) {
                        some = true;
                        mine_at = at + i;
                        mine_x = x[i];
                        upto += w[i];
                        over = upto > bound;
                    }
                }
                const int found = first_over(over, some);
                if (tid == found) sh_token = mine_at, sh_logit = mine_x;
                before += all;
                __syncthreads();
                if (passed) break;
            }
            token = sh_token;
        }
    }
    // the accepted drafts, the token and their log probabilities, then nothing
    for (int i = tid; i <= K; i += kThreads) {
        const int64_t at = static_cast<int64_t>(b) * (K + 1) + i;
        const int t = i < acc ? drafts[i] : i == acc ? token : -1;
        float lp = 0.0f;
        if (i <= acc) {
            float v = __builtin_nanf("");
            if (i < acc) v = draft_x[i];
            else if (t >= 0) v = kGreedy ? load_one<kBf16>(row_of<kBf16>(a, b, i), t) : sh_logit;
            lp = static_cast<float>(((static_cast<double>(v) - tops[i]) * a.c - log2_64(i < acc ? sums[i] : sum)) * kLn2);
        }
        a.tokens[at] = t;
        a.logprob[at] = lp;
    }
    if (tid == 0) a.accepted[b] = acc;
}

struct Call {
    const void *x, *y, *drafts;
    const float* u;
    int32_t *accepted, *tokens;
    float* logprob;
    int B, K, V;
    int64_t ldb_x, ldt_x, ldb_y, ldt_y;
    int tok_bytes;
    const int32_t* counts;
    double temperature;
    int dtype, mem;
};

struct Plan {
    int rows, segments, segment, chunks, runs, groups;
    int64_t part, best, picked, sums, bytes;  // offsets
};
Plan make_plan(int B, int K, int V, bool drafts, bool greedy) {
    Plan p{};
    p.rows = K + 1 + (drafts && !greedy ? K : 0);
    const int64_t rows = static_cast<int64_t>(B) * p.rows;
    const int most = (V + kMinSegment - 1) / kMinSegment;
    p.segments = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (kFill + rows - 1) / rows)));
    const int batch = V / p.segments >= kWhole ? kWhole : 8;  // (a part of a batch takes as long as a whole one)
    p.segment = ((V + p.segments - 1) / p.segments + batch - 1) / batch * batch;
    p.segments = (V + p.segment - 1) / p.segment;
    p.runs = (V + kChunk * kThreads - 1) / (kChunk * kThreads);
    p.chunks = greedy ? 0 : (V + kChunk * p.runs - 1) / (kChunk * p.runs);
    // a chunk a wave, more where there would be many workgroups
    p.groups = greedy ? 1 : std::min((p.chunks + kWaves - 1) / kWaves, std::max(1, kDrawFill / B));
    p.part = static_cast<int64_t>(B) * kCountStride * 4;
    p.best = p.part + rows * p.segments * 16;
    p.picked = p.best + (greedy ? rows * p.segments * 8 : 0);
    p.sums = p.picked + (rows * 4 + 15) / 16 * 16;
    p.bytes = p.sums + static_cast<int64_t>(B) * p.chunks * 32;
    return p;
}

int check_sizes(int B, int K, int V, double temperature) {
    if (B < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d must be >= 1", B);
    if (B > kMaxRaggedBatch) return set_error(DT_ERR_UNSUPPORTED, "B=%d > %d", B, kMaxRaggedBatch);
    if (K < 0 || K > kMaxDrafts) return set_error(K < 0 ? DT_ERR_INVALID_ARG : DT_ERR_UNSUPPORTED, "K=%d drafts outside [0, %d]", K, kMaxDrafts);
    if (V < 1) return set_error(DT_ERR_INVALID_ARG, "V=%d must be >= 1", V);
    if (V > kMaxVocab) return set_error(DT_ERR_UNSUPPORTED, "V=%d > %d", V, kMaxVocab);
    if (!(temperature == 0.0 || (temperature >= 1e-6 && temperature <= 1e6)))
        return set_error(DT_ERR_INVALID_ARG, "temperature %g must be 0 or from 1e-6 to 1e6", temperature);
    return DT_OK;
}

template <int kRows>
int launch_rows(const Call& c, const Plan& p, void* ws, hipStream_t s) {
    VerifyArgs<kRows> a{};
    char* w = static_cast<char*>(ws);
    const bool greedy = c.temperature == 0.0;
    a.x = c.x;
    a.y = greedy ? nullptr : c.y;
    a.drafts = c.drafts;
    a.u = c.u;
    a.accepted = c.accepted, a.tokens = c.tokens, a.logprob = c.logprob;
    a.count = reinterpret_cast<int32_t*>(w);
    a.part = reinterpret_cast<double2*>(w + p.part);
    a.best = reinterpret_cast<float2*>(w + p.best);
    a.picked = reinterpret_cast<float*>(w + p.picked);
    a.sums = reinterpret_cast<double*>(w + p.sums);
    a.ldb_x = c.ldb_x, a.ldt_x = c.ldt_x, a.ldb_y = c.ldb_y, a.ldt_y = c.ldt_y;
    a.c = greedy ? kLog2e : kLog2e / c.temperature;
    a.c_hi = std::nextafterf(static_cast<float>(a.c), 0.0f);
    a.c_lo = static_cast<float>(a.c - static_cast<double>(a.c_hi));
    a.K = c.K, a.V = c.V, a.tok_bytes = c.tok_bytes;
    a.rows = p.rows, a.segments = p.segments, a.segment = p.segment, a.chunks = p.chunks, a.runs = p.runs;
    for (int b = 0; b < c.B; ++b) a.n[b] = static_cast<uint8_t>(c.counts ? c.counts[b] : c.K);
    const dim3 first(p.segments, p.rows, c.B), second(p.groups, c.B), block(kThreads);
#define DT_GO(M, G)                                                                           \
    do {                                                                                      \
        hipLaunchKernelGGL((verify_rows_kernel<M, G, kRows>), first, block, 0, s, a);         \
        DT_HIP_TRY(hipGetLastError());                                                        \
        hipLaunchKernelGGL((verify_draw_kernel<M, G, kRows>), second, block, 0, s, a);        \
        DT_HIP_TRY(hipGetLastError());                                                        \
    } while (0)
    if (c.dtype == DT_BF16) {
        if (greedy) DT_GO(true, true);
        else DT_GO(true, false);
    } else {
        if (greedy) DT_GO(false, true);
        else DT_GO(false, false);
    }
#undef DT_GO
    return DT_OK;
}
int launch(const Call& c, const Plan& p, void* ws, hipStream_t s) {
    return c.B > kFewRows ? launch_rows<kMaxRaggedBatch>(c, p, ws, s) : launch_rows<kFewRows>(c, p, ws, s);
}

// rows of V values at ld apart do not reach back into each other's batch or leave 64 bits
bool bad_strides(int B, int T, int64_t ldb, int64_t ldt) {
    constexpr int64_t kMost = static_cast<int64_t>(1) << 52;
    return ldb < 0 || ldt < 0 || ldb > kMost / B || ldt > kMost / std::max(T, 1);
}

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" {

int dt_verify_drafts_workspace(int B, int K, int V, int has_draft_logits, double temperature, int64_t* bytes) {
    clear_error();
    if (!bytes) return set_error(DT_ERR_INVALID_ARG, "bytes is NULL");
    DT_TRY(check_sizes(B, K, V, temperature));
    *bytes = make_plan(B, K, V, has_draft_logits != 0, temperature == 0.0).bytes;
    return DT_OK;
}

int dt_verify_drafts(dt_ctx* ctx, const void* logits, const void* drafts, const float* uniforms, const void* draft_logits, int B, int K,
                     int V, int64_t ldb, int64_t ldt, int64_t ldb_draft, int64_t ldt_draft, int token_bytes, const int32_t* counts,
                     double temperature, int32_t* accepted, int32_t* tokens, float* logprob, void* ws, int64_t ws_bytes, int dtype,
                     int mem, void* stream) {
    clear_error();
    DT_TRY(check_sizes(B, K, V, temperature));
    if (!logits || !accepted || !tokens || !logprob || (K > 0 && !drafts))
        return set_error(DT_ERR_INVALID_ARG, "logits, drafts, accepted, tokens and logprob must be non-NULL");
    if (temperature > 0.0 && !uniforms) return set_error(DT_ERR_INVALID_ARG, "uniforms must be non-NULL");
    if (dtype != DT_FP32_EXACT && dtype != DT_BF16) return set_error(DT_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (mem != DT_MEM_DEVICE && mem != DT_MEM_HOST) return set_error(DT_ERR_INVALID_ARG, "unknown mem %d", mem);
    if (token_bytes != 4 && token_bytes != 8) return set_error(DT_ERR_INVALID_ARG, "token_bytes=%d must be 4 or 8", token_bytes);
    if (bad_strides(B, K + 1, ldb, ldt) || (draft_logits && bad_strides(B, K, ldb_draft, ldt_draft)))
        return set_error(DT_ERR_INVALID_ARG, "row strides out of range");
    if (counts)
        for (int b = 0; b < B; ++b)
            if (counts[b] < 0 || counts[b] > K) return set_error(DT_ERR_INVALID_ARG, "counts[%d]=%d outside [0, K=%d]", b, counts[b], K);
    const size_t esz = dtype == DT_BF16 ? 2 : 4;
    const auto off = [](const void* p, size_t by) { return reinterpret_cast<uintptr_t>(p) % by != 0; };
    const bool greedy = temperature == 0.0;
    const Plan p = make_plan(B, K, V, draft_logits != nullptr, greedy);
    if (mem == DT_MEM_DEVICE) {
        if (off(logits, esz) || off(draft_logits, esz) || off(drafts, token_bytes) || off(uniforms, 4) || off(accepted, 4) || off(tokens, 4) ||
            off(logprob, 4))
            return set_error(DT_ERR_INVALID_ARG, "logits, drafts, uniforms and results must be aligned to their elements");
        if (!ws || ws_bytes < p.bytes || !aligned16(ws))
            return set_error(DT_ERR_INVALID_ARG, "the workspace has %lld bytes (16-byte aligned), the call needs %lld", (long long)(ws ? ws_bytes : 0), (long long)p.bytes);
    } else if (K > 0) {
        for (int b = 0; b < B; ++b)
            for (int i = 0; i < (counts ? counts[b] : K); ++i) {
                const int64_t at = static_cast<int64_t>(b) * K + i;
                const int64_t t = token_bytes == 4 ? static_cast<const int32_t*>(drafts)[at] : static_cast<const int64_t*>(drafts)[at];
                if (t < 0 || t >= V) return set_error(DT_ERR_INVALID_ARG, "draft %lld of row %d outside [0, V=%d)", (long long)t, b, V);
            }
    }
    if (!ctx) return set_error(DT_ERR_INVALID_ARG, "ctx is NULL");
    DeviceScope scope;
    DT_TRY(scope.enter(ctx->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    Call c{logits, draft_logits, drafts, uniforms, accepted, tokens, logprob, B, K, V, ldb, ldt, ldb_draft, ldt_draft, token_bytes,
           counts, temperature, dtype, mem};
    if (mem == DT_MEM_DEVICE) return launch(c, p, ws, s);

    // host memory: staged through the context's buffers, synchronous
    const size_t row = V * esz;
    const auto stage = [&](int at, const void* from, int T, int64_t lb, int64_t lt) -> int {
        DT_TRY(ctx->stage[at].ensure(std::max<size_t>(16, static_cast<size_t>(B) * T * row)));
        for (int b = 0; b < B && T > 0; ++b)
            DT_HIP_TRY(hipMemcpy2DAsync(static_cast<char*>(ctx->stage[at].ptr) + b * T * row, row,
                                        static_cast<const char*>(from) + b * lb * esz, std::max<size_t>(lt * esz, row), row, T,
                                        hipMemcpyHostToDevice, s));
        return DT_OK;
    };
    if (ldt < V && K > 0) return set_error(DT_ERR_INVALID_ARG, "host rows %lld values apart overlap", (long long)ldt);
    if (draft_logits && ldt_draft < V && K > 1) return set_error(DT_ERR_INVALID_ARG, "host rows %lld values apart overlap", (long long)ldt_draft);
    DT_TRY(stage(0, logits, K + 1, ldb, ldt));
    c.x = ctx->stage[0].ptr;
    c.ldt_x = V;
    c.ldb_x = static_cast<int64_t>(K + 1) * V;
    if (draft_logits) {
        DT_TRY(stage(1, draft_logits, K, ldb_draft, ldt_draft));
        c.y = ctx->stage[1].ptr;
        c.ldt_y = V;
        c.ldb_y = static_cast<int64_t>(K) * V;
    }
    const size_t toks = static_cast<size_t>(B) * K * token_bytes, outs = static_cast<size_t>(B) * (K + 1) * 4;
    DT_TRY(ctx->stage[2].ensure(std::max<size_t>(16, toks)));
    DT_TRY(ctx->stage[3].ensure(outs));
    DT_TRY(ctx->stage[4].ensure(2 * outs + B * 4));
    DT_TRY(ctx->stage[5].ensure(p.bytes));
    if (toks) DT_HIP_TRY(hipMemcpyAsync(ctx->stage[2].ptr, drafts, toks, hipMemcpyHostToDevice, s));
    if (uniforms) DT_HIP_TRY(hipMemcpyAsync(ctx->stage[3].ptr, uniforms, outs, hipMemcpyHostToDevice, s));
    c.drafts = ctx->stage[2].ptr;
    c.u = static_cast<const float*>(ctx->stage[3].ptr);
    char* out = static_cast<char*>(ctx->stage[4].ptr);
    c.tokens = reinterpret_cast<int32_t*>(out);
    c.logprob = reinterpret_cast<float*>(out + outs);
    c.accepted = reinterpret_cast<int32_t*>(out + 2 * outs);
    DT_TRY(launch(c, p, ctx->stage[5].ptr, s));
    DT_HIP_TRY(hipMemcpyAsync(tokens, c.tokens, outs, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipMemcpyAsync(logprob, c.logprob, outs, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipMemcpyAsync(accepted, c.accepted, static_cast<size_t>(B) * 4, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

}  // extern "C"
