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
// A token is one side of a border or the other, and there are as many borders as tokens in the vocabulary: sums whose terms are off by
// 2^-24 would give another token about once in a few hundred calls. So probabilities and sums are held in 64 bits, the terms to 10^-12.
//
// Work: every row is read once for its sum (first kernel: a row in segments, as many as fill the CUs), and behind a refused draft the two
// rows that the weights come from once more, mostly from the caches (second kernel: 2048 values of a batch row a workgroup; each
// works out from the first kernel's sums which draft was refused). The last workgroup of a batch row to leave its weights' sum finds
// the segment that the border lies in, and in it the token.

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
constexpr int kOwn = 8;                       // values of a thread in the second kernel
constexpr int kSegment = kOwn * kThreads;
constexpr int kMinSegment = 2048;             // values of a segment of the first kernel at least
constexpr int kFill = 2048;                   // workgroups that the first kernel aims at, eight a CU
constexpr double kLog2e = 1.4426950408889634074;
constexpr double kLn2 = 0.69314718055994530942;
constexpr double kFar = -1000.0;              // 2^kFar and below counts as 0
constexpr double kNear = 500.0;               // a term may be 2^kNear; above it the sum's reference moves
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
    int32_t* count;       // [B]: workgroups of the second kernel that are done
    double2* part;        // [B][rows][segments]: one of the logits as reference, and the sum of 2^(c (x - reference))
    float2* best;         // [B][K + 1][segments] at T = 0: the largest logit, its index (as bits)
    double* total;        // [B][own segments]
    int64_t ldb_x, ldt_x, ldb_y, ldt_y;
    double c;             // log2(e) / T
    int K, V, tok_bytes;
    int rows;             // of a batch row: K + 1, and K of the drafts
    int segments, segment;  // of the first kernel, values of one
    int own_segments;     // of the second
    uint8_t n[kRows];     // drafts of each batch row
};

// 2^t to 10^-12 for t <= 1000, 0 below kFar; NaN stays. (2^f on [-1/2, 1/2] as its interpolation in nine Chebyshev points.)
__device__ __forceinline__ double exp2_64(double t) {
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
    v = __builtin_amdgcn_ldexp(v, static_cast<int>(__double_as_longlong(m)));
    return t < kFar ? 0.0 : v;
}

template <bool kBf16>
constexpr int kPer = kBf16 ? 8 : 4;  // values of a 16-byte piece

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
    for (int i = 0; i < kPer<kBf16>; ++i) {
        x[i] = -__builtin_huge_valf();
        if (at + i < end) {
            if constexpr (kBf16) x[i] = __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[at + i]) << 16);
            else x[i] = static_cast<const float*>(row)[at + i];
        }
    }
}
template <bool kBf16>
__device__ __forceinline__ float load_one(const void* row, int at) {
    if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[at]) << 16);
    else return static_cast<const float*>(row)[at];
}

// row r of a batch row: the model's (r <= K) or the drafts'
template <bool kBf16, int kRows>
__device__ __forceinline__ const void* row_of(const VerifyArgs<kRows>& a, int b, int r) {
    const int64_t at = r <= a.K ? b * a.ldb_x + r * a.ldt_x : b * a.ldb_y + (r - a.K - 1) * a.ldt_y;
    return static_cast<const char*>(r <= a.K ? a.x : a.y) + at * (kBf16 ? 2 : 4);
}

// a sum of 2^(c (x - ref)), joined with another. (Differences of logits are exact in 64 bits, or their smaller one does not count; their
// products with c are not, which would show in logits of 10^6 and more.)
__device__ __forceinline__ void join(double c, double& ref, double& sum, double r2, double s2) {
    const double to = ref > r2 ? ref : r2;
    sum = sum * exp2_64(c * (ref - to)) + s2 * exp2_64(c * (r2 - to));
    ref = to;
}

template <bool kBf16, bool kGreedy, int kRows>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyArgs<kRows> a) {
    constexpr int P = kPer<kBf16>;
    constexpr int kPieces = kBf16 ? 2 : 4;  // under way at once
    __shared__ double2 red[kWaves];
    __shared__ float2 red_best[kWaves];
    const int b = blockIdx.z, r = blockIdx.y, seg = blockIdx.x, n = a.n[b];
    if (seg == 0 && r == 0 && threadIdx.x == 0) a.count[b] = 0;
    if (r <= a.K ? r > n : r - a.K - 1 >= n) return;
    const void* row = row_of<kBf16>(a, b, r);
    const int from = seg * a.segment, end = min(a.V, from + a.segment);
    const double c = a.c;
    double ref = kLowest, sum = 0.0;
    float top = -__builtin_huge_valf();
    int top_at = from;
    for (int at = from + static_cast<int>(threadIdx.x) * P; at < end; at += kPieces * kThreads * P) {
        float x[kPieces][P];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) load_piece<kBf16>(row, at + i * kThreads * P, end, x[i]);
        float most = x[0][0];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                most = fmaxf(most, x[i][j]);
                if (kGreedy && x[i][j] > top) top = x[i][j], top_at = at + i * kThreads * P + j;
            }
        if ((most - ref) * c > kNear) {  // (seldom: the first values, and those far above them)
            sum *= exp2_64((ref - most) * c);
            ref = most;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) sum += exp2_64((x[i][j] - ref) * c);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        join(c, ref, sum, __shfl_xor(ref, o, 64), __shfl_xor(sum, o, 64));
        if constexpr (kGreedy) {
            const float t2 = __shfl_xor(top, o, 64);
            const int a2 = __shfl_xor(top_at, o, 64);
            if (t2 > top || (t2 == top && a2 < top_at)) top = t2, top_at = a2;
        }
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = make_double2(ref, sum);
        if constexpr (kGreedy) red_best[threadIdx.x >> 6] = make_float2(top, __int_as_float(top_at));
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) {
        join(c, ref, sum, red[i].x, red[i].y);
        if constexpr (kGreedy) {
            const float t2 = red_best[i].x;
            const int a2 = __float_as_int(red_best[i].y);
            if (t2 > top || (t2 == top && a2 < top_at)) top = t2, top_at = a2;
        }
    }
    a.part[(static_cast<int64_t>(b) * a.rows + r) * a.segments + seg] = make_double2(ref, sum);
    if constexpr (kGreedy) a.best[(static_cast<int64_t>(b) * (a.K + 1) + r) * a.segments + seg] = make_float2(top, __int_as_float(top_at));
}

__device__ __forceinline__ double log2_p(double c, float x, double2 row) { return fma(x - row.x, c, -row.y); }

template <int kRows>
__device__ __forceinline__ int draft_of(const VerifyArgs<kRows>& a, int b, int i) {
    const int64_t at = static_cast<int64_t>(b) * a.K + i;
    if (a.tok_bytes == 4) return static_cast<const int32_t*>(a.drafts)[at];
    const int64_t t = static_cast<const int64_t*>(a.drafts)[at];
    return t < 0 || t >= a.V ? -1 : static_cast<int>(t);
}

// sums before a thread's own of the workgroup's, in the threads' order, and of all
__device__ __forceinline__ double scan(double v, double (&red)[kWaves], double* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double before = __shfl_up(s, o, 64);
        if (lane >= o) s += before;
    }
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

template <bool kBf16, bool kGreedy, int kRows>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs<kRows> a) {
    __shared__ double2 lse[kMaxRows];  // each row's reference, and log2 of its sum; NaN of a row that has none
    __shared__ int best[kMaxDrafts + 1];
    __shared__ float score[kMaxDrafts + 1];
    __shared__ int drafts[kMaxDrafts];
    __shared__ double red[kWaves];
    __shared__ int sh_accepted, sh_last, sh_at;
    const int b = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, n = a.n[b], K = a.K, V = a.V;

    // the rows' sums: 16 lanes a row
    const int own_rows = n + 1 + (a.y ? n : 0);
    for (int i = tid >> 4; i < own_rows; i += kThreads / 16) {
        const int r = i <= n ? i : K + 1 + (i - n - 1);
        const double2* p = a.part + (static_cast<int64_t>(b) * a.rows + r) * a.segments;
        double ref = kLowest, sum = 0.0;
        float top = -__builtin_huge_valf();
        int top_at = 0;
        for (int s = tid & 15; s < a.segments; s += 16) {
            const double2 v = p[s];
            join(a.c, ref, sum, v.x, v.y);
            if (kGreedy) {
                const float2 w = a.best[(static_cast<int64_t>(b) * (K + 1) + r) * a.segments + s];
                if (w.x > top) top = w.x, top_at = __float_as_int(w.y);
            }
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
            join(a.c, ref, sum, __shfl_xor(ref, o, 16), __shfl_xor(sum, o, 16));
            if (kGreedy) {
                const float t2 = __shfl_xor(top, o, 16);
                const int a2 = __shfl_xor(top_at, o, 16);
                if (t2 > top || (t2 == top && a2 < top_at)) top = t2, top_at = a2;
            }
        }
        if ((tid & 15) == 0) {
            const double l = sum > 0.0 ? log2(sum) : __builtin_nan("");
            lse[i <= n ? i : K + 1 + (i - n - 1)] = make_double2(ref, l);
            if (kGreedy) best[i] = l == l ? top_at : -1;
        }
    }
    __syncthreads();
    if (tid < 64) {
        bool ok = false;
        if (tid < n) {
            const int d = draft_of(a, b, tid);
            float lp = 0.0f;
            if (d >= 0 && d < V) {
                const double t = log2_p(a.c, load_one<kBf16>(row_of<kBf16>(a, b, tid), d), lse[tid]);
                lp = static_cast<float>(t * kLn2);
                if (kGreedy) ok = d == best[tid];
                else {
                    double q = 1.0;
                    if (a.y) q = exp2_64(log2_p(a.c, load_one<kBf16>(row_of<kBf16>(a, b, K + 1 + tid), d), lse[K + 1 + tid]));
                    ok = a.u[static_cast<int64_t>(b) * (K + 1) + tid] * q < exp2_64(t);
                }
            }
            drafts[tid] = d;
            score[tid] = lp;
        }
        const uint64_t yes = __ballot(ok);
        if (tid == 0) sh_accepted = yes == ~0ull ? 64 : __builtin_ctzll(~yes);
    }
    __syncthreads();
    const int acc = sh_accepted;
    // results of row b: the accepted drafts, `token` and its log probability, then nothing
    const auto finish = [&](int token) {
        for (int i = tid; i <= K; i += kThreads) {
            const int64_t at = static_cast<int64_t>(b) * (K + 1) + i;
            if (i < acc) {
                a.tokens[at] = drafts[i];
                a.logprob[at] = score[i];
            } else if (i == acc) {
                a.tokens[at] = token;
                a.logprob[at] = token < 0 ? __builtin_nanf("")
                                          : static_cast<float>(log2_p(a.c, load_one<kBf16>(row_of<kBf16>(a, b, i), token), lse[i]) * kLn2);
            } else {
                a.tokens[at] = -1;
                a.logprob[at] = 0.0f;
            }
        }
        if (tid == 0) a.accepted[b] = acc;
    };
    if constexpr (kGreedy) {
        finish(best[acc]);
        return;
    }

    // the weights of the thread's values, at seg * kSegment + tid * kOwn
    const void* px = row_of<kBf16>(a, b, acc);
    const bool refused = acc < n;
    const int not_this = refused && !a.y ? drafts[acc] : -1;
    const void* qx = refused && a.y ? row_of<kBf16>(a, b, K + 1 + acc) : nullptr;
    const double2 lp = lse[acc], lq = lse[qx ? K + 1 + acc : acc];
    bool plain = false;  // w = p: the difference left nothing
    const auto weights = [&](int at, double (&w)[kOwn]) {
        constexpr int P = kPer<kBf16>;
#pragma unroll
        for (int i = 0; i < kOwn / P; ++i) {
            float x[P];
            load_piece<kBf16>(px, at + i * P, V, x);
#pragma unroll
            for (int j = 0; j < P; ++j) w[i * P + j] = exp2_64(log2_p(a.c, x[j], lp));
        }
        if (plain) return;
        if (qx) {
#pragma unroll
            for (int i = 0; i < kOwn / P; ++i) {
                float x[P];
                load_piece<kBf16>(qx, at + i * P, V, x);
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const double d = w[i * P + j] - exp2_64(log2_p(a.c, x[j], lq));
                    w[i * P + j] = d < 0.0 ? 0.0 : d;  // (NaN stays)
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (at + i == not_this) w[i] = 0.0;
        }
    };
    const auto own_sum = [&](int at, double (&w)[kOwn]) {
        double s = 0.0;
        weights(at, w);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) s += w[i];
        return s;
    };
    double w[kOwn], all;
    scan(own_sum(seg * kSegment + tid * kOwn, w), red, &all);
    double* totals = a.total + static_cast<int64_t>(b) * a.own_segments;
    if (tid == 0) {
        // through to the memory that all XCDs see, and complete before it is counted
        __hip_atomic_store(totals + seg, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        sh_last = __hip_atomic_fetch_add(a.count + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.own_segments - 1;
    }
    __syncthreads();
    if (!sh_last) return;

    // the last workgroup: the border's segment, then its token
    const int each = (a.own_segments + kThreads - 1) / kThreads;
    const auto total_of = [&](int s) {
        return s < a.own_segments ? __hip_atomic_load(totals + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    };
    const auto pick = [&]() -> int {
        double mine = 0.0;
        for (int i = 0; i < each; ++i) mine += total_of(tid * each + i);
        double before = scan(mine, red, &all);
        if (!(all > 0.0)) return all == 0.0 ? -2 : -1;
        const double bound = a.u[static_cast<int64_t>(b) * (K + 1) + K] * all;
        // the first whose sum passes the border; where rounding leaves none, the last that has a weight
        const auto first_over = [&](bool over, bool some, int at) {
            if (tid == 0) sh_at = 0x7fffffff;
            __syncthreads();
            if (over) atomicMin(&sh_at, at);
            __syncthreads();
            const int found = sh_at;
            __syncthreads();
            if (found != 0x7fffffff) return found;
            if (tid == 0) sh_at = -1;
            __syncthreads();
            if (some) atomicMax(&sh_at, at);
            __syncthreads();
            const int last = sh_at;
            __syncthreads();
            return last;
        };
        int my_at = 0;
        double my_before = 0.0;
        {
            bool over = false, some = false;
            for (int i = 0; i < each && !over; ++i) {
                const double t = total_of(tid * each + i);
                if (t > 0.0) {
                    some = true;
                    my_at = tid * each + i;
                    my_before = before;
                    over = before + t > bound;
                }
                before += t;
            }
            const int s = first_over(over, some, my_at);
            if (some && my_at == s) red[0] = my_before;
            __syncthreads();
            my_before = red[0];
            my_at = s;
        }
        const int at = my_at * kSegment + tid * kOwn;
        const double sum = own_sum(at, w);
        double in_segment;
        double upto = my_before + scan(sum, red, &in_segment);
        bool over = false, some = false;
        int token = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (!over && w[i] > 0.0) {
                some = true;
                token = at + i;
                upto += w[i];
                over = upto > bound;
            }
        }
        return first_over(over, some, token);
    };
    int token = pick();
    if (token == -2) {  // (the same for the whole workgroup)
        plain = true;
        // p's sums, by this workgroup alone
        for (int s = 0; s < a.own_segments; ++s) {
            scan(own_sum(s * kSegment + tid * kOwn, w), red, &all);
            if (tid == 0) __hip_atomic_store(totals + s, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        token = pick();
        if (token < 0) token = -1;
    }
    finish(token);
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
    int rows, segments, segment, own_segments;
    int64_t part, best, total, bytes;  // offsets
};
Plan make_plan(int B, int K, int V, bool drafts, bool greedy) {
    Plan p{};
    p.rows = K + 1 + (drafts && !greedy ? K : 0);
    const int64_t rows = static_cast<int64_t>(B) * p.rows;
    const int most = (V + kMinSegment - 1) / kMinSegment;
    p.segments = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (kFill + rows - 1) / rows)));
    p.segment = ((V + p.segments - 1) / p.segments + 7) / 8 * 8;
    p.segments = (V + p.segment - 1) / p.segment;
    p.own_segments = greedy ? 1 : (V + kSegment - 1) / kSegment;
    p.part = (static_cast<int64_t>(B) * 4 + 255) / 256 * 256;
    p.best = p.part + rows * p.segments * 16;
    p.total = p.best + (greedy ? rows * p.segments * 8 : 0);
    p.bytes = p.total + (greedy ? 0 : static_cast<int64_t>(B) * p.own_segments * 8);
    return p;
}

int check_sizes(int B, int K, int V, double temperature) {
    if (B < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d must be >= 1", B);
    if (B > kMaxRaggedBatch) return set_error(DT_ERR_UNSUPPORTED, "B=%d > %d", B, kMaxRaggedBatch);
    if (K < 0 || K > kMaxDrafts) return set_error(K < 0 ? DT_ERR_INVALID_ARG : DT_ERR_UNSUPPORTED, "K=%d drafts outside [0, %d]", K, kMaxDrafts);
    if (V < 1) return set_error(DT_ERR_INVALID_ARG, "V=%d must be >= 1", V);
    if (V > kMaxVocab) return set_error(DT_ERR_UNSUPPORTED, "V=%d > %d", V, kMaxVocab);
    if (!std::isfinite(temperature) || !(temperature >= 0.0))
        return set_error(DT_ERR_INVALID_ARG, "temperature %g must be finite and >= 0", temperature);
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
    a.total = reinterpret_cast<double*>(w + p.total);
    a.ldb_x = c.ldb_x, a.ldt_x = c.ldt_x, a.ldb_y = c.ldb_y, a.ldt_y = c.ldt_y;
    a.c = greedy ? kLog2e : kLog2e / c.temperature;
    a.K = c.K, a.V = c.V, a.tok_bytes = c.tok_bytes;
    a.rows = p.rows, a.segments = p.segments, a.segment = p.segment, a.own_segments = p.own_segments;
    for (int b = 0; b < c.B; ++b) a.n[b] = static_cast<uint8_t>(c.counts ? c.counts[b] : c.K);
    const dim3 first(p.segments, p.rows, c.B), second(p.own_segments, c.B), block(kThreads);
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
