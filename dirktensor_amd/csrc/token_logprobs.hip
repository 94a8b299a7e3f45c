// Log probabilities of given tokens, with each row's entropy and most likely tokens, and the gradient of the
// log probabilities and entropies with respect to the logits.
//
// For a row x of V logits and its token y, with m = max x, e_j = exp(x_j - m), l = sum e_j:
//   logprob = (x_y - m) - log l
//   entropy = log l - sum e_j (x_j - m) / l      (both terms >= 0: no difference of large numbers)
//   dx_j    = g (delta_jy - p_j) - h p_j (log p_j + entropy),   p_j = exp((x_j - m) - log l)
// for d logprob = g, d entropy = h. The top alternatives are the k largest logits, the lower index first of equals.
//
// Both are bound by HBM: the forward reads the logits once, the backward reads them and writes as many.
//
// Forward: a workgroup of 256 threads streams a row (or, where there are few rows, a segment of one) with 16-byte loads;
// a thread keeps its own running maximum, sum and weighted sum, so the loop has no exchange between lanes, and the statistics
// meet once at the end. The alternatives cost no second pass: after the first fifth of the row (more for many) the k-th largest
// of the threads' maxima is a bound that at least k values reach. The threads whose maximum reaches it look at their share of that part
// again (from the caches), and the rest of the row is compared with the bound as it streams by, one comparison for 16 values; what reaches
// it (about 5 k values at most) is collected in LDS, and each takes the place that the number of larger ones gives it. Keys are
// (value, index) pairs, so no two are equal, ties go to the lower index and the order of the collection does not matter. Where more values
// reach the bound than the list holds (rows that rise, or begin with masked values) the maxima of the whole row give another and the
// row is read once more; where that leaves too many as well (equal values) the k-th key is found digit by digit in passes over the
// row. A row cut into segments leaves (m, l, sum, k keys) of each in the workspace and a second kernel joins them.
//
// Measured: 2048 rows of 100352 in fp32, 822 MB, with 5 alternatives 130 us, without 121 (6.3 and 6.8 TB/s; reads past the
// caches reach 7.0), with 64 163. Rows whose first quarter is masked 259, with fifty tokens left 139, of equal values 2140 (selected one
// after another 5 alternatives took 1460, 1470 and 1440, 64 ten times as long). 16 rows with 20 alternatives 13.2 us, both launches
// (25 segments of 16 KB each: the chains from the first load to the sorted keys). The gradient of the 2048 rows, 1.64 GB moved, 300 us
// (5.5 TB/s; a copy of as much 5.7 through the caches, 6.3 past them), of 300 rows of 50277 in bf16, 60 MB, 13.6 us (4.4 TB/s; a copy
// 4.1 and 5.3).

#include "dt_internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace dt {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kMaxTop = 64;
constexpr int kList = 1024;          // values that may reach the bound before the selection goes one by one
constexpr uint32_t kOrderNegInf = 0x007fffffu;  // order_of(-inf): the least there is
constexpr int kBoundBytes = 96 << 10;  // of a run that gives the bound, where more than a fifth of it does
constexpr int kBatch = 16;           // values a thread takes at a time
constexpr int kMinSegment = 4096;    // values of a segment at least
constexpr int kJoinKeys = 8;         // keys of a row's segments that a thread of the second kernel takes at most
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLo = 1.92596303e-8f;  // log2 e - kLog2e
constexpr float kLn2 = 0.693147180559945f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLowest = -3.402823466e38f;

struct LogprobArgs {
    const void* x;
    const void* tok;
    int64_t ldb, ldt;     // strides of x, elements
    int64_t ignore;
    int tok64;
    int T, V, k;
    int segments, seg_len;
    float* logprob;
    float* entropy;       // nullable
    float* m;
    float* l;
    int32_t* top_index;   // [rows][k]
    float* top_logprob;
    float* part;          // [rows][segments][4]: m, l, weighted sum
    uint64_t* part_key;   // [rows][segments][k], sorted
};

// whether a token is skipped: a token that has DT_NO_IGNORE's bits is none of the vocabulary's, not one to ignore
__host__ __device__ __forceinline__ bool is_skipped(int64_t y, int64_t ignore) { return y == ignore && ignore != DT_NO_IGNORE; }

__device__ __forceinline__ int64_t token_at(const void* tok, int tok64, int64_t row) {
    return tok64 ? static_cast<const int64_t*>(tok)[row] : static_cast<const int32_t*>(tok)[row];
}

// (value, index) as a number that orders like the pair, the lower index above; NaN counts as -inf. Never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    x = x != x ? kNegInf : x + 0.0f;  // (-0 and 0 are equal)
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int index) {
    return static_cast<uint64_t>(order_of(x)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

// A run of n values of a row in 16-byte pieces from its first value on, whatever its alignment (global 16-byte accesses
// take any, and a row's bits then do not depend on where it lies), single values after the last whole piece. Piece p belongs to
// thread p % 256; a thread's batch j is its pieces 256 (j kPer + 0 .. kPer - 1) + tid.
template <bool kBf16>
struct Run {
    static constexpr int kEs = kBf16 ? 2 : 4, kPiece = 16 / kEs, kPer = kBatch / kPiece;
    using Piece = std::conditional_t<kBf16, u32x4_at2, u32x4_at4>;
    const uint8_t* x;  // the run's first value
    int n, pieces, batches;
    __device__ __forceinline__ Run(const void* p, int n_) : x(static_cast<const uint8_t*>(p)), n(n_) {
        pieces = n / kPiece;
        batches = (pieces + kThreads * kPer - 1) / (kThreads * kPer);
    }
    __device__ __forceinline__ float one(int i) const {
        if constexpr (kBf16) return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(x)[i]) << 16);
        return reinterpret_cast<const float*>(x)[i];
    }
    __device__ __forceinline__ int tail() const { return pieces * kPiece; }
    __device__ __forceinline__ u32x4 load(int p) const { return *reinterpret_cast<const Piece*>(x + p * 16); }
    // a value that is not read again: past the caches (large reads reach 7.0 TB/s so, 6.1 through them)
    __device__ __forceinline__ u32x4 load_once(int p) const { return __builtin_nontemporal_load(reinterpret_cast<const Piece*>(x + p * 16)); }
    static __device__ __forceinline__ void unpack(const u32x4& w, float* v) {
        if constexpr (kBf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        }
    }
};

struct Stats {
    float m = kNegInf, s = 0.0f, d = 0.0f;  // maximum; sum e; sum e (x - m)
};

// v[i] without memory (as masks: a choice between two elements would put the array there), four at a time for few registers
__device__ __forceinline__ float pick(const float (&v)[kBatch], int i) {
    const auto either = [](uint32_t m, uint32_t a, uint32_t b) { return (a & m) | (b & ~m); };
    const uint32_t odd = 0u - (i & 1), upper = 0u - (i >> 1 & 1);
    uint32_t r = 0;
#pragma unroll
    for (int q = 0; q < kBatch / 4; ++q) {
        const auto u = [&](int j) { return __float_as_uint(v[4 * q + j]); };
        const uint32_t four = either(upper, either(odd, u(3), u(2)), either(odd, u(1), u(0)));
        r = i >> 2 == q ? four : r;
        asm volatile("" : "+v"(r));
    }
    return __uint_as_float(r);
}

// takes the values, and returns their maximum (-inf in the place of a value that is none)
template <int kN>
__device__ __forceinline__ float take(Stats& st, const float (&v)[kN]) {
    float bm = kNegInf;
#pragma unroll
    for (int i = 0; i < kN; ++i) bm = fmaxf(bm, v[i]);
    if (bm > st.m) {
        const float f = __builtin_amdgcn_exp2f((st.m - bm) * kLog2e);
        st.d = (st.d + st.s * fmaxf(st.m - bm, -1e4f)) * f;  // (further down f is 0: the sum must not become an infinity)
        st.s *= f;
        st.m = bm;
    }
    const float base = st.m == kNegInf ? 0.0f : st.m;
    float s = 0.0f, d = 0.0f;  // (the batch's own sums: fewer roundings one after another)
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        const float t = v[i] - base;
        // (log2 e in two parts: the first alone is off by 1.3e-8, the same way for every term)
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(t, kLog2e, t * kLog2eLo));
        s += e;
        d += e * fmaxf(t, -1e4f);  // (0 for -inf; a NaN shows in s)
    }
    st.s += s;
    st.d += d;
    return bm;
}

// a's statistics and b's
__device__ __forceinline__ void join(Stats& a, float m, float s, float d) {
    const float mx = fmaxf(a.m, m), base = mx == kNegInf ? 0.0f : mx;
    const float fa = __builtin_amdgcn_exp2f((a.m - base) * kLog2e), fb = __builtin_amdgcn_exp2f((m - base) * kLog2e);
    a.d = (a.d + a.s * fmaxf(a.m - base, -1e4f)) * fa + (d + s * fmaxf(m - base, -1e4f)) * fb;
    a.s = a.s * fa + s * fb;
    a.m = mx;
}

// the same total in every thread of the workgroup
__device__ __forceinline__ Stats join_block(Stats st, float (*buf)[3]) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        // (both lanes of a pair join lower first, so they agree to the bit)
        const float m = __shfl_xor(st.m, o, 64), s = __shfl_xor(st.s, o, 64), d = __shfl_xor(st.d, o, 64);
        if (threadIdx.x & o) {
            Stats lower;
            lower.m = m, lower.s = s, lower.d = d;
            join(lower, st.m, st.s, st.d);
            st.m = lower.m, st.s = lower.s, st.d = lower.d;
        } else {
            join(st, m, s, d);
        }
    }
    if ((threadIdx.x & 63) == 0) {
        float* b = buf[threadIdx.x >> 6];
        b[0] = st.m, b[1] = st.s, b[2] = st.d;
    }
    __syncthreads();
    Stats all;
    all.m = buf[0][0], all.s = buf[0][1], all.d = buf[0][2];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(all, buf[w][0], buf[w][1], buf[w][2]);
    return all;
}

// The row's token: its logit, and whether it is one of the vocabulary's or skipped. (Read first, as one load waits for another.)
struct Target {
    float x;
    bool skipped, known;
};
__device__ __forceinline__ Target target_of(const LogprobArgs& a, int64_t row, const void* xrow, bool bf16) {
    const int64_t y = token_at(a.tok, a.tok64, row);
    Target t{0.0f, is_skipped(y, a.ignore), y >= 0 && y < a.V};
    if (t.known) t.x = bf16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(xrow)[y]) << 16) : static_cast<const float*>(xrow)[y];
    return t;
}

struct Finish {
    float m, l, logl;
};
// (a row of nothing but -inf has no distribution: NaN)
__device__ __forceinline__ Finish finish(const LogprobArgs& a, int64_t row, const Target& t, const Stats& st, bool write) {
    Finish f;
    f.m = st.m;
    f.l = st.m == kNegInf ? __builtin_nanf("") : st.s;
    f.logl = logf(f.l);
    if (f.l != f.l) f.m = f.l;  // (a maximum passes NaN over)
    if (!write) return f;
    a.m[row] = f.m;
    a.l[row] = f.l;
    if (a.entropy) a.entropy[row] = f.logl - st.d / f.l;
    a.logprob[row] = t.skipped ? 0.0f : t.known ? (t.x - f.m) - f.logl : __builtin_nanf("");
    return f;
}

struct SelectBuf {
    uint32_t top[kThreads];  // of the threads (find_bound), or how many have a digit (select)
    uint64_t list[kList];
    int count;
};
static_assert(kThreads == 256, "a thread a digit");

// A bound that the k-th largest of the threads' `mine` (order_of their maximum; 0: none) reaches, to 20 bits, the same for all;
// empties the list. Each wave finds it for itself, bit by bit, from four of the 256 a lane.
__device__ __forceinline__ uint32_t find_bound(SelectBuf& b, uint32_t mine, int k) {
    __syncthreads();
    b.top[threadIdx.x] = mine;
    if (threadIdx.x == 0) b.count = 0;
    __syncthreads();
    uint32_t v[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) v[i] = b.top[i * 64 + (threadIdx.x & 63)];
    uint32_t bound = 0;
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t trial = bound | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) n += __popcll(__ballot(v[i] >= trial));
        if (n >= k) bound = trial;
    }
    return bound;
}

// whether the list has run over
__device__ __forceinline__ bool push(SelectBuf& b, uint64_t key) {
    if (*static_cast<volatile int*>(&b.count) >= kList + kThreads) return true;  // (long ago)
    const int at = atomicAdd(&b.count, 1);
    if (at < kList) b.list[at] = key;
    return at >= kList;
}

// The digit of the `least`-th largest key, given how many keys have each and how many lie `above` them all, which grows by those of
// larger digits; n: how many have it. The same for all waves: each finds it for itself, four digits a lane.
__device__ __forceinline__ int find_digit(const SelectBuf& b, int least, int& above, int& n) {
    const int lane = threadIdx.x & 63;
    int h[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += h[i] = static_cast<int>(b.top[lane * 4 + i]);
    int to = sum;  // of the lane's digits and larger
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int more = __shfl_down(to, o, 64);
        if (lane + o < 64) to += more;
    }
    const uint64_t reach = __ballot(above + to >= least);
    const int at = 63 - __clzll(static_cast<long long>(reach | 1));  // (the last lane that does)
    int d = 3, over = above + to - sum;
#pragma unroll
    for (int i = 3; i > 0; --i)
        if (d == i && over + h[i] < least) {
            over += h[i];
            --d;
        }
    n = __shfl(d == 3 ? h[3] : d == 2 ? h[2] : d == 1 ? h[1] : h[0], at, 64);
    above = __shfl(over, at, 64);
    return at * 4 + __shfl(d, at, 64);
}

// The k largest of the collected keys, in order, through out(place, key); places past the last get key 0. Where the list ran
// over, the k largest of all: each(f) calls f(key) for every key of the thread. The `least`-th key's digits are then found from the
// first on, a pass over the keys each, until the list holds what reaches them; no two keys are equal, so it does in the end. A list
// that holds fewer than the `least` that there are lacks only keys of -inf: these are the largest of those by their index.
template <class Each, class Out>
__device__ __forceinline__ void select(SelectBuf& b, int k, int least, Each each, Out out) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (b.count > kList || b.count < least) {
        const bool few = b.count < least;
        uint64_t digits = few ? static_cast<uint64_t>(kOrderNegInf) << 32 : 0, mask = few ? ~uint64_t(0) << 32 : 0;
        int above = few ? b.count : 0;
        for (int at = few ? 24 : 56; at >= 0; at -= 8) {
            if (at == 24) {  // (an index has 24 bits)
                digits |= 0xffull << 24;
                mask |= 0xffull << 24;
                continue;
            }
            __syncthreads();
            b.top[tid] = 0;
            __syncthreads();
            each([&](uint64_t key) {
                if ((key & mask) != digits) return;
                // (often all are alike: one addition then)
                const uint32_t d = static_cast<uint32_t>(key >> at) & 255, first = __builtin_amdgcn_readfirstlane(d);
                const uint64_t alike = __ballot(d == first);
                if (d != first) atomicAdd(&b.top[d], 1u);
                else if ((tid & 63) == __ffsll(static_cast<unsigned long long>(alike)) - 1) atomicAdd(&b.top[d], static_cast<uint32_t>(__popcll(alike)));
            });
            __syncthreads();
            int n;
            const int d = find_digit(b, least, above, n);
            digits |= static_cast<uint64_t>(d) << at;
            mask |= 0xffull << at;
            if (above + n <= kList) break;
        }
        __syncthreads();
        if (tid == 0) b.count = 0;
        __syncthreads();
        each([&](uint64_t key) {
            if ((key & mask) >= digits) push(b, key);
        });
        __syncthreads();
    }
    const int c = b.count;
    for (int i = tid; i < c; i += kThreads) {
        const uint64_t key = b.list[i];
        int larger = 0;
#pragma unroll 8
        for (int j = 0; j < c; ++j) larger += b.list[j] > key;
        if (larger < k) out(larger, key);
    }
    for (int i = c + tid; i < k; i += kThreads) out(i, 0);
}

__device__ __forceinline__ void write_top(const LogprobArgs& a, int64_t row, int place, uint64_t key, const Finish& f) {
    a.top_index[row * a.k + place] = key_index(key);
    a.top_logprob[row * a.k + place] = (key_value(key) - f.m) - f.logl;
}

template <bool kBf16, bool kTop>
__global__ __launch_bounds__(kThreads, 8) void logprob_rows_kernel(LogprobArgs a) {
    __shared__ float sbuf[kWaves][3];
    __shared__ SelectBuf buf;
    using R = Run<kBf16>;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / a.segments;
    const int seg = static_cast<int>(blockIdx.x - row * a.segments);
    const uint8_t* xrow = static_cast<const uint8_t*>(a.x) + ((row / a.T) * a.ldb + (row % a.T) * a.ldt) * R::kEs;
    const int first = seg * a.seg_len;
    const R run(xrow + static_cast<int64_t>(first) * R::kEs, min(a.V - first, a.seg_len));

    Target tgt{};
    if (a.segments == 1) tgt = target_of(a, row, xrow, kBf16);
    Stats st;
    uint32_t bound = 0;
    const int tail = run.tail() + tid;
    float last[1] = {kNegInf};
    if (tail < run.n) {
        last[0] = run.one(tail);
        take(st, last);
    }
    // f(batch's values, its number) for batches from .. to - 1, the next one's loads in flight while one is taken
    auto stream = [&](int from, int to, auto load, auto f) {
        const int whole = min(to, run.pieces / (kThreads * R::kPer));
        u32x4 w[R::kPer];
        if (from < whole) {
#pragma unroll
            for (int i = 0; i < R::kPer; ++i) w[i] = load((from * R::kPer + i) * kThreads + tid);
        }
        int j = from;
        for (; j < whole; ++j) {
            float v[kBatch];
#pragma unroll
            for (int i = 0; i < R::kPer; ++i) R::unpack(w[i], v + i * R::kPiece);
            if (j + 1 < whole) {
#pragma unroll
                for (int i = 0; i < R::kPer; ++i) w[i] = load(((j + 1) * R::kPer + i) * kThreads + tid);
            }
            f(v, j);
        }
        if (j < to) {  // the run's last batch: -inf where there is no piece
            float v[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) v[i] = kNegInf;
#pragma unroll
            for (int i = 0; i < R::kPer; ++i) {
                const int p = (j * R::kPer + i) * kThreads + tid;
                if (p < run.pieces) R::unpack(load(p), v + i * R::kPiece);
            }
            f(v, j);
        }
    };
    // use(key) for those of a batch's values that reach `least`, or all. Few do: a mask finds them, and each is taken from the
    // registers (read again, it would wait for the next batch's loads, which are under way).
    const auto look = [&](const float(&v)[kBatch], int j, bool all, float least, auto&& use) {
        uint32_t hits = (1u << kBatch) - 1;
        if (!all) {
            hits = 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) hits |= v[i] >= least ? 1u << i : 0u;
        }
        while (hits) {
            const int i = __ffs(hits) - 1, p = (j * R::kPer + i / R::kPiece) * kThreads + tid, at = p * R::kPiece + i % R::kPiece;
            hits &= hits - 1;
            if (p < run.pieces) use(key_of(pick(v, i), first + at));
        }
    };
    const auto cached = [&](int p) { return run.load(p); };
    const auto once = [&](int p) { return run.load_once(p); };
    if constexpr (kTop) {
        // How much of the run gives the bound: more of it leaves fewer values to list, but is looked at twice, which the caches must
        // hold. From one to two (fp32) or three (bf16) fifths, us: 2048 rows of 100352 in bf16, 64 alternatives, 123 and 105, of 32000 in
        // fp32 67 and 63; past kBoundBytes 159 and 188 (100352 in fp32, three fifths). Runs of a few batches give it from all of them;
        // the first batch stays in registers.
        const int fifths = kBf16 ? (a.k > 32 ? 3 : a.k > 8 ? 2 : 1) : (a.k > 32 ? 2 : 1);
        const int fifth = (run.batches + 4) / 5, most = kBoundBytes / (kThreads * kBatch * R::kEs);
        const int part = run.batches <= 4 ? run.batches : max(fifth, min((run.batches * fifths + 4) / 5, most));
        float v0[kBatch];
        stream(0, min(part, 1), cached, [&](const float(&v)[kBatch], int) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) v0[i] = v[i];
            take(st, v);
        });
        stream(1, part, cached, [&](const float(&v)[kBatch], int) { take(st, v); });
        const bool any = tail < run.n || tid < run.pieces, whole = run.n <= kList;
        const uint32_t mine = any ? order_of(st.m) : 0;
        bound = find_bound(buf, mine, a.k);
        // (values of -inf are listed only where the list holds the whole run: else they would fill it)
        float least = bound <= kOrderNegInf ? kLowest : key_value(static_cast<uint64_t>(bound) << 32);
        const auto list = [&](uint64_t key) {
            if (push(buf, key)) least = -kNegInf;  // (the list is of no use any more)
        };
        if (whole || (any && mine >= bound)) {
            if (tail < run.n && (whole || last[0] >= least)) push(buf, key_of(last[0], first + tail));
            if (part > 0) look(v0, 0, whole, least, list);
            stream(1, part, cached, [&](const float(&v)[kBatch], int j) { look(v, j, whole, least, list); });
        }
        stream(part, run.batches, once, [&](const float(&v)[kBatch], int j) {
            if (take(st, v) >= least || whole) look(v, j, whole, least, list);
        });
        // Too many: the threads' maxima of the whole run give a better bound.
        __syncthreads();
        if (buf.count > kList) {
            bound = find_bound(buf, any ? order_of(st.m) : 0, a.k);
            least = bound <= kOrderNegInf ? kLowest : key_value(static_cast<uint64_t>(bound) << 32);
            if (tail < run.n && last[0] >= least) push(buf, key_of(last[0], first + tail));
            stream(0, run.batches, cached, [&](const float(&v)[kBatch], int j) { look(v, j, false, least, list); });
        }
    } else {
        stream(0, run.batches, once, [&](const float(&v)[kBatch], int) { take(st, v); });
    }
    const Stats all = join_block(st, sbuf);
    Finish f{};
    if (a.segments == 1) f = finish(a, row, tgt, all, tid == 0);
    else if (tid == 0) {
        float* p = a.part + (row * a.segments + seg) * 4;
        p[0] = all.m, p[1] = all.s, p[2] = all.d;
    }
    if constexpr (kTop) {
        select(
            buf, a.k, min(a.k, run.n),
            [&](auto&& use) {
                if (tail < run.n) use(key_of(last[0], first + tail));
                stream(0, run.batches, cached, [&](const float(&v)[kBatch], int j) { look(v, j, true, kNegInf, use); });
            },
            [&](int place, uint64_t key) {
                if (a.segments == 1) write_top(a, row, place, key, f);
                else a.part_key[(row * a.segments + seg) * a.k + place] = key;
            });
    }
}

// Joins a row's segments.
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void logprob_join_kernel(LogprobArgs a) {
    __shared__ float sbuf[kWaves][3];
    __shared__ SelectBuf buf;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const uint8_t* xrow = static_cast<const uint8_t*>(a.x) + ((row / a.T) * a.ldb + (row % a.T) * a.ldt) * (kBf16 ? 2 : 4);
    const Target tgt = target_of(a, row, xrow, kBf16);
    Stats st;
    if (tid < a.segments) {  // (at most kThreads of them)
        const float* p = a.part + (row * a.segments + tid) * 4;
        st.m = p[0], st.s = p[1], st.d = p[2];
    }
    const uint64_t* keys = a.part_key + row * a.segments * a.k;
    const int n = a.segments * a.k;
    uint64_t key[kJoinKeys], mine = 0;  // all under way at once
#pragma unroll
    for (int i = 0; i < kJoinKeys; ++i) key[i] = i * kThreads + tid < n ? keys[i * kThreads + tid] : 0;
    const Stats all = join_block(st, sbuf);
    const Finish f = finish(a, row, tgt, all, tid == 0);
    if (a.k == 0) return;
#pragma unroll
    for (int i = 0; i < kJoinKeys; ++i) mine = key[i] > mine ? key[i] : mine;
    const uint32_t bound = find_bound(buf, static_cast<uint32_t>(mine >> 32), a.k);
    const auto each = [&](auto&& use) {
#pragma unroll
        for (int i = 0; i < kJoinKeys; ++i)
            if (key[i] != 0) use(key[i]);
    };
    each([&](uint64_t k) {
        if (static_cast<uint32_t>(k >> 32) >= bound) push(buf, k);
    });
    select(buf, a.k, a.k, each, [&](int place, uint64_t k) { write_top(a, row, place, k, f); });
}

// Segments a row: about four workgroups a CU, none shorter than kMinSegment, or twice that where there are as many workgroups or many
// keys, which each segment leaves k of; their keys a few a thread. fp32 rows of 100352, us: 1000 of them, 20 alternatives, in one
// segment 72, two 80; 300 in three 35, in seven 40; 16 in segments of 4096 13.2, of 2048 15.1, of 8192 14.3, with 64 alternatives 24, 26
// and 17.
void cut(int64_t rows, int V, int k, int* segments, int* seg_len) {
    constexpr int64_t kTarget = 1024, kCus = 256;
    const bool longer = k > 32 || rows * ((V + kMinSegment - 1) / kMinSegment) >= 4 * kCus;
    const int least = longer ? 2 * kMinSegment : kMinSegment;
    int64_t s = std::min<int64_t>((kTarget + rows / 2) / rows, (V + least - 1) / least);
    s = std::min<int64_t>(s, kThreads);
    if (k > 0) s = std::min<int64_t>(s, kJoinKeys * kThreads / k);
    s = std::max<int64_t>(s, 1);
    *seg_len = static_cast<int>(((V + s - 1) / s + 7) / 8 * 8);
    *segments = (V + *seg_len - 1) / *seg_len;
}

int64_t workspace_bytes(int64_t rows, int V, int k) {
    int segments = 0, len = 0;
    cut(rows, V, k, &segments, &len);
    return segments == 1 ? 0 : rows * segments * (4 * static_cast<int64_t>(sizeof(float)) + k * static_cast<int64_t>(sizeof(uint64_t)));
}

int launch_logprobs(LogprobArgs a, int64_t rows, bool bf16, void* ws, hipStream_t s) {
    cut(rows, a.V, a.k, &a.segments, &a.seg_len);
    // (keys first: they are the wider)
    a.part_key = static_cast<uint64_t*>(ws);
    a.part = reinterpret_cast<float*>(a.part_key + rows * a.segments * a.k);
    const dim3 g(static_cast<unsigned>(rows * a.segments)), t(kThreads);
    if (bf16) {
        if (a.k) hipLaunchKernelGGL((logprob_rows_kernel<true, true>), g, t, 0, s, a);
        else hipLaunchKernelGGL((logprob_rows_kernel<true, false>), g, t, 0, s, a);
    } else {
        if (a.k) hipLaunchKernelGGL((logprob_rows_kernel<false, true>), g, t, 0, s, a);
        else hipLaunchKernelGGL((logprob_rows_kernel<false, false>), g, t, 0, s, a);
    }
    DT_HIP_TRY(hipGetLastError());
    if (a.segments > 1) {
        if (bf16) hipLaunchKernelGGL((logprob_join_kernel<true>), dim3(static_cast<unsigned>(rows)), t, 0, s, a);
        else hipLaunchKernelGGL((logprob_join_kernel<false>), dim3(static_cast<unsigned>(rows)), t, 0, s, a);
        DT_HIP_TRY(hipGetLastError());
    }
    return DT_OK;
}

struct LogprobBwdArgs {
    const void* x;
    void* dx;
    const void* tok;
    const float* g;
    const float* h;  // nullable
    const float* m;
    const float* l;
    const float* entropy;
    int64_t ldb, ldt, ldb_out, ldt_out;
    int64_t ignore;
    int tok64;
    int T, V;
    int segments, seg_len;
    int64_t row0;    // the launch's first row
    int far;         // the gradient is too large to be found in a cache by whoever reads it: it is written past them
};

constexpr int kBwdPieces = 4;  // 16-byte pieces of a thread: few rows then fill the CUs too, and many leave no long tail

// One workgroup a segment of a row; each value is read and written by one thread, so dx may be x.
template <bool kBf16>
__global__ __launch_bounds__(kThreads) void logprob_bwd_kernel(LogprobBwdArgs a) {
    using R = Run<kBf16>;
    const int tid = threadIdx.x;
    const int in_launch = blockIdx.x / a.segments;
    const int64_t row = a.row0 + in_launch;
    const int first = static_cast<int>(blockIdx.x - in_launch * a.segments) * a.seg_len;
    const int n = min(a.V - first, a.seg_len);
    const int64_t b = row / a.T, t = row % a.T;
    const uint8_t* x = static_cast<const uint8_t*>(a.x) + (b * a.ldb + t * a.ldt + first) * R::kEs;
    uint8_t* dx = static_cast<uint8_t*>(a.dx) + (b * a.ldb_out + t * a.ldt_out + first) * R::kEs;
    const R run(x, n);
    // all of a thread's values are under way before the row's own numbers, which wait for one another
    u32x4 w[kBwdPieces];
#pragma unroll
    for (int i = 0; i < kBwdPieces; ++i)
        if (tid + i * kThreads < run.pieces) w[i] = run.load_once(tid + i * kThreads);
    const int64_t y = token_at(a.tok, a.tok64, row);
    float g = a.g[row];
    int hit = -1;
    if (is_skipped(y, a.ignore)) g = 0.0f;
    else if (y < 0 || y >= a.V) g = __builtin_nanf("");
    else if (y >= first && y < first + n) hit = static_cast<int>(y) - first;
    const float h = a.h ? a.h[row] : 0.0f;
    const float m = a.m[row], logl = logf(a.l[row]);
    // -dx = p (g + h (log p + entropy)); a row without a distribution (its sum is NaN) is NaN throughout
    const float lead = logl != logl ? logl : a.h ? g + h * a.entropy[row] : g;
    // log p is cut at -1000, where p is 0 and the bracket must not be an infinity
    auto grad = [&](float v) {
        if constexpr (kBf16) {  // (in the log2 domain: an error of 2^-22 of log p does not count beside the result's rounding)
            const float l2 = fmaxf(__builtin_fmaf(v - m, kLog2e, -logl * kLog2e), -1000.0f);
            return -__builtin_amdgcn_exp2f(l2) * __builtin_fmaf(h * kLn2, l2, lead);
        } else {
            const float lp = fmaxf((v - m) - logl, -1000.0f);
            // exp(lp) with what the product with log2 e rounds away (2^-24 of it: 2e-6 of p at lp = -20) put back
            const float t2 = lp * kLog2e;
            const float lo = __builtin_fmaf(lp, kLog2eLo, __builtin_fmaf(lp, kLog2e, -t2));
            const float e = __builtin_amdgcn_exp2f(t2);
            return -__builtin_fmaf(e, lo * kLn2, e) * __builtin_fmaf(h, lp, lead);
        }
    };
    auto put = [&](int i, float d) {
        if constexpr (kBf16) reinterpret_cast<uint16_t*>(dx)[i] = static_cast<uint16_t>(__builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){d, 0.0f}, bf16x2)));
        else reinterpret_cast<float*>(dx)[i] = d;
    };
    const int tl = run.tail() + tid;
    if (tl < n) put(tl, grad(run.one(tl)) + (tl == hit ? g : 0.0f));
#pragma unroll
    for (int j = 0; j < kBwdPieces; ++j) {
        const int p = tid + j * kThreads;
        if (p >= run.pieces) continue;
        float v[R::kPiece];
        R::unpack(w[j], v);
#pragma unroll
        for (int i = 0; i < R::kPiece; ++i) v[i] = grad(v[i]);
        if (hit >= 0 && hit / R::kPiece == p) {
#pragma unroll
            for (int i = 0; i < R::kPiece; ++i) v[i] += hit % R::kPiece == i ? g : 0.0f;
        }
        u32x4 o;
        if constexpr (kBf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){v[2 * i], v[2 * i + 1]}, bf16x2));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = __float_as_uint(v[i]);
        }
        auto* to = reinterpret_cast<typename R::Piece*>(dx + p * 16);
        if (a.far) __builtin_nontemporal_store(o, to);
        else *to = o;
    }
}

int launch_logprobs_bwd(LogprobBwdArgs a, int64_t rows, bool bf16, hipStream_t s) {
    a.seg_len = kBwdPieces * kThreads * (bf16 ? 8 : 4);
    // (256 MB of cache behind the L2s; 2048 rows of 100352 in fp32 308 us through them, 299 past them, 300 of 50277 in bf16 14.1
    // and 14.9)
    a.far = rows * a.V * (bf16 ? 2 : 4) > (256 << 20);
    a.segments = (a.V + a.seg_len - 1) / a.seg_len;
    // (a launch has fewer than 2^32 threads; one takes 335000 rows of 100352 in fp32, 135 GB)
    const int64_t most = 0x7fffff / a.segments;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const dim3 grid(static_cast<unsigned>(std::min(most, rows - a.row0) * a.segments));
        if (bf16) hipLaunchKernelGGL((logprob_bwd_kernel<true>), grid, dim3(kThreads), 0, s, a);
        else hipLaunchKernelGGL((logprob_bwd_kernel<false>), grid, dim3(kThreads), 0, s, a);
        DT_HIP_TRY(hipGetLastError());
    }
    return DT_OK;
}

int check_logits(int B, int T, int V, int64_t ldb, int64_t ldt, int token_bytes, int dtype, int mem) {
    if (B < 1 || T < 1 || V < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d, T=%d, V=%d must be >= 1", B, T, V);
    if (V > (1 << 24)) return set_error(DT_ERR_UNSUPPORTED, "V=%d exceeds %d", V, 1 << 24);
    if (static_cast<int64_t>(B) * T > 0x7fffff) return set_error(DT_ERR_UNSUPPORTED, "%lld rows", (long long)B * T);
    if (ldb < 0 || ldt < 0) return set_error(DT_ERR_INVALID_ARG, "strides %lld, %lld must be >= 0", (long long)ldb, (long long)ldt);
    if (token_bytes != 4 && token_bytes != 8) return set_error(DT_ERR_INVALID_ARG, "token_bytes=%d must be 4 or 8", token_bytes);
    if (dtype != DT_FP32_EXACT && dtype != DT_BF16) return set_error(DT_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (mem != DT_MEM_DEVICE && mem != DT_MEM_HOST) return set_error(DT_ERR_INVALID_ARG, "unknown mem %d", mem);
    return DT_OK;
}

bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_host_tokens(const void* tok, int token_bytes, int64_t rows, int V, int64_t ignore) {
    for (int64_t i = 0; i < rows; ++i) {
        const int64_t y = token_bytes == 8 ? static_cast<const int64_t*>(tok)[i] : static_cast<const int32_t*>(tok)[i];
        if (!is_skipped(y, ignore) && (y < 0 || y >= V))
            return set_error(DT_ERR_INVALID_ARG, "token %lld of row %lld outside [0, %d)", (long long)y, (long long)i, V);
    }
    return DT_OK;
}

// copies B x T rows of host logits into a staging buffer, densely
int stage_rows(void* dst, const void* src, int B, int T, int V, int64_t ldb, int64_t ldt, size_t es, hipStream_t s) {
    if ((T == 1 || ldt == V) && (B == 1 || ldb == static_cast<int64_t>(T) * V)) {
        DT_HIP_TRY(hipMemcpyAsync(dst, src, static_cast<size_t>(B) * T * V * es, hipMemcpyHostToDevice, s));
        return DT_OK;
    }
    for (int b = 0; b < B; ++b)
        for (int t = 0; t < T; ++t)
            DT_HIP_TRY(hipMemcpyAsync(static_cast<uint8_t*>(dst) + (static_cast<size_t>(b) * T + t) * V * es,
                                      static_cast<const uint8_t*>(src) + (b * ldb + t * ldt) * es, V * es, hipMemcpyHostToDevice, s));
    return DT_OK;
}

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" {

int dt_token_logprobs_workspace(int B, int T, int V, int top_k, int64_t* bytes) {
    clear_error();
    if (!bytes) return set_error(DT_ERR_INVALID_ARG, "bytes is NULL");
    DT_TRY(check_logits(B, T, V, 0, 0, 4, DT_BF16, DT_MEM_DEVICE));
    if (top_k < 0 || top_k > kMaxTop || top_k > V)
        return set_error(DT_ERR_INVALID_ARG, "top_k=%d outside [0, %d]", top_k, std::min(kMaxTop, V));
    *bytes = workspace_bytes(static_cast<int64_t>(B) * T, V, top_k);
    return DT_OK;
}

int dt_token_logprobs(dt_ctx* ctx, const void* logits, const void* tokens, int B, int T, int V, int64_t ldb, int64_t ldt,
                      int token_bytes, int64_t ignore_index, int top_k, float* logprob, float* entropy, float* m, float* l,
                      int32_t* top_index, float* top_logprob, void* ws, int64_t ws_bytes, int dtype, int mem, void* stream) {
    clear_error();
    if (!logits || !tokens || !logprob || !m || !l)
        return set_error(DT_ERR_INVALID_ARG, "logits, tokens, logprob, m and l must be non-NULL");
    DT_TRY(check_logits(B, T, V, ldb, ldt, token_bytes, dtype, mem));
    if (top_k < 0 || top_k > kMaxTop || top_k > V)
        return set_error(DT_ERR_INVALID_ARG, "top_k=%d outside [0, %d]", top_k, std::min(kMaxTop, V));
    if (top_k > 0 && (!top_index || !top_logprob))
        return set_error(DT_ERR_INVALID_ARG, "top_index and top_logprob must be non-NULL with top_k=%d", top_k);
    const int64_t rows = static_cast<int64_t>(B) * T;
    const int64_t need = workspace_bytes(rows, V, top_k);
    const size_t es = dtype == DT_BF16 ? 2 : 4;
    if (mem == DT_MEM_DEVICE) {
        if (!aligned_to(logits, es) || !aligned_to(tokens, token_bytes))
            return set_error(DT_ERR_INVALID_ARG, "logits or tokens are not aligned to their type");
        if (!aligned16(ws)) return set_error(DT_ERR_INVALID_ARG, "the workspace must be 16-byte aligned");
        if (need > 0 && (!ws || ws_bytes < need))
            return set_error(DT_ERR_INVALID_ARG, "the workspace has %lld bytes, the call needs %lld", (long long)(ws ? ws_bytes : 0), (long long)need);
    } else {
        DT_TRY(check_host_tokens(tokens, token_bytes, rows, V, ignore_index));
    }
    if (!ctx) return set_error(DT_ERR_INVALID_ARG, "ctx is NULL");
    DeviceScope scope;
    DT_TRY(scope.enter(ctx->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    LogprobArgs a{};
    a.x = logits;
    a.tok = tokens;
    a.ldb = ldb;
    a.ldt = ldt;
    a.ignore = ignore_index;
    a.tok64 = token_bytes == 8;
    a.T = T;
    a.V = V;
    a.k = top_k;
    a.logprob = logprob;
    a.entropy = entropy;
    a.m = m;
    a.l = l;
    a.top_index = top_index;
    a.top_logprob = top_logprob;
    if (mem == DT_MEM_DEVICE) return launch_logprobs(a, rows, dtype == DT_BF16, ws, s);

    const size_t nk = static_cast<size_t>(rows) * top_k;
    DT_TRY(ctx->stage[0].ensure(rows * V * es));
    DT_TRY(ctx->stage[1].ensure(rows * token_bytes));
    DT_TRY(ctx->stage[2].ensure(rows * 4 * sizeof(float)));
    DT_TRY(ctx->stage[3].ensure(nk * 8 + 16));
    if (need > 0) DT_TRY(ctx->stage[4].ensure(need));
    DT_TRY(stage_rows(ctx->stage[0].ptr, logits, B, T, V, ldb, ldt, es, s));
    DT_HIP_TRY(hipMemcpyAsync(ctx->stage[1].ptr, tokens, rows * token_bytes, hipMemcpyHostToDevice, s));
    a.x = ctx->stage[0].ptr;
    a.tok = ctx->stage[1].ptr;
    a.ldt = V;
    a.ldb = static_cast<int64_t>(T) * V;
    a.logprob = static_cast<float*>(ctx->stage[2].ptr);
    a.entropy = a.logprob + rows;
    a.m = a.logprob + 2 * rows;
    a.l = a.logprob + 3 * rows;
    a.top_index = static_cast<int32_t*>(ctx->stage[3].ptr);
    a.top_logprob = reinterpret_cast<float*>(a.top_index + nk);
    DT_TRY(launch_logprobs(a, rows, dtype == DT_BF16, ctx->stage[4].ptr, s));
    DT_HIP_TRY(hipMemcpyAsync(logprob, a.logprob, rows * 4, hipMemcpyDeviceToHost, s));
    if (entropy) DT_HIP_TRY(hipMemcpyAsync(entropy, a.entropy, rows * 4, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipMemcpyAsync(m, a.m, rows * 4, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipMemcpyAsync(l, a.l, rows * 4, hipMemcpyDeviceToHost, s));
    if (nk) {
        DT_HIP_TRY(hipMemcpyAsync(top_index, a.top_index, nk * 4, hipMemcpyDeviceToHost, s));
        DT_HIP_TRY(hipMemcpyAsync(top_logprob, a.top_logprob, nk * 4, hipMemcpyDeviceToHost, s));
    }
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

int dt_token_logprobs_bwd(dt_ctx* ctx, const float* d_logprob, const float* d_entropy, const void* logits, const void* tokens,
                          const float* m, const float* l, const float* entropy, int B, int T, int V, int64_t ldb, int64_t ldt,
                          int token_bytes, int64_t ignore_index, void* d_logits, int64_t ldb_out, int64_t ldt_out, int dtype,
                          int mem, void* stream) {
    clear_error();
    if (!d_logprob || !logits || !tokens || !m || !l || !d_logits)
        return set_error(DT_ERR_INVALID_ARG, "d_logprob, logits, tokens, m, l and d_logits must be non-NULL");
    if (d_entropy && !entropy) return set_error(DT_ERR_INVALID_ARG, "entropy must be non-NULL with d_entropy");
    DT_TRY(check_logits(B, T, V, ldb, ldt, token_bytes, dtype, mem));
    // (either dimension's rows may lie between the other's)
    const bool by_b = (T == 1 || ldt_out >= V) && (B == 1 || ldb_out >= (T - 1) * ldt_out + V);
    const bool by_t = (B == 1 || ldb_out >= V) && (T == 1 || ldt_out >= (B - 1) * ldb_out + V);
    if (!(by_b || by_t) || ldb_out < 0 || ldt_out < 0)
        return set_error(DT_ERR_INVALID_ARG, "rows of d_logits %lld and %lld apart overlap", (long long)ldb_out, (long long)ldt_out);
    const int64_t rows = static_cast<int64_t>(B) * T;
    const size_t es = dtype == DT_BF16 ? 2 : 4;
    if (mem == DT_MEM_DEVICE) {
        if (!aligned_to(logits, es) || !aligned_to(d_logits, es) || !aligned_to(tokens, token_bytes))
            return set_error(DT_ERR_INVALID_ARG, "logits, d_logits or tokens are not aligned to their type");
    } else {
        DT_TRY(check_host_tokens(tokens, token_bytes, rows, V, ignore_index));
    }
    if (!ctx) return set_error(DT_ERR_INVALID_ARG, "ctx is NULL");
    DeviceScope scope;
    DT_TRY(scope.enter(ctx->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    LogprobBwdArgs a{};
    a.x = logits;
    a.dx = d_logits;
    a.tok = tokens;
    a.g = d_logprob;
    a.h = d_entropy;
    a.m = m;
    a.l = l;
    a.entropy = entropy;
    a.ldb = ldb;
    a.ldt = ldt;
    a.ldb_out = ldb_out;
    a.ldt_out = ldt_out;
    a.ignore = ignore_index;
    a.tok64 = token_bytes == 8;
    a.T = T;
    a.V = V;
    if (mem == DT_MEM_DEVICE) return launch_logprobs_bwd(a, rows, dtype == DT_BF16, s);

    DT_TRY(ctx->stage[0].ensure(rows * V * es));
    DT_TRY(ctx->stage[1].ensure(rows * token_bytes));
    DT_TRY(ctx->stage[2].ensure(rows * 5 * sizeof(float)));
    DT_TRY(stage_rows(ctx->stage[0].ptr, logits, B, T, V, ldb, ldt, es, s));
    DT_HIP_TRY(hipMemcpyAsync(ctx->stage[1].ptr, tokens, rows * token_bytes, hipMemcpyHostToDevice, s));
    float* st = static_cast<float*>(ctx->stage[2].ptr);
    const float* src[5] = {d_logprob, m, l, d_entropy, d_entropy ? entropy : nullptr};
    for (int i = 0; i < 5; ++i)
        if (src[i]) DT_HIP_TRY(hipMemcpyAsync(st + i * rows, src[i], rows * 4, hipMemcpyHostToDevice, s));
    a.x = a.dx = ctx->stage[0].ptr;  // (in place)
    a.tok = ctx->stage[1].ptr;
    a.g = st;
    a.m = st + rows;
    a.l = st + 2 * rows;
    a.h = d_entropy ? st + 3 * rows : nullptr;
    a.entropy = st + 4 * rows;
    a.ldt = a.ldt_out = V;
    a.ldb = a.ldb_out = static_cast<int64_t>(T) * V;
    DT_TRY(launch_logprobs_bwd(a, rows, dtype == DT_BF16, s));
    for (int b = 0; b < B; ++b)
        for (int t = 0; t < T; ++t)
            DT_HIP_TRY(hipMemcpyAsync(static_cast<uint8_t*>(d_logits) + (b * ldb_out + t * ldt_out) * es,
                                      static_cast<uint8_t*>(ctx->stage[0].ptr) + (static_cast<size_t>(b) * T + t) * V * es, V * es,
                                      hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

}  // extern "C"
