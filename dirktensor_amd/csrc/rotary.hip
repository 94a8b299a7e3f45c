// Rotation of queries and keys to their positions, with or without each head's RMSNorm in the same pass, and the gradients.
//
// A pair (a, b) of a head's values, of those that turn (the first `dims` of 128: d and d + dims/2, or 2i and 2i + 1), at
// position p goes to
//   a' = mag (a cos t - b sin t),   b' = mag (b cos t + a sin t),   t = p f_i
// and the rest of the head stays. With the norm, y = x inv w with inv = 1 / sqrt(mean x^2 + eps) over the head is what turns.
// Gradients: g = the rotation's transpose (angle -t) of the output's gradient; with the norm, n = x inv,
//   dx = inv (w g - n mean(w g n)),   dw = sum over tokens and heads of g n.
//
// All of it is bound by HBM (each value is read and written once), where it is not bound by the launch.
//
// A wave takes eight heads of one token, eight lanes a head, 16 values a lane in pieces of 16 bytes: both values of each pair lie in one
// lane, the eight lanes' pieces beside each other (in fp32 four pieces a lane; four of a lane behind each other took 198 in place of
// 104 us past the caches), and a head's sums are three lane exchanges away. The angles need no table: lane i works out pair i's angle for the token, in 64
// bits down to a fraction of a quarter turn, and the lanes read the pairs that they need from LDS; so no table bounds the positions, and
// nothing is fetched for them. An angle is off by 3 2^-53 of itself and, from the fraction's rounding to 32 bits, by 2.4 10^-8 radians: the second is the
// larger up to 2^26 radians, and near 2^53 nothing is left of a position's fraction.
//
// Measured, 128 values a head: 8 tokens of 16 heads, 4.0 us, a launch; 12 x 5 with the norm 4.4; 2 x 8192 tokens of 16 heads and 16 key
// heads in fp32, 537 MB, 88 (6.1 TB/s, where the best copy reaches 6.25); 4 x 4096 of 16 and 16 in bf16 with the norm, 268 MB, 54 (5.0);
// the gradients of 4 x 8192 of 16 and 4 in bf16, 503 MB, 91 (5.5) and 5.0 for the weights' columns; of 777 of 16 and 16 in fp32, 38 MB,
// 11.1 and 3.8: 1536 waves have one part of a token there and 18 of them a second one, so it is twice the chain of positions, angles, values, and the
// columns' sums over lanes and waves; adding the workgroups' columns in the same launch would need a counter that nothing has cleared.

#include "dt_internal.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace dt {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPairs = DT_HEAD_DIM / 2;
constexpr int kGroupHeads = 8;  // heads of a wave
constexpr int kFewRows = 32;
constexpr int kMaxHeads = 1024;
constexpr int kGridRows = 32768;  // batch rows of the grid's second dimension
constexpr int kCus = 256;
constexpr int kBwdGroups = 3 * kCus;
constexpr int64_t kCacheBytes = 256 << 20;

// kRows: places for the batch rows' first positions, by value
template <int kRows>
struct RotaryArgs {
    const void* in[2];    // q, k rows (of the backward: the outputs' gradients)
    const void* x[2];     // backward with norm: the forward's inputs
    void* out[2];
    const float* w[2];    // norm weights [128]
    float* dw[2];         // their gradients
    float* partial;       // [blocks][128] column sums, q's blocks first
    int64_t ld_in[2], ld_x[2], ld_out[2];
    const void* positions;  // [tokens], or NULL: start[b] + t
    int pos_bytes;
    int has_starts;       // start is set (otherwise there may be more rows than places)
    int tokens, B, T;
    int heads[2];
    int octets;           // dims / 16
    int blocks[2];        // backward: workgroups of q, of k
    int parts[2];         // of a token's heads, one wave's each
    float mag, sign, eps;
    double turns[kPairs];  // a position's step of each pair, in whole turns
    int32_t start[kRows];
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){lo, hi}, bf16x2));
}

template <bool kBf16>
constexpr int kPer = kBf16 ? 8 : 4;  // values of a piece

// kPast: past the caches
template <bool kBf16, bool kPast>
__device__ __forceinline__ u32x4 load_piece(const void* p, int64_t at) {
    const u32x4* from = reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + at * (kBf16 ? 2 : 4));
    if constexpr (kPast) return __builtin_nontemporal_load(from);
    else return *from;
}
template <bool kBf16>
__device__ __forceinline__ void open_piece(u32x4 w, float (&x)[kPer<kBf16>]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kBf16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            x[i] = __uint_as_float(w[i]);
        }
    }
}
template <bool kBf16, bool kPast>
__device__ __forceinline__ void store_piece(void* p, int64_t at, const float (&x)[kPer<kBf16>]) {
    u32x4 w;
    u32x4* to;
    if constexpr (kBf16) {
        w = (u32x4){pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7])};
        to = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at);
    } else {
        w = (u32x4){__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
        to = reinterpret_cast<u32x4*>(static_cast<float*>(p) + at);
    }
    if constexpr (kPast) __builtin_nontemporal_store(w, to);
    else *to = w;
}

// A lane's 16 values as pieces, and where they lie in the head. In the half layout two pieces go together, number t and t + dims/2 (in
// pieces); those that do not turn are taken two by two. In the interleaved layout a piece has whole pairs.
template <bool kBf16, bool kInter>
struct Pieces {
    static constexpr int P = kPer<kBf16>, kN = 16 / P;
    float x[kN][P];

    static __device__ __forceinline__ int offset(int i, int lane, int octets) {
        const int t = (lane & 7) + (i >> 1) * 8;
        if constexpr (kInter) return (t + (i & 1) * (8 * kN / 2)) * P;
        const int half = octets * (8 / P);
        return (t < half ? t + (i & 1) * half : 2 * t + (i & 1)) * P;
    }
    // as loaded, and as values
    struct Raw {
        u32x4 w[kN];
        template <bool kPast>
        __device__ __forceinline__ void load(const void* p, int64_t head, int lane, int octets) {
#pragma unroll
            for (int i = 0; i < kN; ++i) w[i] = load_piece<kBf16, kPast>(p, head + offset(i, lane, octets));
        }
    };
    __device__ __forceinline__ void open(const Raw& r) {
#pragma unroll
        for (int i = 0; i < kN; ++i) open_piece<kBf16>(r.w[i], x[i]);
    }
    template <bool kPast>
    __device__ __forceinline__ void load(const void* p, int64_t head, int lane, int octets) {
        Raw r;
        r.template load<kPast>(p, head, lane, octets);
        open(r);
    }
    template <bool kPast>
    __device__ __forceinline__ void store(void* p, int64_t head, int lane, int octets) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) store_piece<kBf16, kPast>(p, head + offset(i, lane, octets), x[i]);
    }
    // the same places of a row of fp32
    __device__ __forceinline__ void load_row(const float* p, int lane, int octets) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int at = offset(i, lane, octets);
#pragma unroll
            for (int j = 0; j < P; j += 4) {
                const floatx4 w = *reinterpret_cast<const floatx4*>(p + at + j);
                x[i][j] = w[0], x[i][j + 1] = w[1], x[i][j + 2] = w[2], x[i][j + 3] = w[3];
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kN; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) x[i][j] = 0.0f;
    }
    static __device__ __forceinline__ void turn_pair(float& u, float& v, float2 f) {
        const float p = u, r = v;
        u = p * f.x - r * f.y;
        v = r * f.x + p * f.y;
    }
    __device__ __forceinline__ void turn(const float2* cs, int lane, int octets) {
        if constexpr (kInter) {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int at = offset(i, lane, octets);
                if (at < 16 * octets) {
#pragma unroll
                    for (int j = 0; j < P / 2; ++j) turn_pair(x[i][2 * j], x[i][2 * j + 1], cs[at / 2 + j]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; i += 2) {
                const int at = offset(i, lane, octets);
                if (at < 8 * octets) {
#pragma unroll
                    for (int j = 0; j < P; ++j) turn_pair(x[i][j], x[i + 1][j], cs[at + j]);
                }
            }
        }
    }
};

// the position of token t of batch row b
template <int kRows>
__device__ __forceinline__ double position(const RotaryArgs<kRows>& a, int b, int t) {
    if (a.positions) {
        const int64_t token = static_cast<int64_t>(b) * a.T + t;
        return a.pos_bytes == 4 ? static_cast<const int32_t*>(a.positions)[token]
                                : static_cast<double>(static_cast<const int64_t*>(a.positions)[token]);
    }
    return static_cast<double>(a.has_starts ? a.start[b] : 0) + t;
}

// cos and sin (times mag) of the pairs at a position into the wave's part of LDS
template <int kRows>
__device__ __forceinline__ void angles(const RotaryArgs<kRows>& a, double at, int lane, float2* cs) {
    if (lane < 8 * a.octets) {
        double t = at * a.turns[lane];
        t = 4.0 * (t - rint(t));       // quarter turns, in [-2, 2]
        const double q = rint(t);
        float s, c;
        sincospif(0.5f * static_cast<float>(t - q), &s, &c);  // (of at most an eighth of a turn)
        const int quarter = static_cast<int>(q);
        if (quarter & 1) {
            const float u = s;
            s = c, c = -u;
        }
        if (quarter & 2) s = -s, c = -c;
        cs[lane] = make_float2(a.mag * c, a.mag * a.sign * s);
    }
    // (the wave's own part: its accesses are in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// over the eight lanes of a head: with the neighbour, the other pair of four, and mirrored
template <int kCtrl>
__device__ __forceinline__ float moved(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum_head(float x) {
    x += moved<0xb1>(x);
    x += moved<0x4e>(x);
    return x + moved<0x141>(x);
}
// with the other row of 16 of a half, with the other half
template <bool k32>
__device__ __forceinline__ float sum_halves(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto r = k32 ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// 1 / sqrt(x): the instruction's, once corrected
__device__ __forceinline__ float inverse_root(float x) {
    const float r = __builtin_amdgcn_rsqf(x);
    return fmaf(r, fmaf(-0.5f * x * r, r, 0.5f), r);
}

// 1 / sqrt(mean x^2 + eps) of the head
template <bool kBf16, bool kInter>
__device__ __forceinline__ float inverse_rms(const Pieces<kBf16, kInter>& v, float eps) {
    using V = Pieces<kBf16, kInter>;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += v.x[i / V::P][i % V::P] * v.x[i / V::P][i % V::P];
    ss = sum_head(ss);
    float inv = inverse_root(fmaf(ss, 1.0f / DT_HEAD_DIM, eps));
    // Squares past fp32's range: once more, of values 2^-70 times as large. (An infinity among the values has a sum that stays one, and
    // the factor 0: finite values of its head become 0, as the formula has it, the infinity NaN.)
    if (__any(ss == __builtin_huge_valf())) {
        float s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = v.x[i / V::P][i % V::P] * 0x1p-70f;
            s2 += y * y;
        }
        s2 = sum_head(s2);
        if (ss == __builtin_huge_valf()) inv = s2 == __builtin_huge_valf() ? 0.0f : 0x1p-70f * inverse_root(s2 * (1.0f / DT_HEAD_DIM));
    }
    return inv;
}

// A workgroup takes a token, its waves the groups of eight heads: q's, then k's.
template <bool kBf16, bool kNorm, bool kInter, bool kPast, int kRows>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs<kRows> a) {
    using V = Pieces<kBf16, kInter>;
    __shared__ float2 cs[kWaves][kPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x, b = blockIdx.z * kGridRows + blockIdx.y;
    if (b >= a.B) return;
    const int64_t token = static_cast<int64_t>(b) * a.T + t;
    for (int first = wave * kGroupHeads; first < a.heads[0] + a.heads[1]; first += blockDim.x / 64 * kGroupHeads) {
        int head = first + (lane >> 3);
        const bool second = head >= a.heads[0];
        if (second) head -= a.heads[0];
        const bool have = !second || head < a.heads[1];
        V x, w;
        if (have) x.template load<kPast>(second ? a.in[1] : a.in[0], token * (second ? a.ld_in[1] : a.ld_in[0]) + head * DT_HEAD_DIM, lane, a.octets);
        else x.zero();
        if constexpr (kNorm) w.load_row(second && have ? a.w[1] : a.w[0], lane, a.octets);
        if (first == wave * kGroupHeads) angles(a, position(a, b, t), lane, cs[wave]);
        if constexpr (kNorm) {
            const float inv = inverse_rms(x, a.eps);
#pragma unroll
            for (int i = 0; i < 16; ++i) x.x[i / V::P][i % V::P] = x.x[i / V::P][i % V::P] * inv * w.x[i / V::P][i % V::P];
        }
        x.turn(cs[wave], lane, a.octets);
        if (have)
            x.template store<kPast>(second ? a.out[1] : a.out[0], token * (second ? a.ld_out[1] : a.ld_out[0]) + head * DT_HEAD_DIM, lane, a.octets);
    }
}

// The norm's backward: workgroups of q (the first blocks[0]) or of k; their waves take tokens (or, where these are few, their groups of
// eight heads) in turn, and each workgroup leaves the column sums of g n.
template <bool kBf16, bool kInter, bool kPast, int kRows>
__global__ __launch_bounds__(kThreads) void head_norm_rotary_bwd_kernel(RotaryArgs<kRows> a) {
    using V = Pieces<kBf16, kInter>;
    __shared__ float2 cs[kWaves][kPairs];
    __shared__ float sums[kWaves][DT_HEAD_DIM];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int which = static_cast<int>(blockIdx.x) >= a.blocks[0];
    const int block = blockIdx.x - (which ? a.blocks[0] : 0);
    const int heads = a.heads[which], step = a.blocks[which] * kWaves;
    const int parts = a.parts[which], span = parts > 1 ? kGroupHeads : heads;  // of a token, heads of a part
    V w, dw;
    w.load_row(a.w[which], lane, a.octets);
    dw.zero();
    // The next eight heads' values are under way while some are worked on. (Lanes without a head read another's, and behind the last
    // token it is read again: a load under a condition would make the wait for one a wait for all.)
    typename V::Raw next_g, next_x;
    const auto fetch = [&](int token, int first) {
        token = min(token, a.tokens - 1);
        const int head = min(first + (lane >> 3), heads - 1);
        next_g.template load<kPast>(a.in[which], token * a.ld_in[which] + head * DT_HEAD_DIM, lane, a.octets);
        next_x.template load<kPast>(a.x[which], token * a.ld_x[which] + head * DT_HEAD_DIM, lane, a.octets);
    };
    // token and part, row and place in the row: divided once (a step is 3072 tokens at most, and as many rows where these have one)
    const int item = block * kWaves + wave;
    int token = item / parts, part = item - token * parts, b = token / a.T, t = token - b * a.T;
    const int step_token = step / parts, step_part = step - step_token * parts;
    const int step_b = step_token / a.T, step_t = step_token - step_b * a.T;
    if (token < a.tokens) fetch(token, part * span);
    while (token < a.tokens) {
        angles(a, position(a, b, t), lane, cs[wave]);
        int next_token = token + step_token, next_part = part + step_part;
        if (next_part >= parts) next_part -= parts, ++next_token;
        const int end = min(part * span + span, heads);
        for (int first = part * span; first < end; first += kGroupHeads) {
            const int head = first + (lane >> 3);
            const bool have = head < end, more = first + kGroupHeads < end;
            V g, x;
            g.open(next_g);
            x.open(next_x);
            fetch(more ? token : next_token, more ? first + kGroupHeads : next_part * span);
            if (!have) g.zero(), x.zero();
            g.turn(cs[wave], lane, a.octets);
            const float inv = inverse_rms(x, a.eps);
            float dot = 0.0f;
#pragma unroll
            for (int i = 0; i < V::kN; ++i)
#pragma unroll
                for (int j = 0; j < V::P; ++j) {
                    x.x[i][j] *= inv;
                    dw.x[i][j] += g.x[i][j] * x.x[i][j];
                    g.x[i][j] *= w.x[i][j];
                    dot += g.x[i][j] * x.x[i][j];
                }
            dot = sum_head(dot) * (1.0f / DT_HEAD_DIM);
#pragma unroll
            for (int i = 0; i < V::kN; ++i)
#pragma unroll
                for (int j = 0; j < V::P; ++j) g.x[i][j] = inv * (g.x[i][j] - x.x[i][j] * dot);
            if (have) g.template store<kPast>(a.out[which], token * a.ld_out[which] + head * DT_HEAD_DIM, lane, a.octets);
        }
        b += step_b;
        t += step_t + (next_token - token - step_token);  // (one more where the parts pass a token's end: less than 2 T)
        if (t >= a.T) t -= a.T, ++b;
        token = next_token;
        part = next_part;
    }
    // the eight heads of a wave, then the waves
#pragma unroll
    for (int i = 0; i < V::kN; ++i)
#pragma unroll
        for (int j = 0; j < V::P; ++j) {
            float s = dw.x[i][j];
            s += moved<0x128>(s);  // rotated by 8 within 16
            s = sum_halves<true>(sum_halves<false>(s));
            if (lane < 8) sums[wave][V::offset(i, lane, a.octets) + j] = s;
        }
    __syncthreads();
    if (threadIdx.x < DT_HEAD_DIM) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) s += sums[i][threadIdx.x];
        a.partial[static_cast<int64_t>(blockIdx.x) * DT_HEAD_DIM + threadIdx.x] = s;
    }
}

// The workgroups' column sums, added in a fixed order: 16 columns of q or k a workgroup, 16 runs of rows.
constexpr int kSumCols = 16;
__global__ __launch_bounds__(kThreads) void head_norm_dw_kernel(const float* partial, int q_blocks, int k_blocks, float* dq, float* dk) {
    __shared__ float red[kThreads / kSumCols][kSumCols + 1];
    const int which = blockIdx.y, rows = which ? k_blocks : q_blocks;
    const float* p = partial + (which ? static_cast<int64_t>(q_blocks) * DT_HEAD_DIM : 0);
    const int c = threadIdx.x % kSumCols, r = threadIdx.x / kSumCols, col = blockIdx.x * kSumCols + c;
    float s = 0.0f;
#pragma unroll 8
    for (int i = r; i < rows; i += kThreads / kSumCols) s += p[static_cast<int64_t>(i) * DT_HEAD_DIM + col];
    red[r][c] = s;
    __syncthreads();
    if (r == 0) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < kThreads / kSumCols; ++i) s += red[i][c];
        (which ? dk : dq)[col] = s;
    }
}

struct Call {
    const void *q, *k, *xq, *xk;
    void *oq, *ok;
    const float *wq, *wk;
    float *dwq, *dwk;
    int B, T, H, Hk, D;
    int64_t ldq, ldk, ldxq, ldxk, ldoq, ldok;
    const void* positions;
    int pos_bytes;
    const int32_t* starts;
    const dt_rotary* rot;
    float eps;
    int dtype, mem;
    bool norm, backward;
};

bool good_magnitude(double m) {  // (the kernels have it in 32 bits)
    const float f = static_cast<float>(m);
    return std::isfinite(f) && f >= 0x1p-126f;
}

bool good_rotary(const dt_rotary* r) {
    if (r->dims < 16 || r->dims > DT_HEAD_DIM || r->dims % 16) return false;
    if (r->layout != DT_ROTARY_HALF && r->layout != DT_ROTARY_INTERLEAVED) return false;
    if (!good_magnitude(r->magnitude)) return false;
    for (int i = 0; i < r->dims / 2; ++i)
        if (!std::isfinite(r->frequency[i])) return false;
    return true;
}

int check_most(int B, int T, int H, int Hk) {
    if (H + static_cast<int64_t>(Hk) > kMaxHeads) return set_error(DT_ERR_UNSUPPORTED, "%d and %d heads are more than %d", H, Hk, kMaxHeads);
    // (a launch's threads and the indices of groups of heads stay within 31 bits)
    if (static_cast<int64_t>(B) * T > 0x7fffff) return set_error(DT_ERR_UNSUPPORTED, "B*T = %lld tokens", (long long)B * T);
    return DT_OK;
}

int check_call(const dt_ctx* ctx, const Call& c) {
    if (c.B < 1 || c.T < 1 || c.H < 1 || c.Hk < 0)
        return set_error(DT_ERR_INVALID_ARG, "B=%d, T=%d, H=%d must be >= 1, Hk=%d >= 0", c.B, c.T, c.H, c.Hk);
    if (!c.q || !c.oq) return set_error(DT_ERR_INVALID_ARG, "q and its output must be non-NULL");
    if (!c.rot) return set_error(DT_ERR_INVALID_ARG, "rotary is NULL");
    if (!good_rotary(c.rot))
        return set_error(DT_ERR_INVALID_ARG, "the rotary needs dims of 16, 32 .. %d, a known layout, a magnitude above 0 and finite frequencies", DT_HEAD_DIM);
    if (c.D != DT_HEAD_DIM) return set_error(DT_ERR_UNSUPPORTED, "head_dim D=%d, kernels are built for D=%d", c.D, DT_HEAD_DIM);
    DT_TRY(check_most(c.B, c.T, c.H, c.Hk));
    if (c.Hk > 0 && (!c.k || !c.ok)) return set_error(DT_ERR_INVALID_ARG, "k and its output must be non-NULL with Hk=%d", c.Hk);
    if (c.Hk > 0 && (c.oq == c.ok || c.oq == c.k || c.ok == c.q || (c.xk && (c.oq == c.xk || c.ok == c.xq))))
        return set_error(DT_ERR_INVALID_ARG, "an output is the other's, or the other's input");
    if (c.dtype != DT_FP32_EXACT && c.dtype != DT_BF16) return set_error(DT_ERR_INVALID_ARG, "unknown dtype %d", c.dtype);
    if (c.mem != DT_MEM_DEVICE && c.mem != DT_MEM_HOST) return set_error(DT_ERR_INVALID_ARG, "unknown mem %d", c.mem);
    if (c.positions && c.starts) return set_error(DT_ERR_INVALID_ARG, "positions and starts exclude each other");
    if (c.positions && c.pos_bytes != 4 && c.pos_bytes != 8)
        return set_error(DT_ERR_INVALID_ARG, "pos_bytes=%d must be 4 or 8", c.pos_bytes);
    if (c.starts && c.B > kMaxRaggedBatch) return set_error(DT_ERR_UNSUPPORTED, "B=%d > %d rows with starts", c.B, kMaxRaggedBatch);
    if (c.norm && (!c.wq || (c.Hk > 0 && !c.wk))) return set_error(DT_ERR_INVALID_ARG, "norm weights must be non-NULL");
    if (c.norm && (!(c.eps >= 1e-30f) || !std::isfinite(c.eps))) return set_error(DT_ERR_INVALID_ARG, "eps %g must be at least 1e-30", c.eps);
    if (c.norm && c.backward && (!c.xq || !c.dwq || (c.Hk > 0 && (!c.xk || !c.dwk))))
        return set_error(DT_ERR_INVALID_ARG, "the forward's inputs and the weights' gradients must be non-NULL");
    const int64_t dq = static_cast<int64_t>(c.H) * DT_HEAD_DIM, dk = static_cast<int64_t>(c.Hk) * DT_HEAD_DIM;
    const bool xs = c.norm && c.backward;
    if (c.ldq < dq || c.ldoq < dq || (xs && c.ldxq < dq) || (c.Hk > 0 && (c.ldk < dk || c.ldok < dk || (xs && c.ldxk < dk))))
        return set_error(DT_ERR_INVALID_ARG, "row strides are below the heads' %lld or %lld values", (long long)dq, (long long)dk);
    if (c.mem == DT_MEM_DEVICE) {
        const int64_t per = c.dtype == DT_BF16 ? 8 : 4;
        bool bad = !aligned16(c.q) || !aligned16(c.oq) || c.ldq % per || c.ldoq % per;
        if (c.Hk > 0) bad = bad || !aligned16(c.k) || !aligned16(c.ok) || c.ldk % per || c.ldok % per;
        if (xs) bad = bad || !aligned16(c.xq) || c.ldxq % per || (c.Hk > 0 && (!aligned16(c.xk) || c.ldxk % per));
        if (c.norm) bad = bad || !aligned16(c.wq) || (c.Hk > 0 && !aligned16(c.wk));
        if (bad) return set_error(DT_ERR_INVALID_ARG, "device rows, their strides and norm weights must be 16-byte aligned");
        if (c.positions && reinterpret_cast<uintptr_t>(c.positions) % c.pos_bytes)
            return set_error(DT_ERR_INVALID_ARG, "positions are not aligned to their size");
    }
    // (rows that another row's results would overwrite)
    const auto shifted = [&](const void* in, const void* out, int64_t ld_in, int64_t ld_out) { return in == out && ld_in != ld_out; };
    if (static_cast<int64_t>(c.B) * c.T > 1 &&
        (shifted(c.q, c.oq, c.ldq, c.ldoq) || (xs && shifted(c.xq, c.oq, c.ldxq, c.ldoq)) ||
         (c.Hk > 0 && (shifted(c.k, c.ok, c.ldk, c.ldok) || (xs && shifted(c.xk, c.ok, c.ldxk, c.ldok))))))
        return set_error(DT_ERR_INVALID_ARG, "an output in its input's place needs the same stride");
    if (!ctx) return set_error(DT_ERR_INVALID_ARG, "ctx is NULL");
    return DT_OK;
}

// Workgroups of the norm's backward for `heads` heads beside `others`: their share of as many as fit the CUs by the groups of eight,
// as a group that is not full takes as long, so that q's and k's end together and the sums that they leave stay few.
// parts: a wave has a whole token's heads, whose angles are worked out once then, where that leaves waves enough.
int bwd_blocks(int64_t tokens, int heads, int others, int* parts) {
    const int groups = (heads + kGroupHeads - 1) / kGroupHeads, all = groups + (others + kGroupHeads - 1) / kGroupHeads;
    const int most = std::max(1, kBwdGroups * groups / all);
    *parts = tokens < static_cast<int64_t>(most) * kWaves ? groups : 1;
    return static_cast<int>(std::min<int64_t>((tokens * *parts + kWaves - 1) / kWaves, most));
}

template <int kRows>
int launch_rows(const Call& c, void* ws, hipStream_t s) {
    RotaryArgs<kRows> a{};
    a.in[0] = c.q, a.in[1] = c.k;
    a.x[0] = c.xq, a.x[1] = c.xk;
    a.out[0] = c.oq, a.out[1] = c.ok;
    a.w[0] = c.wq, a.w[1] = c.wk;
    a.ld_in[0] = c.ldq, a.ld_in[1] = c.ldk;
    a.ld_x[0] = c.ldxq, a.ld_x[1] = c.ldxk;
    a.ld_out[0] = c.ldoq, a.ld_out[1] = c.ldok;
    a.positions = c.positions;
    a.pos_bytes = c.pos_bytes;
    a.tokens = c.B * c.T;
    a.B = c.B;
    a.T = c.T;
    a.has_starts = c.starts != nullptr;
    a.heads[0] = c.H, a.heads[1] = c.Hk;
    a.octets = c.rot->dims / 16;
    a.mag = static_cast<float>(c.rot->magnitude);
    a.sign = c.backward ? -1.0f : 1.0f;
    a.eps = c.eps;
    for (int i = 0; i < c.rot->dims / 2; ++i) a.turns[i] = c.rot->frequency[i] / 6.283185307179586476925;
    if (c.starts) std::copy_n(c.starts, c.B, a.start);
    const bool bf16 = c.dtype == DT_BF16, inter = c.rot->layout == DT_ROTARY_INTERLEAVED;
    const dim3 block(kThreads);
    // Rows that the last-level cache (256 MB) cannot hold go past it: 537 MB moved in fp32 95 us, 88 past it. Smaller results stay in it, as
    // what follows reads them. With 67 to 168 MB stored past it the norm alone took 53.8 us in place of 55.9 (134 MB, calls back to back on
    // new inputs) or 72 in place of 70 (one call); with an operator behind it that reads the results it was 91 in place of 86 (134 MB, elementwise),
    // 175 in place of 171 (67 MB, attention), 42 in place of 39 (84 MB) and 62 in place of 63 (101 MB, keys into a cache); the gradient of
    // 67 to 101 MB with such a reader 3 to 4 us more of 61 to 86.
    const int64_t bytes = static_cast<int64_t>(a.tokens) * (c.H + c.Hk) * DT_HEAD_DIM * (bf16 ? 2 : 4);
    const bool past = bytes * (c.norm && c.backward ? 2 : 1) >= kCacheBytes;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    const auto choose = [&](bool which, auto go) {
        if (which) go(yes);
        else go(no);
    };
    const int groups = (c.H + c.Hk + kGroupHeads - 1) / kGroupHeads;
    choose(bf16, [&](auto M) {
        choose(inter, [&](auto I) {
            choose(past, [&](auto O) {
                constexpr bool kM = decltype(M)::value, kI = decltype(I)::value, kO = decltype(O)::value;
                if (c.norm && c.backward) {
                    a.blocks[0] = bwd_blocks(a.tokens, c.H, c.Hk, &a.parts[0]);
                    a.blocks[1] = c.Hk > 0 ? bwd_blocks(a.tokens, c.Hk, c.H, &a.parts[1]) : 0;
                    a.partial = static_cast<float*>(ws);
                    hipLaunchKernelGGL((head_norm_rotary_bwd_kernel<kM, kI, kO, kRows>), dim3(a.blocks[0] + a.blocks[1]), block, 0, s, a);
                } else {
                    const dim3 grid(c.T, std::min(c.B, kGridRows), (c.B + kGridRows - 1) / kGridRows), waves(64 * std::min(groups, kWaves));
                    if (c.norm) hipLaunchKernelGGL((rotary_kernel<kM, true, kI, kO, kRows>), grid, waves, 0, s, a);
                    else hipLaunchKernelGGL((rotary_kernel<kM, false, kI, kO, kRows>), grid, waves, 0, s, a);
                }
            });
        });
    });
    DT_HIP_TRY(hipGetLastError());
    if (c.norm && c.backward) {
        hipLaunchKernelGGL(head_norm_dw_kernel, dim3(DT_HEAD_DIM / kSumCols, c.Hk > 0 ? 2 : 1), block, 0, s, a.partial, a.blocks[0],
                           a.blocks[1], c.dwq, c.dwk);
        DT_HIP_TRY(hipGetLastError());
    }
    return DT_OK;
}

int launch(const Call& c, void* ws, hipStream_t s) {
    return c.starts && c.B > kFewRows ? launch_rows<kMaxRaggedBatch>(c, ws, s) : launch_rows<kFewRows>(c, ws, s);
}

int64_t workspace_bytes(const Call& c) {
    if (!c.norm || !c.backward) return 0;
    const int64_t tokens = static_cast<int64_t>(c.B) * c.T;
    int parts;
    return (bwd_blocks(tokens, c.H, c.Hk, &parts) + (c.Hk > 0 ? bwd_blocks(tokens, c.Hk, c.H, &parts) : 0)) *
           static_cast<int64_t>(DT_HEAD_DIM * sizeof(float));
}

int run(dt_ctx* ctx, const Call& call, void* ws, int64_t ws_bytes, void* stream) {
    DT_TRY(check_call(ctx, call));
    Call c = call;
    const int64_t need = workspace_bytes(c);
    if (c.mem == DT_MEM_DEVICE && need > 0 && (!ws || ws_bytes < need || !aligned16(ws)))
        return set_error(DT_ERR_INVALID_ARG, "the workspace has %lld bytes (16-byte aligned), the call needs %lld", (long long)(ws ? ws_bytes : 0), (long long)need);
    DeviceScope scope;
    DT_TRY(scope.enter(ctx->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (c.mem == DT_MEM_DEVICE) return launch(c, ws, s);

    // host memory: staged through the context's buffers, synchronous
    const size_t esz = c.dtype == DT_BF16 ? 2 : 4, tok = static_cast<size_t>(c.B) * c.T;
    const bool xs = c.norm && c.backward;
    const size_t wbytes = DT_HEAD_DIM * sizeof(float);
    DT_TRY(ctx->stage[6].ensure(4 * wbytes));
    char* wbuf = static_cast<char*>(ctx->stage[6].ptr);
    for (int i = 0; i < (c.Hk > 0 ? 2 : 1); ++i) {
        const size_t row = static_cast<size_t>(i ? c.Hk : c.H) * DT_HEAD_DIM * esz;
        const void*& in = i ? c.k : c.q;
        const void*& x = i ? c.xk : c.xq;
        int64_t &ld = i ? c.ldk : c.ldq, &ldx = i ? c.ldxk : c.ldxq;
        DT_TRY(ctx->stage[i].ensure(tok * row));
        DT_HIP_TRY(hipMemcpy2DAsync(ctx->stage[i].ptr, row, in, ld * esz, row, tok, hipMemcpyHostToDevice, s));
        if (xs) {
            DT_TRY(ctx->stage[2 + i].ensure(tok * row));
            DT_HIP_TRY(hipMemcpy2DAsync(ctx->stage[2 + i].ptr, row, x, ldx * esz, row, tok, hipMemcpyHostToDevice, s));
            x = ctx->stage[2 + i].ptr;
            ldx = row / esz;
        }
        if (c.norm) {
            const float*& w = i ? c.wk : c.wq;
            DT_HIP_TRY(hipMemcpyAsync(wbuf + i * wbytes, w, wbytes, hipMemcpyHostToDevice, s));
            w = reinterpret_cast<const float*>(wbuf + i * wbytes);
        }
        // (a row's values are read before it is written, by the same lanes)
        in = ctx->stage[i].ptr;
        ld = row / esz;
        (i ? c.ok : c.oq) = ctx->stage[i].ptr;
        (i ? c.ldok : c.ldoq) = row / esz;
    }
    c.dwq = reinterpret_cast<float*>(wbuf + 2 * wbytes);
    c.dwk = reinterpret_cast<float*>(wbuf + 3 * wbytes);
    if (c.positions) {
        DT_TRY(ctx->stage[4].ensure(tok * c.pos_bytes));
        DT_HIP_TRY(hipMemcpyAsync(ctx->stage[4].ptr, c.positions, tok * c.pos_bytes, hipMemcpyHostToDevice, s));
        c.positions = ctx->stage[4].ptr;
    }
    if (need > 0) DT_TRY(ctx->stage[5].ensure(need));
    DT_TRY(launch(c, ctx->stage[5].ptr, s));
    for (int i = 0; i < (c.Hk > 0 ? 2 : 1); ++i) {
        const size_t row = static_cast<size_t>(i ? c.Hk : c.H) * DT_HEAD_DIM * esz;
        DT_HIP_TRY(hipMemcpy2DAsync(i ? call.ok : call.oq, (i ? call.ldok : call.ldoq) * esz, ctx->stage[i].ptr, row, row, tok,
                                    hipMemcpyDeviceToHost, s));
        if (xs) DT_HIP_TRY(hipMemcpyAsync(i ? call.dwk : call.dwq, i ? c.dwk : c.dwq, wbytes, hipMemcpyDeviceToHost, s));
    }
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" {

int dt_rotary_init(dt_rotary* rot, int dims, int layout, double theta, int scaling, double factor, double original_length, double low,
                   double high, double magnitude) {
    clear_error();
    if (!rot) return set_error(DT_ERR_INVALID_ARG, "rotary is NULL");
    if (dims < 16 || dims > DT_HEAD_DIM || dims % 16)
        return set_error(DT_ERR_INVALID_ARG, "dims=%d must be a multiple of 16, at most %d", dims, DT_HEAD_DIM);
    if (layout != DT_ROTARY_HALF && layout != DT_ROTARY_INTERLEAVED) return set_error(DT_ERR_INVALID_ARG, "unknown layout %d", layout);
    if (!std::isfinite(theta) || !(theta > 1.0)) return set_error(DT_ERR_INVALID_ARG, "theta %g must be finite and above 1", theta);
    if (scaling < DT_ROTARY_UNSCALED || scaling > DT_ROTARY_RAMP) return set_error(DT_ERR_INVALID_ARG, "unknown scaling %d", scaling);
    if (scaling != DT_ROTARY_UNSCALED && (!std::isfinite(factor) || !(factor >= 1.0)))
        return set_error(DT_ERR_INVALID_ARG, "factor %g must be finite and at least 1", factor);
    if (scaling == DT_ROTARY_RAMP &&
        (!std::isfinite(original_length) || !(original_length > 0.0) || !std::isfinite(low) || !std::isfinite(high) || !(low < high)))
        return set_error(DT_ERR_INVALID_ARG, "a ramp needs an original length above 0 and low < high, got %g, %g, %g", original_length, low, high);
    if (!good_magnitude(magnitude)) return set_error(DT_ERR_INVALID_ARG, "magnitude %g must be above 0 and within fp32's range", magnitude);
    if (scaling == DT_ROTARY_THETA) theta *= std::pow(factor, static_cast<double>(dims) / (dims - 2));
    if (!std::isfinite(theta)) return set_error(DT_ERR_INVALID_ARG, "theta times the factor's power is past the range");
    *rot = {};
    rot->dims = dims;
    rot->layout = layout;
    rot->magnitude = magnitude;
    for (int i = 0; i < dims / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / dims);
        if (scaling == DT_ROTARY_LINEAR) f /= factor;
        if (scaling == DT_ROTARY_RAMP) {
            const double turns = f * original_length / 6.283185307179586476925;
            const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
            f *= keep + (1.0 - keep) / factor;
        }
        rot->frequency[i] = f;
    }
    return DT_OK;
}

int dt_rotary_fwd(dt_ctx* ctx, const void* q, const void* k, void* q_out, void* k_out, int B, int T, int H, int Hk, int D, int64_t ldq,
                  int64_t ldk, int64_t ldq_out, int64_t ldk_out, const void* positions, int pos_bytes, const int32_t* starts,
                  const dt_rotary* rotary, int backward, int dtype, int mem, void* stream) {
    clear_error();
    if (backward != 0 && backward != 1) return set_error(DT_ERR_INVALID_ARG, "backward must be 0 or 1");
    Call c{};
    c.q = q, c.k = k, c.oq = q_out, c.ok = k_out;
    c.B = B, c.T = T, c.H = H, c.Hk = Hk, c.D = D;
    c.ldq = ldq, c.ldk = ldk, c.ldoq = ldq_out, c.ldok = ldk_out;
    c.positions = positions, c.pos_bytes = pos_bytes, c.starts = starts, c.rot = rotary;
    c.dtype = dtype, c.mem = mem, c.backward = backward;
    return run(ctx, c, nullptr, 0, stream);
}

int dt_head_norm_rotary_fwd(dt_ctx* ctx, const void* q, const void* k, const float* q_weight, const float* k_weight, void* q_out,
                            void* k_out, int B, int T, int H, int Hk, int D, int64_t ldq, int64_t ldk, int64_t ldq_out,
                            int64_t ldk_out, const void* positions, int pos_bytes, const int32_t* starts, const dt_rotary* rotary,
                            float eps, int dtype, int mem, void* stream) {
    clear_error();
    Call c{};
    c.q = q, c.k = k, c.oq = q_out, c.ok = k_out, c.wq = q_weight, c.wk = k_weight;
    c.B = B, c.T = T, c.H = H, c.Hk = Hk, c.D = D;
    c.ldq = ldq, c.ldk = ldk, c.ldoq = ldq_out, c.ldok = ldk_out;
    c.positions = positions, c.pos_bytes = pos_bytes, c.starts = starts, c.rot = rotary;
    c.eps = eps, c.dtype = dtype, c.mem = mem, c.norm = true;
    return run(ctx, c, nullptr, 0, stream);
}

int dt_head_norm_rotary_bwd_workspace(int B, int T, int H, int Hk, int64_t* bytes) {
    clear_error();
    if (!bytes) return set_error(DT_ERR_INVALID_ARG, "bytes is NULL");
    if (B < 1 || T < 1 || H < 1 || Hk < 0) return set_error(DT_ERR_INVALID_ARG, "B=%d, T=%d, H=%d must be >= 1, Hk=%d >= 0", B, T, H, Hk);
    DT_TRY(check_most(B, T, H, Hk));
    Call c{};
    c.B = B, c.T = T, c.H = H, c.Hk = Hk, c.norm = c.backward = true;
    *bytes = workspace_bytes(c);
    return DT_OK;
}

int dt_head_norm_rotary_bwd(dt_ctx* ctx, const void* d_q_out, const void* d_k_out, const void* q, const void* k, const float* q_weight,
                            const float* k_weight, void* d_q, void* d_k, float* d_q_weight, float* d_k_weight, int B, int T, int H,
                            int Hk, int D, int64_t ld_dq_out, int64_t ld_dk_out, int64_t ldq, int64_t ldk, int64_t ld_dq,
                            int64_t ld_dk, const void* positions, int pos_bytes, const int32_t* starts, const dt_rotary* rotary,
                            float eps, void* ws, int64_t ws_bytes, int dtype, int mem, void* stream) {
    clear_error();
    Call c{};
    c.q = d_q_out, c.k = d_k_out, c.xq = q, c.xk = k, c.oq = d_q, c.ok = d_k;
    c.wq = q_weight, c.wk = k_weight, c.dwq = d_q_weight, c.dwk = d_k_weight;
    c.B = B, c.T = T, c.H = H, c.Hk = Hk, c.D = D;
    c.ldq = ld_dq_out, c.ldk = ld_dk_out, c.ldxq = ldq, c.ldxk = ldk, c.ldoq = ld_dq, c.ldok = ld_dk;
    c.positions = positions, c.pos_bytes = pos_bytes, c.starts = starts, c.rot = rotary;
    c.eps = eps, c.dtype = dtype, c.mem = mem, c.norm = c.backward = true;
    return run(ctx, c, ws, ws_bytes, stream);
}

}  // extern "C"
