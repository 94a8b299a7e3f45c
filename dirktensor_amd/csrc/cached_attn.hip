// Attention of the newest tokens over a key/value cache, optionally behind a prefix that the whole batch shares.
//
// For query token t of batch row b (one of cnt), head hq, the keys are those of the prefix (all of them) and those of
// the row's slot at positions < len - cnt + t + 1 (all len without causality); with s_j = scale q.k_j,
//   m = max_j s_j,  l = sum_j exp(s_j - m),  o = sum_j exp(s_j - m) v_j / l.
//
// What bounds it: a few query rows meet every held key once, so the cache's bytes (132 a key and head for K and for V
// in 8 bits) are all that counts until about a hundred query rows share a key; arithmetic is far from its bound.
//
// Work decomposition
//   * Query rows that share a key/value head's keys go together, 16 to a matrix tile: the tokens and the query heads of
//     its group for a batch row's own keys; for a shared prefix those of the whole batch, so that the prefix is read
//     once for all of them. One kernel does both, in two launches.
//   * A workgroup takes kNT tiles of 16 query rows and one chunk of the keys; chunks are as long as leaves a few
//     workgroups a CU, and at least 128 keys. Each of its four waves takes every fourth block of 32 keys and keeps its
//     own running maximum, sum and O; they meet in LDS once at the end. No wave waits for another in the loop, and no key
//     passes through LDS: the cache lies in memory in the order in which the matrix instructions read it (kv_cache.h).
//   * A chunk leaves its (m, l, unnormalised O) in the workspace, and a second kernel joins a row's chunks, the prefix's
//     and its own, in a fixed order. Where one chunk has all of a row's keys it writes the result itself.
//
// Arithmetic: S^T = K Q^T with v_mfma_f32_16x16x32_bf16 on the held values, which bf16 holds exactly (int8 and e4m3
// alike); the key's scale multiplies the 32-bit score. P times the value's scale is rounded to bf16 (half a step,
// 2^-9, for each term of the sum) for O^T += V^T P^T; m, l and O stay in 32 bits, l sums the unrounded probabilities.
// In fp32 mode q (divided by the power of two below its row's largest magnitude) and P are split into three bf16 values
// each, whose sum is the fp32 value, so every product is exact in the 32-bit accumulation.

#include "kv_cache.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace dt {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kD = DT_HEAD_DIM;
constexpr int kMinChunk = kWaves * kKvBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

struct CachedAttnArgs {
    KvView c;
    const void* q;
    void* o;
    float* m;  // nullable
    float* l;  // nullable
    float* part_o;   // [row][parts][kD]
    float* part_ml;  // [row][parts][2]
    int64_t ldq;     // token stride of q, elements
    int B, T, H, G;  // G: query heads a key/value head
    int causal;
    float scale;
    int chunk;       // keys a workgroup
    int parts;       // partial results a row at most
    int part0;       // the first of this launch's
    int direct;      // one chunk has all keys: write the result
    int prefix;      // the slot of the prefix whose keys all query rows share, or -1: each batch row its own
    int prefix_len;
    int tiles;       // workgroups over the query rows
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){lo, hi}, bf16x2));
}
__device__ __forceinline__ float bf16_round(float x) { return __uint_as_float(pack2(0.0f, x) & 0xffff0000u); }

// over the four lanes n, n + 16, n + 32, n + 48 that hold a query's keys (v_permlane swaps with x as both operands leave
// the two halves' values in the pair)
__device__ __forceinline__ float max_groups(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 8 held values (two words of 8-bit ones) as the bf16 operand of a matrix instruction
template <int kFormat>
__device__ __forceinline__ bf16x8 widen(uint32_t a, uint32_t b) {
    union { uint32_t u[4]; bf16x8 v; } r;
    if constexpr (kFormat == DT_KV_FP8) {
        r.u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
        r.u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
        r.u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
        r.u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i < 2 ? a : b;
            const int s = 16 * (i & 1);
            r.u[i] = pack2(static_cast<float>(static_cast<int8_t>(w >> s)), static_cast<float>(static_cast<int8_t>(w >> (s + 8))));
        }
    }
    return r.v;
}

// A block's K (two tiles of 16 keys) or V (eight tiles of 16 values) as loaded: 16-byte pieces of a lane
template <int kFormat>
struct Block {
    static constexpr int kPieces = kFormat == DT_KV_BF16 ? 8 : 4;
    u32x4 w[kPieces];
    // operand i of 8: K tile i / 4, step i % 4; V tile i
    __device__ __forceinline__ bf16x8 operand(int i) const {
        if constexpr (kFormat == DT_KV_BF16) return __builtin_bit_cast(bf16x8, w[i]);
        else return widen<kFormat>(w[i >> 1][(i & 1) * 2], w[i >> 1][(i & 1) * 2 + 1]);
    }
};

template <int kFormat>
__device__ __forceinline__ void load_k(Block<kFormat>& r, const uint8_t* k, int lane) {
    constexpr int kEs = kv_elem_bytes(kFormat), kPer = Block<kFormat>::kPieces / 2;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            r.w[t * kPer + i] = *reinterpret_cast<const u32x4*>(k + (t * 16 + (lane & 15)) * kD * kEs + i * 64 + (lane >> 4) * 16);
}
template <int kFormat>
__device__ __forceinline__ void load_v(Block<kFormat>& r, const uint8_t* v, int lane) {
#pragma unroll
    for (int i = 0; i < Block<kFormat>::kPieces; ++i) r.w[i] = *reinterpret_cast<const u32x4*>(v + i * 1024 + lane * 16);
}
// the first of the 8 values that a lane group's operand of step s covers, in load_k's order
template <int kFormat>
__device__ __forceinline__ int k_dim(int s, int g) {
    if constexpr (kFormat == DT_KV_BF16) return s * 32 + g * 8;
    return (s >> 1) * 64 + g * 16 + (s & 1) * 8;
}

struct QueryRow {
    int b, t, hq;
};
// row r of those that share key/value head hk's keys: tokens, then the group's heads; for the prefix the batch first
__device__ __forceinline__ QueryRow query_row(const CachedAttnArgs& a, int r, int b, int hk) {
    const int g = r % a.G, bt = r / a.G;
    if (a.prefix >= 0) return {bt / a.T, bt % a.T, hk * a.G + g};
    return {b, bt, hk * a.G + g};
}

template <int kFormat, bool kF32, int kNT>
__global__ __launch_bounds__(kThreads) void cached_attn_kernel(CachedAttnArgs a, KvRows rows) {
    constexpr int kQS = kF32 ? 3 : 1;
    __shared__ __align__(16) float obuf[2][kNT * 16][kD + 4];
    __shared__ float ml[kWaves][2][kNT * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, g = lane >> 4;

    // workgroups in launch order: eight (chunk, head, batch row) triples, one an XCD, all their query tiles before
    // the next eight, so that the tiles which read the same keys run beside each other on one XCD's L2
    int64_t id = blockIdx.x;
    const int64_t chunks_total = gridDim.x / a.tiles;
    int64_t item;
    int tile;
    {
        const int64_t full = chunks_total / 8 * 8 * a.tiles;
        if (id < full) {
            const int64_t oct = id / (8 * a.tiles);
            const int rem = static_cast<int>(id - oct * 8 * a.tiles);
            tile = rem >> 3;
            item = oct * 8 + (rem & 7);
        } else {
            id -= full;
            const int left = static_cast<int>(chunks_total % 8);
            tile = static_cast<int>(id / left);
            item = chunks_total / 8 * 8 + id % left;
        }
    }
    const int hk = static_cast<int>(item % a.c.heads);
    item /= a.c.heads;
    const int nb = a.prefix >= 0 ? 1 : a.B;
    const int b = static_cast<int>(item % nb), chunk = static_cast<int>(item / nb);

    const int len = a.prefix >= 0 ? a.prefix_len : rows.len[b];
    const int slot = a.prefix >= 0 ? a.prefix : rows.slot[b];
    const int k0 = chunk * a.chunk;
    if (k0 >= len && !(a.direct && chunk == 0)) return;  // (whole workgroups)
    const int k1 = min(len, k0 + a.chunk);
    const int nrows = (a.prefix >= 0 ? a.B : 1) * a.T * a.G;
    const int row0 = tile * kNT * 16;

    // Q fragments and each lane's query: keys below lim are seen
    int lim[kNT];
    bf16x8 qf[kNT][kQS][4];
    float qscale[kNT];
    int minlim = len;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
        const int r = row0 + nt * 16 + n;
        lim[nt] = len;
        qscale[nt] = a.scale;
        const bool have = r < nrows;
        const QueryRow qr = query_row(a, have ? r : row0, b, hk);
        const int64_t at = (static_cast<int64_t>(qr.b) * a.T + qr.t) * a.ldq + qr.hq * kD;
        if (have && a.prefix < 0 && a.causal) {
            const int cnt = rows.cnt[b];
            if (qr.t < cnt) lim[nt] = max(0, min(len, len - cnt + qr.t + 1));
        }
        minlim = min(minlim, lim[nt]);
        if constexpr (!kF32) {
            const uint16_t* q = static_cast<const uint16_t*>(a.q) + at;
#pragma unroll
            for (int s = 0; s < 4; ++s) qf[nt][0][s] = *reinterpret_cast<const bf16x8*>(q + k_dim<kFormat>(s, g));
        } else {
            const float* q = static_cast<const float*>(a.q) + at;
            float x[4][8];
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const floatx4 lo = *reinterpret_cast<const floatx4*>(q + k_dim<kFormat>(s, g));
                const floatx4 hi = *reinterpret_cast<const floatx4*>(q + k_dim<kFormat>(s, g) + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[s][j] = lo[j], x[s][4 + j] = hi[j];
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[s][j]) & 0x7f800000u);
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
            // exponents from 2^-126 to 2^126 have a reciprocal; rows beyond (and with infinities, NaN) stay as they are
            const bool norm = top >= 0x00800000u && top <= 0x7e800000u;
            const float inv = norm ? __uint_as_float(0x7f000000u - top) : 1.0f;
            qscale[nt] = norm ? a.scale * __uint_as_float(top) : a.scale;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x[s][j] * inv, h = bf16_round(v), m = bf16_round(v - h);
                    qf[nt][0][s][j] = static_cast<__bf16>(h);
                    qf[nt][1][s][j] = static_cast<__bf16>(m);
                    qf[nt][2][s][j] = static_cast<__bf16>(v - h - m);
                }
        }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) minlim = min(minlim, __shfl_xor(minlim, o, 64));

    const int64_t head = static_cast<int64_t>(slot) * a.c.heads + hk;
    constexpr int kEs = kv_elem_bytes(kFormat);
    const uint8_t* kp = a.c.k + head * a.c.keys * kD * kEs;
    const uint8_t* vp = a.c.v + head * a.c.keys * kD * kEs;
    const float* ksp = a.c.ks + head * a.c.keys;
    const float* vsp = a.c.vs + head * a.c.keys;

    floatx4 acc[kNT][8];
    float mrun[kNT], lrun[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
        mrun[nt] = kNegInf;
        lrun[nt] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[nt][i] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int kb = k0 + wave * kKvBlock; kb < k1; kb += kWaves * kKvBlock) {
        Block<kFormat> kr, vr;
        load_k<kFormat>(kr, kp + static_cast<int64_t>(kb) * kD * kEs, lane);
        floatx4 ks[2], vs[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) ks[t] = *reinterpret_cast<const floatx4*>(ksp + kb + t * 16 + g * 4);
        load_v<kFormat>(vr, vp + static_cast<int64_t>(kb) * kD * kEs, lane);
#pragma unroll
        for (int t = 0; t < 2; ++t) vs[t] = *reinterpret_cast<const floatx4*>(vsp + kb + t * 16 + g * 4);

        floatx4 s[kNT][2];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) s[nt][0] = s[nt][1] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bf16x8 kf = kr.operand(i);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int x = kQS - 1; x >= 0; --x)
                    s[nt][i >> 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[nt][x][i & 3], s[nt][i >> 2], 0, 0, 0);
        }

        const bool mask = kb + kKvBlock > minlim;  // (the same for the whole wave)
        bf16x8 pf[kNT][kQS];
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
            float mx = kNegInf;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float v = s[nt][t][i] * (ks[t][i] * qscale[nt]);
                    if (mask && kb + t * 16 + g * 4 + i >= lim[nt]) v = kNegInf;
                    s[nt][t][i] = v;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(max_groups(mx), mrun[nt]);
            const float base = mx == kNegInf ? 0.0f : mx;  // (nothing seen yet: every p is 0)
            if (__any(mx != mrun[nt])) {
                const float f = __builtin_amdgcn_exp2f((mrun[nt] - base) * kLog2e);
                lrun[nt] *= f;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[nt][i] *= f;
                mrun[nt] = mx;
            }
            float p[8], sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f((s[nt][t][i] - base) * kLog2e);
                    sum += e;
                    p[t * 4 + i] = e * vs[t][i];
                    // a masked key's scale may be anything, NaN too
                    if (mask && kb + t * 16 + g * 4 + i >= lim[nt]) p[t * 4 + i] = 0.0f;
                }
            lrun[nt] += sum;
            union { uint32_t u[4]; bf16x8 v; } f;
#pragma unroll
            for (int x = 0; x < kQS; ++x) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f.u[j] = pack2(p[2 * j], p[2 * j + 1]);
                    if (x + 1 < kQS) {
                        p[2 * j] -= __uint_as_float(f.u[j] << 16);
                        p[2 * j + 1] -= __uint_as_float(f.u[j] & 0xffff0000u);
                    }
                }
                pf[nt][x] = f.v;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bf16x8 vf = vr.operand(i);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int x = kQS - 1; x >= 0; --x)
                    acc[nt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[nt][x], acc[nt][i], 0, 0, 0);
        }
    }

    // the four waves' results: scaled to the common maximum, waves 2 and 3 onto 0 and 1, then 1 onto 0
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
        lrun[nt] = sum_groups(lrun[nt]);
        if (g == 0) {
            ml[wave][0][nt * 16 + n] = mrun[nt];
            ml[wave][1][nt * 16 + n] = lrun[nt];
        }
    }
    __syncthreads();
    float mall[kNT], lall[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
        float mx = kNegInf;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, ml[w][0][nt * 16 + n]);
        const float base = mx == kNegInf ? 0.0f : mx;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f((ml[w][0][nt * 16 + n] - base) * kLog2e);
            sum += f * ml[w][1][nt * 16 + n];
            if (w == wave) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[nt][i] *= f;
            }
        }
        mall[nt] = mx;
        lall[nt] = sum;
    }
#pragma unroll
    for (int step = 2; step >= 1; step >>= 1) {
        if (wave >= step && wave < 2 * step) {
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<floatx4*>(&obuf[wave - step][nt * 16 + n][i * 16 + g * 4]) = acc[nt][i];
        }
        __syncthreads();
        if (wave < step) {
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    acc[nt][i] += *reinterpret_cast<const floatx4*>(&obuf[wave][nt * 16 + n][i * 16 + g * 4]);
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
        const int r = row0 + nt * 16 + n;
        if (r >= nrows) continue;
        const QueryRow qr = query_row(a, r, b, hk);
        const int64_t row = (static_cast<int64_t>(qr.b) * a.T + qr.t) * a.H + qr.hq;
        if (a.direct) {
            const bool nan = lall[nt] != lall[nt];  // (a maximum passes NaN scores over: they show in the sum)
            const bool empty = qr.t >= rows.cnt[qr.b] || (mall[nt] == kNegInf && !nan);
            const float inv = empty ? 0.0f : 1.0f / lall[nt];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t at = row * kD + i * 16 + g * 4;
                floatx4 v = acc[nt][i] * inv;
                if (empty) v = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (kF32) *reinterpret_cast<floatx4*>(static_cast<float*>(a.o) + at) = v;
                else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
            }
            if (g == 0) {
                if (a.m) a.m[row] = empty ? kNegInf : nan ? lall[nt] : mall[nt];
                if (a.l) a.l[row] = empty ? 0.0f : lall[nt];
            }
        } else {
            const int64_t part = row * a.parts + a.part0 + chunk;
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<floatx4*>(a.part_o + part * kD + i * 16 + g * 4) = acc[nt][i];
            if (g == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(mall[nt], lall[nt]);
        }
    }
}

// Joins a row's partial results: one workgroup a row, 32 threads across the 128 values, eight runs of parts.
template <bool kF32>
__global__ __launch_bounds__(kThreads) void cached_attn_join_kernel(CachedAttnArgs a, KvRows rows, int prefix_parts, int own_chunk) {
    __shared__ float red[kWaves];
    __shared__ float lred[8];
    __shared__ __align__(16) float obuf[8][kD];
    const int64_t row = blockIdx.x;
    const int b = static_cast<int>(row / (static_cast<int64_t>(a.T) * a.H));
    const int t = static_cast<int>(row / a.H % a.T);
    const int len = rows.len[b];
    const int parts = t < rows.cnt[b] ? prefix_parts + (len + own_chunk - 1) / own_chunk : 0;
    const float* pml = a.part_ml + row * a.parts * 2;
    const float* po = a.part_o + row * a.parts * kD;
    float mx = kNegInf;
    for (int p = threadIdx.x; p < parts; p += kThreads) mx = fmaxf(mx, pml[2 * p]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = mx == kNegInf ? 0.0f : mx;
    const int run = threadIdx.x >> 5, d = (threadIdx.x & 31) * 4;
    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int p = run; p < parts; p += 8) {
        const float2 s = *reinterpret_cast<const float2*>(pml + 2 * p);
        const floatx4 v = *reinterpret_cast<const floatx4*>(po + static_cast<int64_t>(p) * kD + d);
        const float f = __builtin_amdgcn_exp2f((s.x - base) * kLog2e);
        l += f * s.y;
        acc += f * v;
    }
    *reinterpret_cast<floatx4*>(&obuf[run][d]) = acc;
    if ((threadIdx.x & 31) == 0) lred[run] = l;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    l = 0.0f;
    acc = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        l += lred[i];
        acc += *reinterpret_cast<const floatx4*>(&obuf[i][d]);
    }
    const bool nan = l != l;  // (a maximum passes NaN scores over: they show in the sum)
    const bool empty = mx == kNegInf && !nan;
    acc = empty ? (floatx4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / l);
    const int64_t at = row * kD + d;
    if constexpr (kF32) *reinterpret_cast<floatx4*>(static_cast<float*>(a.o) + at) = acc;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack2(acc[0], acc[1]), pack2(acc[2], acc[3]));
    if (threadIdx.x == 0) {
        if (a.m) a.m[row] = nan ? l : mx;
        if (a.l) a.l[row] = empty ? 0.0f : l;
    }
}

// How a call is cut: chunks of the batch rows' own keys and of the prefix's, partial results a row.
struct Plan {
    int own_chunk = kMinChunk, prefix_chunk = kMinChunk;
    int own_parts = 0, prefix_parts = 0;  // the longest row's
    int own_nt = 1, prefix_nt = 1;
    bool direct = false;
    int64_t ws_bytes = 0;
};

// query tiles of 16 rows that a workgroup takes
int tiles_for(int64_t rows, int dtype) {
    if (dtype != DT_BF16) return 1;
    return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

// keys a chunk: about `target` workgroups over all of `keys` (times heads and query tiles), whole blocks for every wave
int chunk_for(int64_t keys, int64_t per_key, int target) {
    const int64_t c = (keys * per_key + target - 1) / target;
    return static_cast<int>(std::min<int64_t>(std::max<int64_t>((c + kMinChunk - 1) / kMinChunk, 1) * kMinChunk, kMaxCacheTokens));
}

Plan make_plan(const dt_kv_cache* c, int B, int T, int H, const KvRows& rows, const dt_kv_cache* prefix, int prefix_len, int dtype) {
    constexpr int kTarget = 1024;  // workgroups: four a CU
    Plan p;
    const int G = H / c->heads;
    const int64_t own_rows = static_cast<int64_t>(T) * G, all_rows = own_rows * B;
    p.own_nt = tiles_for(own_rows, dtype);
    p.prefix_nt = tiles_for(all_rows, dtype);
    int64_t keys = 0;
    int longest = 0;
    for (int b = 0; b < B; ++b) {
        if (rows.cnt[b] == 0) continue;
        keys += rows.len[b];
        longest = std::max(longest, rows.len[b]);
    }
    const int64_t own_tiles = (own_rows + 16 * p.own_nt - 1) / (16 * p.own_nt);
    p.own_chunk = chunk_for(keys, own_tiles * c->heads, kTarget);
    p.own_parts = (longest + p.own_chunk - 1) / p.own_chunk;
    if (prefix && prefix_len > 0) {
        const int64_t tiles = (all_rows + 16 * p.prefix_nt - 1) / (16 * p.prefix_nt);
        p.prefix_chunk = chunk_for(prefix_len, tiles * c->heads, kTarget);
        p.prefix_parts = (prefix_len + p.prefix_chunk - 1) / p.prefix_chunk;
    }
    p.direct = p.prefix_parts == 0 && p.own_parts <= 1;
    if (!p.direct) p.ws_bytes = all_rows * c->heads * (p.own_parts + p.prefix_parts) * (kD + 2) * static_cast<int64_t>(sizeof(float));
    return p;
}

template <int kFormat, bool kF32>
int launch_tiles(CachedAttnArgs a, const KvRows& rows, int nt, int64_t items, int64_t qrows, hipStream_t s) {
    a.tiles = static_cast<int>((qrows + 16 * nt - 1) / (16 * nt));
    const int64_t grid = items * a.tiles;
    if (grid == 0) return DT_OK;
    if (grid > 0x7fffff) return set_error(DT_ERR_UNSUPPORTED, "the call needs %lld workgroups", (long long)grid);
    const dim3 g(static_cast<unsigned>(grid)), t(kThreads);
    if (nt == 1) hipLaunchKernelGGL((cached_attn_kernel<kFormat, kF32, 1>), g, t, 0, s, a, rows);
    else if constexpr (!kF32) {
        if (nt == 2) hipLaunchKernelGGL((cached_attn_kernel<kFormat, kF32, 2>), g, t, 0, s, a, rows);
        else hipLaunchKernelGGL((cached_attn_kernel<kFormat, kF32, 4>), g, t, 0, s, a, rows);
    }
    DT_HIP_TRY(hipGetLastError());
    return DT_OK;
}

int launch_part(const CachedAttnArgs& a, const KvRows& rows, int format, int dtype, int nt, int64_t items, int64_t qrows, hipStream_t s) {
    const bool f32 = dtype != DT_BF16;
    if (format == DT_KV_INT8)
        return f32 ? launch_tiles<DT_KV_INT8, true>(a, rows, nt, items, qrows, s) : launch_tiles<DT_KV_INT8, false>(a, rows, nt, items, qrows, s);
    if (format == DT_KV_FP8)
        return f32 ? launch_tiles<DT_KV_FP8, true>(a, rows, nt, items, qrows, s) : launch_tiles<DT_KV_FP8, false>(a, rows, nt, items, qrows, s);
    return f32 ? launch_tiles<DT_KV_BF16, true>(a, rows, nt, items, qrows, s) : launch_tiles<DT_KV_BF16, false>(a, rows, nt, items, qrows, s);
}

int run(const dt_kv_cache* c, CachedAttnArgs a, const KvRows& rows, const dt_kv_cache* prefix, int prefix_slot, int prefix_len,
        const Plan& p, void* ws, int dtype, hipStream_t s) {
    const int64_t own_rows = static_cast<int64_t>(a.T) * a.G, all_rows = own_rows * a.B;
    a.parts = p.own_parts + p.prefix_parts;
    a.part_o = static_cast<float*>(ws);
    a.part_ml = ws ? a.part_o + all_rows * c->heads * a.parts * kD : nullptr;
    a.direct = p.direct;
    if (p.prefix_parts > 0) {
        CachedAttnArgs f = a;
        f.c = prefix->view();
        f.prefix = prefix_slot;
        f.prefix_len = prefix_len;
        f.chunk = p.prefix_chunk;
        f.part0 = 0;
        DT_TRY(launch_part(f, rows, c->format, dtype, p.prefix_nt, static_cast<int64_t>(p.prefix_parts) * c->heads, all_rows, s));
    }
    a.c = c->view();
    a.prefix = -1;
    a.prefix_len = 0;
    a.chunk = p.own_chunk;
    a.part0 = p.prefix_parts;
    // (a call with nothing to see still writes its empty rows)
    const int64_t items = static_cast<int64_t>(p.direct ? 1 : p.own_parts) * a.B * c->heads;
    DT_TRY(launch_part(a, rows, c->format, dtype, p.own_nt, items, own_rows, s));
    if (p.direct) return DT_OK;
    const dim3 g(static_cast<unsigned>(all_rows * c->heads)), t(kThreads);
    if (dtype == DT_BF16) hipLaunchKernelGGL((cached_attn_join_kernel<false>), g, t, 0, s, a, rows, p.prefix_parts, p.own_chunk);
    else hipLaunchKernelGGL((cached_attn_join_kernel<true>), g, t, 0, s, a, rows, p.prefix_parts, p.own_chunk);
    DT_HIP_TRY(hipGetLastError());
    return DT_OK;
}

// what dt_cached_attn_fwd and its workspace query check alike; fills rows
int check_call(const dt_kv_cache* cache, int B, int T, int H, int D, const int32_t* slots, const int32_t* counts,
               const dt_kv_cache* prefix, int prefix_slot, int dtype, KvRows* rows) {
    if (D != DT_HEAD_DIM) return set_error(DT_ERR_UNSUPPORTED, "head_dim D=%d, kernels are built for D=%d", D, DT_HEAD_DIM);
    if (B < 1 || T < 1 || H < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d, T=%d, H=%d must be >= 1", B, T, H);
    if (B > kMaxRaggedBatch) return set_error(DT_ERR_UNSUPPORTED, "B=%d > %d", B, kMaxRaggedBatch);
    if (T > DT_MAX_SEQ_LEN) return set_error(DT_ERR_INVALID_ARG, "T=%d exceeds max_seq_len %d", T, DT_MAX_SEQ_LEN);
    if (dtype != DT_FP32_EXACT && dtype != DT_BF16) return set_error(DT_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (!cache) return set_error(DT_ERR_INVALID_ARG, "cache is NULL");
    if (H % cache->heads || H > kMaxCacheHeads)
        return set_error(DT_ERR_INVALID_ARG, "H=%d is no multiple of the cache's %d heads, or above %d", H, cache->heads, kMaxCacheHeads);
    // (row and workgroup indices within a launch stay within 31 bits)
    if (static_cast<int64_t>(B) * T * H > 0x7fffff) return set_error(DT_ERR_UNSUPPORTED, "B*T*H = %lld query rows", (long long)B * T * H);
    DT_TRY(kv_check_slots(cache, B, slots, false, rows));
    DT_TRY(kv_check_counts(B, T, counts, rows));
    for (int b = 0; b < B; ++b) rows->len[b] = cache->len[rows->slot[b]];
    if (prefix) {
        if (prefix->heads != cache->heads || prefix->format != cache->format || prefix->ctx != cache->ctx)
            return set_error(DT_ERR_INVALID_ARG, "the prefix's cache has another context, format or number of heads");
        if (prefix_slot < 0 || prefix_slot >= prefix->slots)
            return set_error(DT_ERR_INVALID_ARG, "prefix_slot=%d outside [0, %d)", prefix_slot, prefix->slots);
    }
    return DT_OK;
}

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" {

int dt_cached_attn_workspace(const dt_kv_cache* cache, int B, int T, int H, int D, const int32_t* slots, const int32_t* counts,
                             const dt_kv_cache* prefix, int prefix_slot, int dtype, int64_t* bytes) {
    clear_error();
    if (!bytes) return set_error(DT_ERR_INVALID_ARG, "bytes is NULL");
    KvRows rows;
    DT_TRY(check_call(cache, B, T, H, D, slots, counts, prefix, prefix_slot, dtype, &rows));
    *bytes = make_plan(cache, B, T, H, rows, prefix, prefix ? prefix->len[prefix_slot] : 0, dtype).ws_bytes;
    return DT_OK;
}

int dt_cached_attn_fwd(dt_kv_cache* cache, const void* q, void* o, float* m, float* l, int B, int T, int H, int D, int64_t ldq,
                       float scale, int causal, const int32_t* slots, const int32_t* counts, const dt_kv_cache* prefix,
                       int prefix_slot, void* ws, int64_t ws_bytes, int dtype, int mem, void* stream) {
    clear_error();
    if (!q || !o) return set_error(DT_ERR_INVALID_ARG, "q and o must be non-NULL");
    if (mem != DT_MEM_DEVICE && mem != DT_MEM_HOST) return set_error(DT_ERR_INVALID_ARG, "unknown mem %d", mem);
    if (!(scale > 0.0f) || !std::isfinite(scale)) return set_error(DT_ERR_INVALID_ARG, "scale %g must be finite and > 0", scale);
    if (causal != 0 && causal != 1) return set_error(DT_ERR_INVALID_ARG, "causal must be 0 or 1");
    KvRows rows;
    DT_TRY(check_call(cache, B, T, H, D, slots, counts, prefix, prefix_slot, dtype, &rows));
    const size_t esz = dtype == DT_BF16 ? 2 : 4;
    const int64_t dm = static_cast<int64_t>(H) * kD;
    if (ldq < dm) return set_error(DT_ERR_INVALID_ARG, "row stride %lld is below %lld", (long long)ldq, (long long)dm);
    if (mem == DT_MEM_DEVICE && (!aligned16(q) || !aligned16(o) || !aligned16(ws) || ldq * esz % 16))
        return set_error(DT_ERR_INVALID_ARG, "device q/o/workspace and q's row stride must be 16-byte aligned");
    const int prefix_len = prefix ? prefix->len[prefix_slot] : 0;
    const Plan p = make_plan(cache, B, T, H, rows, prefix, prefix_len, dtype);
    if (mem == DT_MEM_DEVICE && p.ws_bytes > 0 && (!ws || ws_bytes < p.ws_bytes))
        return set_error(DT_ERR_INVALID_ARG, "the workspace has %lld bytes, the call needs %lld", (long long)(ws ? ws_bytes : 0), (long long)p.ws_bytes);
    dt_ctx* ctx = cache->ctx;
    DT_TRY(check_device_binding(ctx));
    hipStream_t s = static_cast<hipStream_t>(stream);
    CachedAttnArgs a{};
    a.q = q;
    a.o = o;
    a.m = m;
    a.l = l;
    a.ldq = ldq;
    a.B = B;
    a.T = T;
    a.H = H;
    a.G = H / cache->heads;
    a.causal = causal;
    a.scale = scale;
    if (mem == DT_MEM_DEVICE) return run(cache, a, rows, prefix, prefix_slot, prefix_len, p, ws, dtype, s);

    // host memory: staged through the context's buffers, synchronous
    const size_t tok = static_cast<size_t>(B) * T, row = dm * esz, nst = tok * H * sizeof(float);
    DT_TRY(ctx->stage[0].ensure(tok * row));
    DT_TRY(ctx->stage[1].ensure(tok * row));
    DT_TRY(ctx->stage[2].ensure(nst));
    DT_TRY(ctx->stage[3].ensure(nst));
    if (p.ws_bytes > 0) DT_TRY(ctx->stage[4].ensure(p.ws_bytes));
    DT_HIP_TRY(hipMemcpy2DAsync(ctx->stage[0].ptr, row, q, ldq * esz, row, tok, hipMemcpyHostToDevice, s));
    a.q = ctx->stage[0].ptr;
    a.o = ctx->stage[1].ptr;
    a.m = static_cast<float*>(ctx->stage[2].ptr);
    a.l = static_cast<float*>(ctx->stage[3].ptr);
    a.ldq = dm;
    DT_TRY(run(cache, a, rows, prefix, prefix_slot, prefix_len, p, ctx->stage[4].ptr, dtype, s));
    DT_HIP_TRY(hipMemcpyAsync(o, a.o, tok * row, hipMemcpyDeviceToHost, s));
    if (m) DT_HIP_TRY(hipMemcpyAsync(m, a.m, nst, hipMemcpyDeviceToHost, s));
    if (l) DT_HIP_TRY(hipMemcpyAsync(l, a.l, nst, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

}  // extern "C"
