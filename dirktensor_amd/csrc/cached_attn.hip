// Attention of the newest tokens over a key/value cache, optionally behind a prefix that the whole batch shares.
//
// For query token t of batch row b (one of cnt), head hq, the keys are those of the prefix (all of them) and those of
// the row's slot at positions < len - cnt + t + 1 (all len without causality); with s_j = scale q.k_j,
//   m = max_j s_j,  l = sum_j exp(s_j - m),  o = sum_j exp(s_j - m) v_j / l.
//
// What bounds it: a few query rows meet every held key once, so the cache's bytes (132 a key and head for K and for V
// in 8 bits, 68 in 4) are all that counts until about a hundred query rows share a key; arithmetic is far from its bound.
//
// Work decomposition
//   * Query rows that share a key/value head's keys go together, 16 to a matrix tile: the tokens and the query heads of
//     its group for a batch row's own keys; for a shared prefix those of the whole batch, so that the prefix is read
//     once for all of them. Where there are more than 16, a wave takes two tiles and widens each held value once for
//     both (64 queries over a prefix in int8: 377 and 530 TFLOP/s; 256: 324 and 761, in fp8 390 and 1023; whole calls at 16 heads over
//     131072 keys reach 452 and 613 in int8, 549 and 768 in fp8).
//   * A workgroup has four waves: as many of them as there are tiles (one or two, up to four in exact mode) take query rows
//     and the rest is spread over the keys, 32 at a time. Every wave keeps its own running maximum, sum and O; those of one
//     tile meet in LDS once at the end. No wave waits for another in the loop, and no key passes through LDS: the cache lies
//     in memory in the order in which the matrix instructions read it (kv_cache.h).
//   * The keys of all (head, batch row, query tile) triples form one list, cut into as many equal shares as workgroups fit the
//     CUs (two each), so ragged lengths leave no CU idle; a share may end within a triple and go on in the next. Short
//     lists are not cut within a triple: a workgroup, or where there are many a wave, then has all keys of one, and no
//     second kernel is needed. The prefix's keys are cut into chunks for workgroups of the same launch.
//   * A workgroup that has all of a triple's keys writes the result itself; otherwise it leaves (m, l, unnormalised O) in the
//     workspace, and a second kernel joins a row's parts, the prefix's and its own, in a fixed order.
//
// Measured at 16 heads, us: one sequence of 1000 in bf16 9.8 (latency: 16 workgroups); 16 sequences of up to 4096 in int8, 167 MB,
// 28 and 4.4 for the join (6.0 TB/s); 32 of 8192 in fp8, 1.1 GB, 161 without a join (6.9 TB/s, what a read of this size reaches); 64 of
// up to 512 behind a prefix of 4096 in int8 27 and 4.4 (94 MB, and the prefix's widening and products beside it); 12 by 5 tokens
// behind 2777 in fp8 13 and 4; 4 of 1500 in exact mode, int8, 12 and 4. In 4 bits: 32 of 8192, 571 MB, 92 without a join (6.2 TB/s; about
// 223 vector instructions a block, 64 % of what the CUs can issue); 12 by 5 tokens of 16 heads on 4 key/value heads, up to 1500 each behind 2777,
// 18 and 5.7 (in exact mode 138 and 23 and 5.5); 64 and 256 tokens behind 131008 keys 545 and 631 TFLOP/s.
//
// Arithmetic: S^T = K Q^T with v_mfma_f32_16x16x32_bf16 on the held values, which bf16 holds exactly (int8 and e4m3
// alike); the key's scale multiplies the 32-bit score. P times the value's scale is rounded to bf16 (at most half a step,
// 2^-8 relative, for each term of the sum) for O^T += V^T P^T; m, l and O stay in 32 bits, l sums the unrounded probabilities.
// In fp32 mode q (divided by 2^9 times the power of two below its row's largest magnitude) and P are split into three bf16 values
// each, whose sum is the fp32 value, so every product is exact in the 32-bit accumulation.
// In 4 bits a row has four scales, so they go into the operands: the conversion to bf16 multiplies by a power of two, exactly, and
// no score or probability is multiplied. In exact mode the parts of q and P meet the same operands.

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

constexpr int kWaves = 4;       // of a workgroup
constexpr int kJoinThreads = 256;
constexpr int kWavesLog = 2;
constexpr int kStepLog = 5 + kWavesLog;  // log2 of the keys of a step: a block a wave
static_assert(1 << kWavesLog == kWaves && 1 << kStepLog == kKvBlock * kWaves, "logarithms");
constexpr int kD = DT_HEAD_DIM;
constexpr int kObufRow = kD + 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLowest = -3.402823466e38f;
constexpr float kSlack = 8.0f;
// O before its division by l exceeds the values by up to 2^kSlack times the number of keys, and so fp32's range where the values lie
// near its end. A wave whose O reaches kLimit (or has left the range) does its stretch once more with V's scales times kLower: O is
// then at most 2^8 (a probability) 2^128 (a value) 2^21 (keys) 2^-32 = 2^125, and such results meet others, times kLower too. What
// that loses are values below 2^-70, in a wave that has others above 2^70. (The check and the way back cost 0.3 us of the 11 of one
// sequence of 1000 in bf16, 0.4 of the 14 of 4 of 1500 in exact mode and 2 of the 86 of 700 tokens behind 2000 in fp8; 32 of 8192 in fp8
// take no longer.)
constexpr float kLimit = 0x1p100f;
constexpr float kLower = 0x1p-32f, kRaise = 0x1p32f;
constexpr int kBufferDword3 = 0x00020000;  // raw buffer, 32-bit data format (gfx9 family)

// blocks in flight a wave: what 256 registers a lane hold, which leave two workgroups a CU. Two of 8 bits with one query tile take 212;
// two of bf16, in exact mode or with two tiles would spill 8, 19 and 79. Two of 4 bits take 104; three and four of them gain nothing (32 of
// 8192 94 and 99 us, profiled, where two take 92 to 98).
constexpr int stages(int format, bool f32, int qt) { return format == DT_KV_BF16 || f32 || qt > 1 ? 1 : 2; }

// The batch rows, by value in the kernel's arguments (kN places, 32 where these are enough: eager calls at 16 heads in int8, one
// sequence of 1000 10.8 us with 256 and 10.4 with 32, 8 of 200 behind 2000 14.6 and 13.7).
template <int kN>
struct AttnRowsOf {
    int32_t len[kN];       // tokens held
    int32_t cum[kN];       // places of one head in the list before this row's, all query tiles
    uint16_t slot[kN];
    uint16_t cnt[kN];      // query tokens
};
using AttnRows = AttnRowsOf<kMaxRaggedBatch>;

struct CachedAttnArgs {
    KvView own, pre;
    const void* q;
    void* o;
    float* m;  // nullable
    float* l;  // nullable
    float* part_o;   // [row][parts][kD]
    float* part_ml;  // [row][parts][2]: the maximum; l, negative where O is times kLower
    int64_t ldq;     // token stride of q, elements
    int B, T, H, G;  // G: query heads a key/value head
    uint64_t by_G, by_T;  // 2^40 / G and / T, rounded up (divided)
    int causal;
    float scale;
    int parts;       // partial results a row at most
    // own keys, in steps of 32 keys a key wave; own_wl: log2 of the waves that take query tiles
    int own_wl, own_qt, own_tiles;  // own_qt: query tiles of such a wave; own_tiles: workgroups for a batch row's query rows
    int own_groups;     // workgroups
    int aligned;        // one (head, batch row, tile) a workgroup; otherwise shares of the list
    int apart;          // one a wave
    int lead;           // places that a triple has in the list before those of its steps, for what beginning it costs
    int head_places;    // of one head: all batch rows and tiles
    int share, extra;
    // prefix
    int pre_slot, pre_len, pre_wl, pre_qt, pre_tiles, pre_chunk;  // pre_chunk: keys a workgroup
    int pre_parts, pre_groups;
};

// steps of a batch row's keys for a query tile (0: there is nothing to see)
__host__ __device__ __forceinline__ int steps_of(int len, int cnt, int wl) {
    const int log = kStepLog - wl;
    return cnt == 0 ? 0 : (len + (1 << log) - 1) >> log;
}
// The list's places in equal shares: the first `extra` workgroups have one more than `share`. group_of: whose share place s is in.
__host__ __device__ __forceinline__ int share_start(const CachedAttnArgs& a, int w) {
    return w * a.share + (w < a.extra ? w : a.extra);
}
__host__ __device__ __forceinline__ int group_of(const CachedAttnArgs& a, int s) {
    const int longer = a.extra * (a.share + 1);
    return s < longer ? s / (a.share + 1) : a.extra + (s - longer) / a.share;
}

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

// keeps the compiler from widening a whole block at once, which would take 64 registers more than there are for two
// workgroups a CU
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

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

// 8 held values of 4 bits times their scale, a power of two (an infinity, which no scale is, gives NaN)
__device__ __forceinline__ bf16x8 widen4(uint32_t w, float scale) {
    union { uint32_t u[4]; bf16x8 v; } r;
    r.u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r.u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r.u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r.u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return r.v;
}

// A block as loaded: 16-byte pieces of K (two tiles of 16 keys) and V (eight tiles of 16 values), and the scales of the lane's
// keys. kOnce: no other wave reads these keys, so they pass the caches by.
template <int kFormat, bool kOnce>
struct Block {
    static constexpr int kPieces = kv_elem_bits(kFormat) / 2;
    u32x4 k[kPieces], v[kPieces];
    floatx4 ks[2], vs[2];
    // fp4: of K the scale of the lane's key and group of values, as a float's exponent; of V the four scales of each of the lane's keys
    uint32_t k4[2];
    u32x4 v4[2];
    // 16 bytes at `at` + the lane's offset of the block that begins at `from` (the immediate offset holds 12 bits)
    template <bool kNt>
    static __device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t off, int from, int at) {
        return __builtin_amdgcn_raw_buffer_load_b128(r, off + (at & 4095), from + (at & ~4095), kNt ? 2 : 0);
    }
    __device__ __forceinline__ void load_k(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t scale_off, int from) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) k[i] = load16<kOnce>(r, off, from, i * kKvRun);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (kFormat == DT_KV_FP4)
                k4[t] = __builtin_amdgcn_raw_buffer_load_b8(r, scale_off + t * 64, from + kv_scale_at(kFormat), 0);
            else
                ks[t] = __builtin_bit_cast(floatx4, load16<false>(r, scale_off, from, kv_scale_at(kFormat) + t * 64));
        }
    }
    __device__ __forceinline__ void load_v(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t scale_off, int from) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) v[i] = load16<kOnce>(r, off, from, kv_tensor_bytes(kFormat) + i * kKvRun);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const u32x4 w = load16<false>(r, scale_off, from, kv_scale_at(kFormat) + 128 + t * 64);
            if constexpr (kFormat == DT_KV_FP4) v4[t] = w;
            else vs[t] = __builtin_bit_cast(floatx4, w);
        }
    }
    // the pieces as values of their own: else the compiler carries them through the loop widened, in twice or four times the
    // registers
    static __device__ __forceinline__ void settle(u32x4 (&w)[kPieces]) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) asm volatile("" : "+v"(w[i]));
    }
    // operand i of 8: K tile i / 4, step i % 4; V tile i. fp4: K times its scale
    __device__ __forceinline__ bf16x8 operand_k(int i) {
        if constexpr (kFormat == DT_KV_FP4) return widen4(k[i >> 2][i & 3], __uint_as_float(k4[i >> 2] << 23));
        else return operand(k, i);
    }
    // fp4: V tiles 2 i and 2 i + 1 times their scales
    __device__ __forceinline__ void operands_v(int i, bf16x8 (&to)[2]) {
        union { uint32_t u[4]; bf16x8 v; } r[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (keys 2 j and 2 j + 1 of the lane's)
            const uint32_t w = v[i >> 1][(i & 1) * 2 + (j >> 1)];
            const float s0 = scale4(v4[j >> 1][2 * j & 3], i), s1 = scale4(v4[j >> 1][(2 * j + 1) & 3], i);
            const auto pair = [&](float s, auto at) {
                return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, decltype(at)::value));
            };
            const uint32_t a = j & 1 ? pair(s0, std::integral_constant<int, 2>()) : pair(s0, std::integral_constant<int, 0>());
            const uint32_t b = j & 1 ? pair(s1, std::integral_constant<int, 3>()) : pair(s1, std::integral_constant<int, 1>());
            r[0].u[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
            r[1].u[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        }
        to[0] = r[0].v;
        to[1] = r[1].v;
    }
    // byte i of a key's scales as an exponent: the conversion's scale operand is a 32-bit number of which it takes the exponent field alone, so
    // the neighbouring bytes that lie in its sign and fraction change nothing (nor did they in 2^20 random words)
    static __device__ __forceinline__ float scale4(uint32_t w, int i) { return __uint_as_float(i < 3 ? w << (23 - 8 * i) : w >> 1); }
    static __device__ __forceinline__ bf16x8 operand(const u32x4 (&w)[kPieces], int i) {
        if constexpr (kFormat == DT_KV_BF16) return __builtin_bit_cast(bf16x8, w[i]);
        else return widen<kFormat>(w[i >> 1][(i & 1) * 2], w[i >> 1][(i & 1) * 2 + 1]);
    }
};

// the first of the 8 values that a lane group's operand of step s covers, in k_offset's order
template <int kFormat>
__device__ __forceinline__ int k_dim(int s, int g) {
    if constexpr (kFormat == DT_KV_BF16) return s * 32 + g * 8;
    if constexpr (kFormat == DT_KV_FP4) return g * 32 + s * 8;
    return (s >> 1) * 64 + g * 16 + (s & 1) * 8;
}

__device__ __forceinline__ int divided(int r, uint64_t by) { return static_cast<int>(static_cast<uint32_t>(r) * by >> 40); }

struct QueryRow {
    int b, t, hq;
};
// row r of those that share key/value head hk's keys: tokens, then the group's heads; for the prefix the batch first
__device__ __forceinline__ QueryRow query_row(const CachedAttnArgs& a, int r, int b, int hk, bool prefix) {
    // (divisions by numbers that are mostly 1; r < 2^23, G <= 2^10 and T <= 2^13, so r times what the reciprocal is too large by, less
    // than G or T, stays below 2^40)
    const int bt = a.G == 1 ? r : divided(r, a.by_G), g = r - bt * a.G;
    if (!prefix) return {b, bt, hk * a.G + g};
    const int of = a.T == 1 ? bt : divided(bt, a.by_T);
    return {of, bt - of * a.T, hk * a.G + g};
}

// One workgroup's stretch of keys for one (head, batch row, tile), or of the prefix for one (head, tile).
struct Work {
    int hk, b, tile;
    int k0, k1;      // keys
    int slot, len, cnt;  // cnt: the batch row's query tokens
    int wl;          // log2 of the waves that take query tiles
    int apart;       // whether each wave has a stretch of its own
    int part;        // where the partial result goes, or -1: the result is written
    bool prefix;
};

// The thread's index as a value of its own: what is derived from it is then not worked out ahead of the loops around and held in
// registers through them.
__device__ __forceinline__ int thread_here() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

template <int kQT>
struct Shared {
    float o[kWaves * kQT][16][kObufRow];
    float ml[kWaves * kQT][3][16];  // base, sum, true maximum
    int lowered[kWaves];            // whether the wave's O is times kLower
};

// A wave's part of a stretch of work: begin puts the loads of its first blocks and of its Q rows under way, attend does the work
// and leaves the results in LDS, join (of the whole workgroup) puts the waves' results together. kQT: query tiles a wave.
template <int kFormat, bool kF32, bool kOnce, int kQT>
struct Stretch {
    static constexpr int kQS = kF32 ? 3 : 1, kStages = stages(kFormat, kF32, kQT);
    static constexpr bool kFp4 = kFormat == DT_KV_FP4;
    Block<kFormat, kOnce> st[kStages];
    static constexpr int kQRegs = kF32 ? 8 : 4;
    u32x4 qraw[kQT][kQRegs];
    __amdgpu_buffer_rsrc_t rsrc;  // the (slot, head)'s blocks
    int k0, kb, k1, step;         // the first block's first key, the next one's, the end, the distance of the wave's blocks
    int at, at_step;              // the byte offset of the next block to load, the distance
    int lane, wave, lim[kQT], minlim;

    // Loads the wave's next block into st[i], K or V. Past its last block nothing is read: the lanes' offset is then beyond the
    // buffer and zeros arrive. (No load is under a condition: the compiler would count it as not issued, and every wait
    // for a block would be one for all loads.)
    __device__ __forceinline__ void load_k(Block<kFormat, kOnce>& b, int key) {
        const uint32_t beyond = key < k1 ? 0u : 0x80000000u;
        // (fp4: the byte of the lane's key and group of values)
        b.load_k(rsrc, lane * 16 + beyond, (kFormat == DT_KV_FP4 ? (lane & 15) * 4 + (lane >> 4) : (lane >> 4) * 16) + beyond, at);
    }
    __device__ __forceinline__ void load_v(Block<kFormat, kOnce>& b, int key) {
        const uint32_t beyond = key < k1 ? 0u : 0x80000000u;
        b.load_v(rsrc, lane * 16 + beyond, (lane >> 4) * 16 + beyond, at);
        at += at_step;
    }

    __device__ __forceinline__ void load_first() {
        kb = k0;
        at = kb / kKvBlock * kv_block_bytes(kFormat);
#pragma unroll
        for (int i = 0; i < kStages; ++i) {
            load_k(st[i], kb + i * step);
            load_v(st[i], kb + i * step);
        }
    }

    __device__ __forceinline__ void begin(const CachedAttnArgs& a, const Work& w) {
        const int tid = thread_here();
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int n = lane & 15, g = lane >> 4;
        const int qw = wave & ((1 << w.wl) - 1), kw = wave >> w.wl;
        step = (1 << kStepLog) >> w.wl;
        k1 = w.k1;
        const KvView& c = w.prefix ? a.pre : a.own;
        rsrc = __builtin_amdgcn_make_buffer_rsrc(c.block<kFormat>(w.slot, w.hk, 0), 0, c.blocks * kv_block_bytes(kFormat), kBufferDword3);
        k0 = w.k0 + kw * kKvBlock;
        at_step = step / kKvBlock * kv_block_bytes(kFormat);
        load_first();
        const int nrows = (w.prefix ? a.B : 1) * a.T * a.G;
        const int row0 = w.apart ? w.tile * (16 * kQT) : w.tile * (16 * kQT) << w.wl;
        minlim = w.len;
#pragma unroll
        for (int x = 0; x < kQT; ++x) {
            const int r = row0 + ((w.apart ? 0 : qw * kQT) + x) * 16 + n;
            const bool have = r < nrows;
            const QueryRow qr = query_row(a, have ? r : row0, w.b, w.hk, w.prefix);
            const int64_t qat = (static_cast<int64_t>(qr.b) * a.T + qr.t) * a.ldq + qr.hq * kD;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if constexpr (kF32) {
                    const u32x4* q = reinterpret_cast<const u32x4*>(static_cast<const float*>(a.q) + qat + k_dim<kFormat>(s, g));
                    qraw[x][2 * s] = q[0];
                    qraw[x][2 * s + 1] = q[1];
                } else {
                    qraw[x][s] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + qat + k_dim<kFormat>(s, g));
                }
            }
            // keys below lim are seen by the lane's query, keys below minlim by all of the wave's
            lim[x] = w.len;
            if (have && !w.prefix && a.causal && qr.t < w.cnt) lim[x] = max(0, min(w.len, w.len - w.cnt + qr.t + 1));
            minlim = min(minlim, lim[x]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) minlim = min(minlim, __shfl_xor(minlim, o, 64));
    }

    // Q as the matrix operand: as it is, or in three parts; returns what the scores are multiplied with
    static __device__ __forceinline__ float operand_q(u32x4 (&qraw)[kQRegs], float scale, bf16x8 (&qf)[kQS][4]) {
#pragma unroll
        for (int i = 0; i < kQRegs; ++i) asm volatile("" : "+v"(qraw[i]));  // (arrived: no wait for them in the loop)
        if constexpr (!kF32) {
#pragma unroll
            for (int s = 0; s < 4; ++s) qf[0][s] = __builtin_bit_cast(bf16x8, qraw[s]);
            return scale;
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < 8; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j) top = max(top, qraw[s][j] & 0x7f800000u);
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, 64)));
            top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, 64)));
            // exponents from 2^-126 to 2^126 have a reciprocal; rows beyond (and with infinities, NaN) stay as they are. Divided by 2^9
            // times their power of two the values are below 2^-8, and 128 products with keys of any size stay in range.
            const bool norm = top >= 0x00800000u && top <= 0x7e800000u;
            const uint32_t by = min(top + (9u << 23), 0x7e800000u);
            const float inv = norm ? __uint_as_float(0x7f000000u - by) : 1.0f;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = __uint_as_float(qraw[2 * s + (j >> 2)][j & 3]) * inv, h = bf16_round(v), m = bf16_round(v - h);
                    qf[0][s][j] = static_cast<__bf16>(h);
                    qf[1][s][j] = static_cast<__bf16>(m);
                    qf[2][s][j] = static_cast<__bf16>(v - h - m);
                }
            return norm ? scale * __uint_as_float(by) : scale;
        }
    }

    // probabilities times V's scales as the matrix operand: rounded to bf16, or in three parts
    static __device__ __forceinline__ void operand_p(float (&p)[8], bf16x8 (&pf)[kQS]) {
#pragma unroll
        for (int y = 0; y < kQS; ++y) {
            union { uint32_t u[4]; bf16x8 v; } h;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h.u[j] = pack2(p[2 * j], p[2 * j + 1]);
                if (y + 1 < kQS) {
                    p[2 * j] -= __uint_as_float(h.u[j] << 16);
                    p[2 * j + 1] -= __uint_as_float(h.u[j] & 0xffff0000u);
                }
            }
            pf[y] = h.v;
        }
    }

    __device__ __forceinline__ void attend(float scale, Shared<kQT>& sh) {
        const int n = lane & 15, g = lane >> 4;
        bf16x8 qf[kQT][kQS][4];
        float qscale[kQT];
#pragma unroll
        for (int x = 0; x < kQT; ++x) qscale[x] = operand_q(qraw[x], scale * kLog2e, qf[x]);  // (scores in the log2 domain)

        // p = exp2(score - base): base is at least the true maximum less kSlack, and moves to it only where a score exceeds it by
        // more, so O is seldom rescaled. Each lane keeps the true maximum and the sum of its own keys.
        floatx4 acc[kQT][8];
        float base[kQT], top[kQT], sum[kQT];
        bool lowered = false;  // (the same for the whole wave)

        // one block: scores, probabilities, O; its registers are filled again, K's behind the scores and V's behind O, with the
        // block kStages steps on
        auto take = [&](Block<kFormat, kOnce>& blk) {
            const int next = kb + kStages * step;
            blk.settle(blk.k);
            floatx4 s[kQT][2];
#pragma unroll
            for (int x = 0; x < kQT; ++x) s[x][0] = s[x][1] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bf16x8 kf = blk.operand_k(i);
#pragma unroll
                for (int x = 0; x < kQT; ++x)
#pragma unroll
                    for (int y = kQS - 1; y >= 0; --y)
                        s[x][i >> 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[x][y][i & 3], s[x][i >> 2], 0, 0, 0);
                keep_order();
            }
            floatx4 f[kQT][2];
#pragma unroll
            for (int x = 0; x < kQT; ++x)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if constexpr (kFormat == DT_KV_FP4) f[x][t] = (floatx4){qscale[x], qscale[x], qscale[x], qscale[x]};
                    else f[x][t] = blk.ks[t] * qscale[x];
                }
            keep_order();
            load_k(blk, next);
            keep_order();
            const bool mask = kb + kKvBlock > minlim;  // (the same for the whole wave)
            bf16x8 pf[kQT][kQS];
            uint32_t none = 0;  // fp4: whether some key of the lane's has a row of V that is none
            if constexpr (kFp4) {
#pragma unroll
                for (int i = 0; i < 8; ++i) none = max(none, blk.v4[i >> 2][i & 3]);
                asm volatile("" : "+v"(none));  // (four instructions; else it becomes a comparison a key)
            } else {
                if (__builtin_expect(lowered, 0)) blk.vs[0] *= kLower, blk.vs[1] *= kLower;
            }
#pragma unroll
            for (int x = 0; x < kQT; ++x) {
                const int rest = lim[x] - kb - g * 4;  // the lane's key 16 t + i is seen if it is below
                float p[8], most = kNegInf;  // (the maximum of the scores themselves: it does not depend on how the keys are cut)
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = s[x][i >> 2][i & 3] * f[x][i >> 2][i & 3];
                if (mask) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if ((i >> 2) * 16 + (i & 3) >= rest) p[i] = kNegInf;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, p[i]);
                top[x] = fmaxf(top[x], most);
                if (__any(most - base[x] > kSlack)) {
                    const float to = max_groups(fmaxf(most, base[x]));
                    const float by = __builtin_amdgcn_exp2f(base[x] - to);
                    sum[x] *= by;
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[x][i] *= by;
                    base[x] = to;
                }
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = __builtin_amdgcn_exp2f(p[i] - base[x]);
                    add += e;
                    if constexpr (kFp4) p[i] = e;  // (V's scales go with V)
                    else p[i] = e * blk.vs[i >> 2][i & 3];
                }
                sum[x] += add;
                if constexpr (kFp4) {
                    if (__builtin_expect(lowered, 0))
#pragma unroll
                        for (int i = 0; i < 8; ++i) p[i] *= kLower;
                    // such a row's values are 0, and the queries that see it get their NaN here
                    if (__builtin_expect(__any(none == 0xffffffffu), 0))
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (blk.v4[i >> 2][i & 3] == 0xffffffffu) p[i] = __uint_as_float(0x7fc00000u);
                }
                if (mask) {  // (a masked key's scale may be anything, NaN too)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if ((i >> 2) * 16 + (i & 3) >= rest) p[i] = 0.0f;
                }
                operand_p(p, pf[x]);
            }
            blk.settle(blk.v);
            const auto add_v = [&](int i, const bf16x8& vf) {
#pragma unroll
                for (int x = 0; x < kQT; ++x)
#pragma unroll
                    for (int y = kQS - 1; y >= 0; --y)
                        acc[x][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[x][y], acc[x][i], 0, 0, 0);
                keep_order();
            };
            if constexpr (kFp4) {
                if (__builtin_expect(__any(none == 0xffffffffu), 0))
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (blk.v4[i >> 2][i & 3] == 0xffffffffu) blk.v4[i >> 2][i & 3] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bf16x8 vf[2];
                    blk.operands_v(i, vf);
                    add_v(2 * i, vf[0]);
                    add_v(2 * i + 1, vf[1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) add_v(i, blk.operand(blk.v, i));
            }
            load_v(blk, next);
            kb += step;
        };
        for (;;) {
#pragma unroll
            for (int x = 0; x < kQT; ++x) {
                base[x] = kLowest;
                top[x] = kNegInf;
                sum[x] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[x][i] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
            }
            // (a way out of the middle of the loop would cost it the same)
            while (kb + (kStages - 1) * step < k1) {
#pragma unroll
                for (int i = 0; i < kStages; ++i) take(st[i]);
            }
#pragma unroll
            for (int i = 0; i + 1 < kStages; ++i)
                if (kb < k1) take(st[i]);
            bool over = false;
#pragma unroll
            for (int x = 0; x < kQT; ++x) {
                sum[x] = sum_groups(sum[x]);
                uint32_t most = 0;  // (as bits: NaN, which an infinite term leaves, lies above all)
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) most = max(most, __float_as_uint(acc[x][i][j]) & 0x7fffffffu);
                over |= most >= __float_as_uint(kLimit) && sum[x] == sum[x];  // (NaN scores stay NaN)
            }
            if (__builtin_expect(lowered || !__any(over), 1)) break;
            lowered = true;
            load_first();
            __builtin_amdgcn_s_waitcnt(0);  // (else the loop's waits would be for the order in which these loads are issued, too)
        }
        // the sum and O relative to base, base, and the true maximum
        if (lane == 0) sh.lowered[wave] = lowered;
#pragma unroll
        for (int x = 0; x < kQT; ++x) {
            const int to = wave * kQT + x;
            top[x] = max_groups(top[x]);
            if (g == 0) {
                sh.ml[to][0][n] = base[x];
                sh.ml[to][1][n] = sum[x];
                sh.ml[to][2][n] = top[x];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<floatx4*>(&sh.o[to][n][i * 16 + g * 4]) = acc[x][i];
        }
    }
};

// The waves' results meet: a thread sums four values of a row over the key waves, scaled to their common maximum. A wave that
// has a stretch of its own does so for itself. kLowered: O of some wave is times kLower, so all of them are taken so.
template <bool kLowered, bool kF32, int kQT, int kRows>
__device__ __forceinline__ void join_waves_as(const CachedAttnArgs& a, const AttnRowsOf<kRows>& rows, const Work& w, const Shared<kQT>& sh) {
    const int tid = thread_here(), wave = w.apart ? __builtin_amdgcn_readfirstlane(tid >> 6) : 0;
    const int wk = w.apart ? 1 : kWaves >> w.wl, tiles = w.apart ? kQT : kQT << w.wl, threads = w.apart ? 64 : 64 * kWaves;
    const int row0 = w.tile * 16 * tiles, nrows = min((w.prefix ? a.B : 1) * a.T * a.G - row0, 16 * tiles);
    for (int it = w.apart ? tid & 63 : tid; it < nrows * (kD / 4); it += threads) {
        const int d = (it & 31) * 4, rt = it >> 5;  // (row within the workgroup's tiles)
        const int tq = (rt >> 4) + wave * kQT, rn = rt & 15;
        float mx = kNegInf;
        for (int k = 0; k < wk; ++k) mx = fmaxf(mx, sh.ml[k * tiles + tq][2][rn]);
        const float base = mx == kNegInf ? 0.0f : mx;
        float l = 0.0f;
        floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < wk; ++k) {
            const int from = k * tiles + tq;
            float f = __builtin_amdgcn_exp2f(sh.ml[from][0][rn] - base);
            l += f * sh.ml[from][1][rn];
            if (kLowered && !sh.lowered[from / kQT]) f *= kLower;
            v += f * *reinterpret_cast<const floatx4*>(&sh.o[from][rn][d]);
        }
        const QueryRow to = query_row(a, row0 + rt, w.b, w.hk, w.prefix);
        const int64_t row = (static_cast<int64_t>(to.b) * a.T + to.t) * a.H + to.hq;
        if (w.part < 0) {
            const bool nan = l != l;  // (a maximum passes NaN scores over: they show in the sum)
            const bool empty = to.t >= rows.cnt[to.b] || (mx == kNegInf && !nan);
            v = empty ? (floatx4){0.0f, 0.0f, 0.0f, 0.0f} : v * (1.0f / l);
            if (kLowered) v *= kRaise;
            const int64_t at = row * kD + d;
            if constexpr (kF32) *reinterpret_cast<floatx4*>(static_cast<float*>(a.o) + at) = v;
            else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
            if (d == 0) {
                if (a.m) a.m[row] = empty ? kNegInf : nan ? l : mx * kLn2;
                if (a.l) a.l[row] = empty ? 0.0f : l;
            }
        } else {
            const int64_t part = row * a.parts + w.part;
            *reinterpret_cast<floatx4*>(a.part_o + part * kD + d) = v;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + part * 2) = make_float2(mx, kLowered ? -l : l);
        }
    }
}
template <bool kF32, int kQT, int kRows>
__device__ __forceinline__ void join_waves(const CachedAttnArgs& a, const AttnRowsOf<kRows>& rows, const Work& w, const Shared<kQT>& sh) {
    int lowered = 0;
    if (w.apart) lowered = sh.lowered[threadIdx.x >> 6];
    else
        for (int i = 0; i < kWaves; ++i) lowered |= sh.lowered[i];
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(lowered), 0)) join_waves_as<true, kF32>(a, rows, w, sh);
    else join_waves_as<false, kF32>(a, rows, w, sh);
}

// kQT, kPreQT: query tiles a wave for a batch row's own keys and for the prefix's
template <int kFormat, bool kF32, bool kOnce, int kQT, int kPreQT, int kRows>
__global__ __launch_bounds__(64 * kWaves, 2) void cached_attn_kernel(CachedAttnArgs a, AttnRowsOf<kRows> rows) {
    __shared__ __align__(16) union {
        Shared<kQT> own;
        Shared<kPreQT> pre;
    } sh;
    __shared__ AttnRowsOf<kRows> rl;
    // All arguments in one trip to their memory, in place of one for each dependent use: the batch rows into LDS (all of
    // them, so no length is waited for), the rest into scalar registers or at least the scalar cache.
    static_assert(64 * kWaves >= kRows, "one batch row a thread");
    if (threadIdx.x < kRows) {
        rl.len[threadIdx.x] = rows.len[threadIdx.x];
        rl.cum[threadIdx.x] = rows.cum[threadIdx.x];
        rl.slot[threadIdx.x] = rows.slot[threadIdx.x];
        rl.cnt[threadIdx.x] = rows.cnt[threadIdx.x];
    }
    asm volatile("" ::"s"(a.own.data), "s"(a.q), "s"(a.part_o), "s"(a.T), "s"(a.parts), "s"(a.share), "s"(a.pre_groups));
    __syncthreads();
    int id = blockIdx.x;
    Work w;
    w.prefix = id < a.pre_groups;
    w.wl = w.prefix ? a.pre_wl : a.apart ? kWavesLog : a.own_wl;
    w.apart = !w.prefix && a.apart;
    const int step_log = kStepLog - w.wl;
    int s = 0, end = 0, steps = 0, off = 0, count = 0;
    // the batch row's entries
    const auto load_row = [&]() {
        w.len = __builtin_amdgcn_readfirstlane(rl.len[w.b]);
        w.cnt = __builtin_amdgcn_readfirstlane(rl.cnt[w.b]);
        w.slot = __builtin_amdgcn_readfirstlane(rl.slot[w.b]);
        steps = steps_of(w.len, w.cnt, w.wl);
    };
    const auto set_keys = [&]() {
        w.k0 = off << step_log;
        w.k1 = min(w.len, (off + count) << step_log);
        if (a.causal && a.T > 1) {  // nothing past the tile's newest query
            const int r = ((w.tile + 1) * (16 * kQT) << (w.apart ? 0 : w.wl)) - 1, t = min(a.T - 1, a.G == 1 ? r : r / a.G);
            w.k1 = min(w.k1, max(0, w.len - w.cnt + t + 1));
        }
    };
    if (w.prefix) {
        // tiles of one chunk beside each other on one XCD (workgroups go to the eight XCDs in turn), which reads it once
        int item = id;
        w.tile = 0;
        if (a.pre_tiles > 1) {
            const int chunks = a.pre_groups / a.pre_tiles, full = chunks / 8 * 8 * a.pre_tiles;
            if (id < full) {
                const int oct = id / (8 * a.pre_tiles), rem = id - oct * 8 * a.pre_tiles;
                w.tile = rem >> 3;
                item = oct * 8 + (rem & 7);
            } else {
                const int left = chunks % 8;
                w.tile = (id - full) / left;
                item = chunks / 8 * 8 + (id - full) % left;
            }
        }
        w.part = item / a.pre.heads;
        w.hk = item - w.part * a.pre.heads;
        w.b = 0;
        w.k0 = w.part * a.pre_chunk;
        w.k1 = min(a.pre_len, w.k0 + a.pre_chunk);
        w.slot = a.pre_slot;
        w.len = a.pre_len;
        w.cnt = 0;
        Stretch<kFormat, kF32, false, kPreQT> st;
        st.begin(a, w);
        st.attend(a.scale, sh.pre);
        __syncthreads();
        join_waves<kF32, kPreQT, kRows>(a, rl, w, sh.pre);
        return;
    }
    {
        id -= a.pre_groups;
        // the list's neighbours on one XCD: they may share keys
        const int full = a.own_groups / 8 * 8;
        if (id < full) id = (id & 7) * (a.own_groups / 8) + (id >> 3);
        if (a.apart) {
            id = id * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            if (id >= a.own.heads * a.B * a.own_tiles) return;
        }
        if (a.aligned) {
            const int hb = a.own_tiles == 1 ? id : id / a.own_tiles;
            w.tile = id - hb * a.own_tiles;
            w.hk = hb / a.B;
            w.b = hb - w.hk * a.B;
            w.part = a.pre_parts > 0 ? a.pre_parts : -1;
            load_row();
            if (steps == 0 && a.pre_parts > 0) return;  // (only the prefix's parts are joined)
            count = steps;
        } else {
            s = share_start(a, id);
            end = share_start(a, id + 1);
            w.hk = s / a.head_places;
            const int in_head = s - w.hk * a.head_places;
            // the last batch row that begins at or before this place (rows without steps begin where the next one does)
            int below = 0;
#pragma unroll
            for (int i = 0; i < (kRows + 63) / 64; ++i) {
                const int at = i * 64 + (threadIdx.x & 63);
                if (i * 64 < a.B) below += __popcll(__ballot(at < a.B && rl.cum[at] <= in_head));
            }
            w.b = __builtin_amdgcn_readfirstlane(below) - 1;
            load_row();
            const int in_row = in_head - __builtin_amdgcn_readfirstlane(rl.cum[w.b]);
            w.tile = in_row / (steps + a.lead);
            off = in_row - w.tile * (steps + a.lead) - a.lead;
            if (off < 0) {
                s -= off;
                off = 0;
            }
            if (s >= end) return;  // (no step in this share)
            count = min(steps - off, end - s);
            w.part = a.pre_parts == 0 && count == steps ? -1 : a.pre_parts + id - group_of(a, s - off);
            s += count;
        }
        set_keys();
    }
    // the share's next triple, whole or as much of it as is left: tile, batch row, head
    const auto next = [&]() {
        if (++w.tile == a.own_tiles) {
            w.tile = 0;
            do {
                if (++w.b == a.B) {
                    w.b = 0;
                    ++w.hk;
                }
                load_row();
            } while (steps == 0);
        }
        off = 0;
        s += a.lead;
        count = min(steps, end - s);
        w.part = a.pre_parts == 0 && count == steps ? -1 : a.pre_parts;  // (its first part)
        s += count;
        set_keys();
    };
    Stretch<kFormat, kF32, kOnce, kQT> st;
    st.begin(a, w);
    for (;;) {
        st.attend(a.scale, sh.own);
        const Work done = w;
        if (w.apart) {  // (in its own part of LDS: a wave's accesses of it are in order)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            join_waves<kF32, kQT, kRows>(a, rl, w, sh.own);
            return;
        }
        const bool more = s + a.lead < end;
        if (more) {  // the next stretch's first loads are under way while this one is put together
            next();
            st.begin(a, w);
        }
        __syncthreads();
        join_waves<kF32, kQT, kRows>(a, rl, done, sh.own);
        if (!more) return;
        __syncthreads();
    }
}

// Joins a row's partial results: one workgroup a row, 32 threads across the 128 values, eight runs of parts.
template <bool kF32, int kRows>
__global__ __launch_bounds__(kJoinThreads) void cached_attn_join_kernel(CachedAttnArgs a, AttnRowsOf<kRows> rows) {
    __shared__ float red[kJoinThreads / 64];
    __shared__ float lred[8];
    __shared__ __align__(16) float obuf[8][kD];
    const int64_t row = blockIdx.x;
    const float* pml = a.part_ml + row * a.parts * 2;
    const float* po = a.part_o + row * a.parts * kD;
    const int run = threadIdx.x >> 5, d = (threadIdx.x & 31) * 4;
    // the first parts' values are under way before it is known how many there are
    floatx4 v0 = {0.0f, 0.0f, 0.0f, 0.0f};
    if (run < a.parts) v0 = *reinterpret_cast<const floatx4*>(po + static_cast<int64_t>(run) * kD + d);
    float2 s0 = make_float2(kNegInf, 0.0f);
    if (static_cast<int>(threadIdx.x) < a.parts) s0 = *reinterpret_cast<const float2*>(pml + 2 * threadIdx.x);
    const int hq = static_cast<int>(row % a.H), bt = static_cast<int>(row / a.H);
    const int b = bt / a.T, t = bt % a.T;
    int parts = 0;
    if (t < rows.cnt[b]) {
        const int steps = steps_of(rows.len[b], rows.cnt[b], a.own_wl);
        int own = steps > 0;
        if (own && !a.aligned) {
            const int first = hq / a.G * a.head_places + rows.cum[b] + ((t * a.G + hq % a.G) / (16 * a.own_qt << a.own_wl)) * (steps + a.lead) + a.lead;
            own = group_of(a, first + steps - 1) - group_of(a, first) + 1;
        }
        if (own == 1 && a.pre_parts == 0) return;  // (written already)
        parts = own + a.pre_parts;
    }
    float mx = static_cast<int>(threadIdx.x) < parts ? s0.x : kNegInf;
    for (int p = threadIdx.x + kJoinThreads; p < parts; p += kJoinThreads) mx = fmaxf(mx, pml[2 * p]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = mx == kNegInf ? 0.0f : mx;
    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    uint32_t signs = 0;
#pragma unroll 4
    for (int p = run; p < parts; p += 8) {
        const float2 s = *reinterpret_cast<const float2*>(pml + 2 * p);
        const floatx4 v = p == run ? v0 : *reinterpret_cast<const floatx4*>(po + static_cast<int64_t>(p) * kD + d);
        const float f = __builtin_amdgcn_exp2f(s.x - base);
        signs |= __float_as_uint(s.y);
        l += f * fabsf(s.y);
        acc += f * v;
    }
    if (__builtin_expect(signs >> 31, 0)) {  // (a run's parts with O times kLower: then all of the run)
        acc = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = run; p < parts; p += 8) {
            const float2 s = *reinterpret_cast<const float2*>(pml + 2 * p);
            const float f = __builtin_amdgcn_exp2f(s.x - base) * (s.y < 0.0f ? 1.0f : kLower);
            acc += f * *reinterpret_cast<const floatx4*>(po + static_cast<int64_t>(p) * kD + d);
        }
    }
    *reinterpret_cast<floatx4*>(&obuf[run][d]) = acc;
    if ((threadIdx.x & 31) == 0) lred[run] = signs >> 31 ? -l : l;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    l = 0.0f;
    acc = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
    signs = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        signs |= __float_as_uint(lred[i]);
        l += fabsf(lred[i]);
        acc += *reinterpret_cast<const floatx4*>(&obuf[i][d]);
    }
    const bool lowered = signs >> 31;
    if (__builtin_expect(lowered, 0)) {
        acc = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < 8; ++i) acc += (lred[i] < 0.0f ? 1.0f : kLower) * *reinterpret_cast<const floatx4*>(&obuf[i][d]);
    }
    const bool nan = l != l;  // (a maximum passes NaN scores over: they show in the sum)
    const bool empty = mx == kNegInf && !nan;
    acc = empty ? (floatx4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / l);
    if (lowered) acc *= kRaise;
    const int64_t at = row * kD + d;
    if constexpr (kF32) *reinterpret_cast<floatx4*>(static_cast<float*>(a.o) + at) = acc;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack2(acc[0], acc[1]), pack2(acc[2], acc[3]));
    if (threadIdx.x == 0) {
        if (a.m) a.m[row] = nan ? l : mx * kLn2;
        if (a.l) a.l[row] = empty ? 0.0f : l;
    }
}

constexpr int kCus = 256;
constexpr int kLead = 2;           // steps that beginning and ending a triple costs
constexpr int kApartSteps = 4;     // up to so many a triple may be one wave's

// Query tiles a wave, and log2 of the waves that take some: as many as there are tiles of 16 rows. Two tiles a wave where there
// are as many, so a held value is widened once for both (the exact mode has no registers for that).
int query_tiles(int64_t rows, bool f32) { return rows > 16 && !f32 ? 2 : 1; }
int query_waves_log(int64_t rows, int qt) { return rows <= 16 * qt ? 0 : rows <= 32 * qt || qt == 2 ? 1 : 2; }

// How a call is cut; fills rows' cum and the arguments that follow from the sizes. Returns the workspace's bytes.
int64_t make_plan(CachedAttnArgs& a, AttnRows& rows, int format, bool f32, bool* join) {
    // (in 4 bits the registers would hold three or four workgroups a CU: 32 of 8192 take 112 and 99 us then and 93 with two, 12 x 5 tokens
    // of 4 key/value heads behind 2777 28, 28 and 21)
    constexpr int kResident = 2 * kCus;
    const int heads = a.own.heads;
    const int64_t own_rows = static_cast<int64_t>(a.T) * a.G, all_rows = own_rows * a.B;
    a.own_qt = query_tiles(own_rows, f32);
    a.own_wl = query_waves_log(own_rows, a.own_qt);
    const int own_take = 16 * a.own_qt << a.own_wl;
    a.own_tiles = static_cast<int>((own_rows + own_take - 1) / own_take);
    int longest = 0, shortest = kMaxCacheTokens;
    int64_t steps = 0, rows_held = 0;
    for (int b = 0; b < a.B; ++b) {
        const int n = steps_of(rows.len[b], rows.cnt[b], a.own_wl);
        steps += n;
        rows_held += n > 0;
        longest = std::max(longest, n);
        shortest = std::min(shortest, n);
    }
    const int64_t all = steps * a.own_tiles * heads, triples = static_cast<int64_t>(heads) * a.B * a.own_tiles;

    // Many short triples: one a wave, whose latencies then overlap. At 16 heads in int8, one a workgroup and one a wave, us: 1024 of 1
    // key 11.3 and 5.4, of 256 keys 17.3 and 12.1, of 512 26.2 and 23.3; 4096 of 256 61 and 45, of 1024 166 and 168; 512 of 256
    // 9.1 and 11.0. In bf16, of twice the bytes, 4096 of 256 behind a prefix of 2048 are as fast either way, of 512 174 and 184.
    a.apart = own_rows <= 16 * a.own_qt && triples >= kResident + (a.pre_len == 0) &&
              longest <= (format == DT_KV_BF16 ? kApartSteps / 2 : kApartSteps) &&
              static_cast<int64_t>(longest) * kResident <= 2 * triples;
    a.pre_tiles = a.pre_qt = 1;
    a.pre_wl = a.pre_chunk = a.pre_parts = a.pre_groups = 0;
    if (a.pre_len > 0) {
        // as many of the workgroups as the prefix has of the waves' work (beginning and ending a triple costs about two steps; half of
        // both where each wave has one of its own)
        a.pre_qt = query_tiles(all_rows, f32);
        a.pre_wl = query_waves_log(all_rows, a.pre_qt);
        const int take = 16 * a.pre_qt << a.pre_wl;
        a.pre_tiles = static_cast<int>((all_rows + take - 1) / take);
        const int unit = (kKvBlock * kWaves) >> a.pre_wl;
        const int64_t pre_steps = (a.pre_len + unit - 1) / unit, per_chunk = static_cast<int64_t>(a.pre_tiles) * heads;
        const int64_t own_work = (all + kLead * rows_held * a.own_tiles * heads) >> a.apart;
        const int64_t groups = std::max<int64_t>(kResident * (pre_steps * per_chunk) / (pre_steps * per_chunk + own_work), 1);
        // but at least three steps each, 192 keys where those leave 64 rows of partial results: these weigh as much as the keys (16 heads
        // in fp8, us for two, three and four: 12 x 5 tokens behind 2777 16.0, 15.9 and 16.3, 8 tokens behind 1000 8.7, 8.9 and 9.5; in
        // exact mode, int8, 12 x 5 behind 2777 23.5, 19.9 and 21.3)
        const int64_t chunks = std::max<int64_t>(1, groups / per_chunk);
        const int64_t each = std::max<int64_t>(take == 64 ? 192 / unit : 3, (pre_steps + chunks - 1) / chunks);
        a.pre_chunk = static_cast<int>(std::min(each, pre_steps) * unit);
        a.pre_parts = (a.pre_len + a.pre_chunk - 1) / a.pre_chunk;
        a.pre_groups = static_cast<int>(a.pre_parts * per_chunk);
    }

    const int64_t slots = std::max<int64_t>(kResident - a.pre_groups, kResident / 4);
    // Triples are not cut where they are short, or so many that the longest does not show in the end: a workgroup's result is then
    // the last where there is no prefix, and no second launch is needed (3 us of the host's time). 16 heads in int8, whole and
    // cut, us: one sequence of 600 8.5 and 9.0, of 1024 10.6 and 8.9, of 1500 13.6 and 9.3; 8 of 1500 14.7 and 14.5; 16 of 2048
    // 23.9 and 27.1, 128 of up to 2048 88 and 92. Behind a prefix of 2048 one of 600 11.3 and 11.0, of 1024 13.5 and 11.0; 8 of
    // 1024 14.7 and 17.7; 16 of up to 2048 22 and 23, of 2048 35 and 31.
    // (An empty list has no shares; one past 2^28 steps has triples enough.)
    const int whole_steps = a.pre_len == 0 ? (triples < kCus ? 8 : 16) : (triples < kCus / 2 ? 4 : 8);
    a.aligned = a.apart || all == 0 || all > (1 << 28) || longest <= whole_steps || 4 * static_cast<int64_t>(longest) * slots <= all;
    int own_parts = 1;
    bool whole = true;  // every triple's keys in one workgroup
    a.own_groups = static_cast<int>(a.apart ? (triples + kWaves - 1) / kWaves : triples);
    if (!a.aligned) {
        // beginning a triple is counted where workgroups have several; one that is cut is begun twice, which no count would mend
        a.lead = rows_held * a.own_tiles * heads > slots ? kLead : 0;
        int64_t cum = 0;
        for (int b = 0; b < a.B; ++b) {
            rows.cum[b] = static_cast<int>(cum);
            const int n = steps_of(rows.len[b], rows.cnt[b], a.own_wl);
            if (n > 0) cum += static_cast<int64_t>(n + a.lead) * a.own_tiles;
        }
        a.head_places = static_cast<int>(cum);
        const int64_t places = cum * heads;
        a.own_groups = static_cast<int>(std::min<int64_t>(all, slots));
        a.share = static_cast<int>(places / a.own_groups);
        a.extra = static_cast<int>(places % a.own_groups);
        own_parts = std::min(longest, (longest - 1) / a.share + 2);
        whole = shortest == longest && a.extra == 0 && a.share % (longest + a.lead) == 0;
    }
    a.parts = own_parts + a.pre_parts;
    *join = !(whole && a.pre_parts == 0);
    return *join ? all_rows * heads * a.parts * (kD + 2) * static_cast<int64_t>(sizeof(float)) : 0;
}

template <int kRows>
int launch_rows(const CachedAttnArgs& a, const AttnRowsOf<kRows>& rows, bool join, int format, int dtype, hipStream_t s) {
    const int64_t groups = static_cast<int64_t>(a.own_groups) + a.pre_groups;
    if (groups > 0x7fffff) return set_error(DT_ERR_UNSUPPORTED, "the call needs %lld workgroups", (long long)groups);
    const bool f32 = dtype != DT_BF16;
    const bool once = a.own_wl == 0 && a.own_tiles == 1;
    if (groups > 0) {
        const dim3 g(static_cast<unsigned>(groups)), t(64 * kWaves);
        const auto go = [&](auto format_, auto f32_) {
            constexpr int F = decltype(format_)::value;
            constexpr bool M = decltype(f32_)::value;
            const auto go_as = [&](auto once_, auto qt_, auto pre_qt_) {
                hipLaunchKernelGGL((cached_attn_kernel<F, M, decltype(once_)::value, decltype(qt_)::value, decltype(pre_qt_)::value, kRows>),
                                   g, t, 0, s, a, rows);
            };
            constexpr std::integral_constant<int, 1> one;
            constexpr std::integral_constant<int, 2> two;
            constexpr std::true_type yes;
            constexpr std::false_type no;
            if constexpr (M) {
                if (once) go_as(yes, one, one);
                else go_as(no, one, one);
            } else {  // (more than one tile: two a wave)
                if (a.own_qt == 2 && once) go_as(yes, two, two);
                else if (a.own_qt == 2) go_as(no, two, two);
                else if (a.pre_qt == 2) go_as(yes, one, two);
                else go_as(yes, one, one);
            }
        };
        const auto go_mode = [&](auto format_) {
            if (f32) go(format_, std::true_type());
            else go(format_, std::false_type());
        };
        if (format == DT_KV_INT8) go_mode(std::integral_constant<int, DT_KV_INT8>());
        else if (format == DT_KV_FP8) go_mode(std::integral_constant<int, DT_KV_FP8>());
        else if (format == DT_KV_FP4) go_mode(std::integral_constant<int, DT_KV_FP4>());
        else go_mode(std::integral_constant<int, DT_KV_BF16>());
        DT_HIP_TRY(hipGetLastError());
    }
    if (!join) return DT_OK;
    const dim3 g(static_cast<unsigned>(static_cast<int64_t>(a.B) * a.T * a.H)), t(kJoinThreads);
    if (f32) hipLaunchKernelGGL((cached_attn_join_kernel<true, kRows>), g, t, 0, s, a, rows);
    else hipLaunchKernelGGL((cached_attn_join_kernel<false, kRows>), g, t, 0, s, a, rows);
    DT_HIP_TRY(hipGetLastError());
    return DT_OK;
}

int launch(const CachedAttnArgs& a, const AttnRows& rows, bool join, int format, int dtype, hipStream_t s) {
    if (a.B > kFewRows) return launch_rows(a, rows, join, format, dtype, s);
    AttnRowsOf<kFewRows> few;
    std::copy_n(rows.len, kFewRows, few.len);
    std::copy_n(rows.cum, kFewRows, few.cum);
    std::copy_n(rows.slot, kFewRows, few.slot);
    std::copy_n(rows.cnt, kFewRows, few.cnt);
    return launch_rows(a, few, join, format, dtype, s);
}

// what dt_cached_attn_fwd and its workspace query check alike; fills rows
int check_call(const dt_kv_cache* cache, int B, int T, int H, int D, const int32_t* slots, const int32_t* counts,
               const dt_kv_cache* prefix, int prefix_slot, int dtype, CachedAttnArgs* a, AttnRows* out) {
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
    KvRows rows;
    DT_TRY(kv_check_slots(cache, B, slots, false, &rows));
    DT_TRY(kv_check_counts(B, T, counts, &rows));
    for (int b = 0; b < B; ++b) {
        out->slot[b] = static_cast<uint16_t>(rows.slot[b]);
        out->cnt[b] = static_cast<uint16_t>(rows.cnt[b]);
        out->len[b] = cache->len[rows.slot[b]];
    }
    if (prefix) {
        if (prefix->heads != cache->heads || prefix->format != cache->format || prefix->ctx != cache->ctx)
            return set_error(DT_ERR_INVALID_ARG, "the prefix's cache has another context, format or number of heads");
        if (prefix_slot < 0 || prefix_slot >= prefix->slots)
            return set_error(DT_ERR_INVALID_ARG, "prefix_slot=%d outside [0, %d)", prefix_slot, prefix->slots);
        a->pre = prefix->view();
        a->pre_slot = prefix_slot;
        a->pre_len = prefix->len[prefix_slot];
    }
    a->own = cache->view();
    a->B = B;
    a->T = T;
    a->H = H;
    a->G = H / cache->heads;
    a->by_G = ((1ull << 40) + a->G - 1) / a->G;
    a->by_T = ((1ull << 40) + T - 1) / T;
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
    CachedAttnArgs a{};
    AttnRows rows{};
    bool join = false;
    DT_TRY(check_call(cache, B, T, H, D, slots, counts, prefix, prefix_slot, dtype, &a, &rows));
    *bytes = make_plan(a, rows, cache->format, dtype != DT_BF16, &join);
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
    CachedAttnArgs a{};
    AttnRows rows{};
    DT_TRY(check_call(cache, B, T, H, D, slots, counts, prefix, prefix_slot, dtype, &a, &rows));
    const size_t esz = dtype == DT_BF16 ? 2 : 4;
    const int64_t dm = static_cast<int64_t>(H) * kD;
    if (ldq < dm) return set_error(DT_ERR_INVALID_ARG, "row stride %lld is below %lld", (long long)ldq, (long long)dm);
    if (mem == DT_MEM_DEVICE && (!aligned16(q) || !aligned16(o) || !aligned16(ws) || ldq * esz % 16))
        return set_error(DT_ERR_INVALID_ARG, "device q/o/workspace and q's row stride must be 16-byte aligned");
    bool join = false;
    const int64_t need = make_plan(a, rows, cache->format, dtype != DT_BF16, &join);
    if (mem == DT_MEM_DEVICE && need > 0 && (!ws || ws_bytes < need))
        return set_error(DT_ERR_INVALID_ARG, "the workspace has %lld bytes, the call needs %lld", (long long)(ws ? ws_bytes : 0), (long long)need);
    dt_ctx* ctx = cache->ctx;
    DeviceScope scope;
    DT_TRY(scope.enter(cache->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    a.q = q;
    a.o = o;
    a.m = m;
    a.l = l;
    a.ldq = ldq;
    a.causal = causal;
    a.scale = scale;
    const int64_t part_floats = static_cast<int64_t>(B) * T * H * a.parts * kD;
    if (mem == DT_MEM_DEVICE) {
        a.part_o = static_cast<float*>(ws);
        a.part_ml = a.part_o + part_floats;
        return launch(a, rows, join, cache->format, dtype, s);
    }

    // host memory: staged through the context's buffers, synchronous
    const size_t tok = static_cast<size_t>(B) * T, row = dm * esz, nst = tok * H * sizeof(float);
    DT_TRY(ctx->stage[0].ensure(tok * row));
    DT_TRY(ctx->stage[1].ensure(tok * row));
    DT_TRY(ctx->stage[2].ensure(nst));
    DT_TRY(ctx->stage[3].ensure(nst));
    if (need > 0) DT_TRY(ctx->stage[4].ensure(need));
    DT_HIP_TRY(hipMemcpy2DAsync(ctx->stage[0].ptr, row, q, ldq * esz, row, tok, hipMemcpyHostToDevice, s));
    a.q = ctx->stage[0].ptr;
    a.o = ctx->stage[1].ptr;
    a.m = static_cast<float*>(ctx->stage[2].ptr);
    a.l = static_cast<float*>(ctx->stage[3].ptr);
    a.ldq = dm;
    a.part_o = static_cast<float*>(ctx->stage[4].ptr);
    a.part_ml = a.part_o + part_floats;
    DT_TRY(launch(a, rows, join, cache->format, dtype, s));
    DT_HIP_TRY(hipMemcpyAsync(o, a.o, tok * row, hipMemcpyDeviceToHost, s));
    if (m) DT_HIP_TRY(hipMemcpyAsync(m, a.m, nst, hipMemcpyDeviceToHost, s));
    if (l) DT_HIP_TRY(hipMemcpyAsync(l, a.l, nst, hipMemcpyDeviceToHost, s));
    DT_HIP_TRY(hipStreamSynchronize(s));
    return DT_OK;
}

}  // extern "C"
