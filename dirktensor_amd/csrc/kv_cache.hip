// The key/value cache: rows are quantised as they are written and read back as the values they stand for.
// Layout and formats: kv_cache.h.
//
// Bound by HBM where there is much to move: a written row costs its 512 (fp32) or 256 (bf16) bytes in and 132 (8 bits), 260 (bf16) or 68
// (4 bits) out, for K and V each. A workgroup takes the 32 keys of one block of one (batch row, head), eight threads to a key,
// 16 values a thread: the row's largest magnitude is then three lane exchanges away, K's values leave the
// registers as one 16-byte store a thread, and V's block, whose order in memory is the attention's, is put
// together in LDS and written whole. A block that the call covers only in part keeps the other keys' bytes: its V values go
// out as single bytes from the registers. Few tokens a sequence (a decode step's one) go another way, as a block would
// leave most threads idle: a wave takes one row of K or of V, two values a lane (kv_append_rows_kernel).
//
// Measured at 16 heads: 2 x 4096 tokens of bf16 into fp8 and back, 102 MB moved each time, 22.6 and 20.5 us (4.5 and 5.0 TB/s; a
// copy of 67 MB each way 4.9 through the caches, 5.5 past them), 17.6 and 19.8 with the rows in the caches (loads past these take
// 22.6 either way, stores past them 34). One token of eight sequences in int8 3.3 us, and read back 3.4, which is what a launch
// takes. In 4 bits 2 x 4096 tokens, 85 MB moved each time, 15.3 and 16.7 us (5.5 and 5.1 TB/s), 12 x 5 tokens 3.1 and 3.6.

#include "kv_cache.h"

#include <algorithm>
#include <cstring>
#include <new>

namespace dt {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr uint32_t kInfBits = 0x7f800000u;

struct KvMoveArgs {
    KvView c;
    void* k;  // rows of the caller: read by append, written by read
    void* v;
    int64_t ldk, ldv;    // token strides, elements
    int64_t bsk, bsv;    // batch strides
};

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){lo, hi}, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// 16 values of a row, 16-byte aligned; returns their largest magnitude as bits: these order like the numbers, an infinity
// above every number and a NaN above that
template <bool kBf16>
__device__ __forceinline__ uint32_t load16(const void* p, int64_t at, float (&x)[16]) {
    uint32_t amax = 0;
    if constexpr (kBf16) {
        const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
        u16x2 most = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = s[i];
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[8 * i + 2 * j] = bf16_lo(u[j]), x[8 * i + 2 * j + 1] = bf16_hi(u[j]);
                most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, u[j] & 0x7fff7fffu));
            }
        }
        amax = static_cast<uint32_t>(max(most[0], most[1])) << 16;
    } else {
        const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 w = s[i];
            x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    return amax;
}

template <bool kBf16>
__device__ __forceinline__ void store16(void* p, int64_t at, const float (&x)[16]) {
    if constexpr (kBf16) {
        uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            d[i] = make_uint4(pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                              pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7]));
    } else {
        float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
}

// A group's values in 4 bits, its scale's byte; amax_bits: the group's largest |x| as bits, finite: whether the row is.
template <int kN>
__device__ __forceinline__ uint32_t quantise4(const float (&x)[kN], uint32_t amax_bits, bool finite, uint32_t (&out)[(kN + 7) / 8]) {
    // amax = 1.f 2^a: the scale's exponent is a - 2, one more where 1.f > 1.5 (6 = 1.5 2^2)
    int e = static_cast<int>(amax_bits >> 23) - 127 - 2 + ((amax_bits & 0x7fffffu) > 0x400000u ? 1 : 0);
    e = !finite || e < -120 ? -120 : e;
    const float inv = finite ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : 0.0f;
    // at the top of the range (scale 2^126) 4 would stand for an infinity: 3 is the last value
    const float lim = e >= 126 ? 3.0f : 6.0f;
    float y[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) y[i] = finite ? __builtin_amdgcn_fmed3f(x[i] * inv, -lim, lim) : 0.0f;
#pragma unroll
    for (int i = 0; i < (kN + 7) / 8; ++i) {
        uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[8 * i], y[8 * i + 1], 1.0f, 0);
        if constexpr (kN >= 8) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[8 * i + 2], y[8 * i + 3], 1.0f, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[8 * i + 4], y[8 * i + 5], 1.0f, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[8 * i + 6], y[8 * i + 7], 1.0f, 3);
        }
        out[i] = w;
    }
    return finite ? static_cast<uint32_t>(127 + e) : kKvNoScale;
}

// 8 values of 4 bits times the scale of a byte
__device__ __forceinline__ void dequantise4(uint32_t w, uint32_t scale, float* x) {
    const float s = __uint_as_float(scale == kKvNoScale ? 0x7fc00000u : scale << 23);
    const floatx2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3)};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = v[i][0] * s, x[2 * i + 1] = v[i][1] * s;
}

// kN (16, or 2 in the low bits of one word) of a row's 128 values, quantised; amax_bits: the row's largest |x| as bits. Returns
// the scale.
constexpr int words_of(int format, int n) { return (n * kv_elem_bytes(format) + 3) / 4; }
template <int kFormat, int kN>
__device__ __forceinline__ float quantise(const float (&x)[kN], uint32_t amax_bits, uint32_t (&out)[words_of(kFormat, kN)]) {
    constexpr int kWords = words_of(kFormat, kN);
    const float amax = __uint_as_float(amax_bits);
    bool finite = amax_bits < kInfBits;
    if constexpr (kFormat == DT_KV_BF16) finite = finite && (pack_bf16x2(amax, 0.0f) & 0x7fffu) < 0x7f80u;
    if (!finite) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) out[i] = 0;
        return __uint_as_float(0x7fc00000u);
    }
    if constexpr (kFormat == DT_KV_BF16) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) out[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
        return 1.0f;
    } else if constexpr (kFormat == DT_KV_INT8) {
        const float s = amax / 127.0f;
        float y[kN], ss = s;
#pragma unroll
        for (int i = 0; i < kN; ++i) y[i] = x[i];
        if (__any(s < 0x1p-100f)) {
            // a scale near the end of the range, whose reciprocal is none, is divided by 2^100 times larger, like the values (which
            // pass 127 where it lost bits below 2^-126); with a scale of 0 (amax below 2^-143) all values are 0
            const float by = s >= 0x1p-100f ? 1.0f : s > 0.0f ? 0x1p100f : 0.0f;
            ss = s > 0.0f ? s * by : 1.0f;
#pragma unroll
            for (int i = 0; i < kN; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * by, -127.0f * ss, 127.0f * ss);
        }
        // The nearest whole number to the exact quotient y / s, ties to even. The sum of y * (1/s) with 1.5 2^23 rounds it; it is
        // off by one at most, and only where the quotient lies next to a half (which values of half the largest do): the remainder
        // y - q s decides. It is a multiple of the smaller unit in the last place of y and s (of y only where |q| <= 1) and no larger
        // than s, so the fma gives it exactly. An odd q moves at half a step too: its bound is the number below.
        constexpr float kMagic = 12582912.0f;
        const float quick = __builtin_amdgcn_rcpf(ss);
        const uint32_t half = __float_as_uint(0.5f * ss);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const float t = __builtin_fmaf(y[i], quick, kMagic);
            const float r = __builtin_fmaf(-(t - kMagic), ss, y[i]);
            const float bound = __uint_as_float(half - (__float_as_uint(t) & 1u));
            y[i] = t + (fabsf(r) > bound ? copysignf(1.0f, r) : 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {  // (the sum's low byte is the value)
            const auto low = [&](int j) { return __float_as_uint(y[4 * i + j]); };
            if constexpr (kN < 4) out[i] = __builtin_amdgcn_perm(low(1), low(0), 0x0c0c0400u);
            else
                out[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(low(3), low(2), 0x04000c0cu),
                                               __builtin_amdgcn_perm(low(1), low(0), 0x0c0c0400u), 0x07060100u);
        }
        return s;
    } else {
        // amax = 1.f 2^a: the scale's exponent is a - 8, one more where 1.f > 1.75 (448 = 1.75 2^8)
        int e = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        e = e < -126 ? -126 : e;
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        // at the top of the range (scale 2^120) 256 would stand for an infinity: 240 is the last value
        const float lim = e >= 120 ? 240.0f : 448.0f;
        float y[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -lim, lim);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
            if constexpr (kN >= 4) w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], w, true);
            out[i] = w;
        }
        return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
}

template <int kFormat>
__device__ __forceinline__ void dequantise(const uint32_t (&w)[kFormat == DT_KV_BF16 ? 8 : 4], float s, float (&x)[16]) {
    if constexpr (kFormat == DT_KV_BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[2 * i] = bf16_lo(w[i]) * s, x[2 * i + 1] = bf16_hi(w[i]) * s;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kFormat == DT_KV_INT8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j))) * s;
            } else {
                const floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), false);
                const floatx2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[i]), true);
                x[4 * i] = lo[0] * s, x[4 * i + 1] = lo[1] * s, x[4 * i + 2] = hi[0] * s, x[4 * i + 3] = hi[1] * s;
            }
        }
    }
}

// V's block in LDS: its 1 KB runs are 16 bytes further apart than in memory, which keeps the eight threads of a key off one
// bank
constexpr int kRunLds = kKvRun + 16;
template <int kFormat>
__device__ __forceinline__ int v_lds_offset(int d, int kk) {
    const int o = v_offset<kFormat>(d, kk);
    return (o >> 10) * kRunLds + (o & (kKvRun - 1));
}

// K's 16 values of thread part c of key kk: one or two 16-byte pieces
template <int kFormat>
__device__ __forceinline__ uint4* k_piece(uint8_t* block, int c, int kk, int i) {
    return reinterpret_cast<uint4*>(block + k_offset<kFormat>(c * 16 + i * 8, kk));
}
template <int kFormat>
__device__ __forceinline__ float* scale_of(uint8_t* block, bool v, int kk) {
    return reinterpret_cast<float*>(block + kv_scale_at(kFormat)) + (v ? kKvBlock : 0) + kk;
}

template <int kFormat, bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    constexpr int kEs = kv_elem_bytes(kFormat), kWords = 4 * kEs, kTensor = kv_tensor_bytes(kFormat);
    __shared__ __align__(16) uint8_t vbuf[kTensor / kKvRun * kRunLds];
    const int b = blockIdx.z, h = blockIdx.y;
    const int start = rows.len[b], cnt = rows.cnt[b];
    const int blk = start / kKvBlock + static_cast<int>(blockIdx.x);
    const int first = blk * kKvBlock;  // position of the block's first key
    if (first >= start + cnt) return;  // (whole workgroups)
    const int kk = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int t = first + kk - start;
    const bool mine = t >= 0 && t < cnt;
    const bool whole = first >= start && first + kKvBlock <= start + cnt;

    float x[16] = {}, y[16] = {};
    uint32_t kmax = 0, vmax = 0;
    if (mine) {
        kmax = load16<kBf16>(a.k, b * a.bsk + t * a.ldk + h * DT_HEAD_DIM + c * 16, x);
        vmax = load16<kBf16>(a.v, b * a.bsv + t * a.ldv + h * DT_HEAD_DIM + c * 16, y);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        kmax = max(kmax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(kmax), o, 64)));
        vmax = max(vmax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(vmax), o, 64)));
    }
    uint32_t qk[kWords], qv[kWords];
    const float sk = quantise<kFormat>(x, kmax, qk);
    const float sv = quantise<kFormat>(y, vmax, qv);

    uint8_t* block = a.c.block<kFormat>(rows.slot[b], h, blk);
    uint8_t* vd = block + kTensor;
    if (mine) {
#pragma unroll
        for (int i = 0; i < kEs; ++i) *k_piece<kFormat>(block, c, kk, i) = make_uint4(qk[4 * i], qk[4 * i + 1], qk[4 * i + 2], qk[4 * i + 3]);
        if (c == 0) {
            *scale_of<kFormat>(block, false, kk) = sk;
            *scale_of<kFormat>(block, true, kk) = sv;
        }
        const auto put = [&](auto* to, auto offset) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int o = offset(c * 16 + i, kk);
                if constexpr (kEs == 2) *reinterpret_cast<uint16_t*>(to + o) = static_cast<uint16_t>(qv[i >> 1] >> (16 * (i & 1)));
                else to[o] = static_cast<uint8_t>(qv[i >> 2] >> (8 * (i & 3)));
            }
        };
        if (whole) put(vbuf, v_lds_offset<kFormat>);
        else put(vd, v_offset<kFormat>);
    }
    if (whole) {  // (the same for the whole workgroup)
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEs; ++i) {
            const int o = (i * kThreads + threadIdx.x) * 16;
            *reinterpret_cast<uint4*>(vd + o) = *reinterpret_cast<const uint4*>(vbuf + (o >> 10) * kRunLds + (o & (kKvRun - 1)));
        }
    }
}

// Few tokens a sequence: a wave takes one row of K (even) or V (odd), lane i its values 2 i and 2 i + 1.
template <int kFormat, bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_append_rows_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    const int lane = threadIdx.x & 63, unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, t = blockIdx.y, h = unit >> 1;
    const bool v = unit & 1;
    if (h >= a.c.heads || t >= rows.cnt[b]) return;
    const int pos = rows.len[b] + t, d = 2 * lane;
    const int64_t at = v ? b * a.bsv + t * a.ldv : b * a.bsk + t * a.ldk;
    const void* src = v ? a.v : a.k;
    float x[2];
    if constexpr (kBf16) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(src) + at + h * DT_HEAD_DIM + d);
        x[0] = bf16_lo(w), x[1] = bf16_hi(w);
    } else {
        const float2 w = *reinterpret_cast<const float2*>(static_cast<const float*>(src) + at + h * DT_HEAD_DIM + d);
        x[0] = w.x, x[1] = w.y;
    }
    uint32_t amax = max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), o, 64)));
    uint32_t q[1];
    const float s = quantise<kFormat, 2>(x, amax, q);
    const int kk = pos & (kKvBlock - 1);
    uint8_t* block = a.c.block<kFormat>(rows.slot[b], h, pos / kKvBlock);
    if (lane == 0) *scale_of<kFormat>(block, v, kk) = s;
    if (!v) {  // (two neighbours lie in one piece)
        uint8_t* to = block + k_offset<kFormat>(d, kk);
        if constexpr (kFormat == DT_KV_BF16) *reinterpret_cast<uint32_t*>(to) = q[0];
        else *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(q[0]);
    } else {
        uint8_t* vd = block + kv_tensor_bytes(kFormat);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint8_t* to = vd + v_offset<kFormat>(d + i, kk);
            if constexpr (kFormat == DT_KV_BF16) *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(q[0] >> (16 * i));
            else *to = static_cast<uint8_t>(q[0] >> (8 * i));
        }
    }
}

// The same of a block in 4 bits. A byte of V has values 16 apart, of two neighbouring threads: these exchange theirs, and each writes
// eight of their sixteen bytes.
template <bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_append_fp4_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    constexpr int kTensor = kv_tensor_bytes(DT_KV_FP4);
    __shared__ __align__(16) uint8_t vbuf[kTensor / kKvRun * kRunLds];
    const int b = blockIdx.z, h = blockIdx.y;
    const int start = rows.len[b], cnt = rows.cnt[b];
    const int blk = start / kKvBlock + static_cast<int>(blockIdx.x);
    const int first = blk * kKvBlock;
    if (first >= start + cnt) return;  // (whole workgroups)
    const int kk = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int t = first + kk - start;
    const bool mine = t >= 0 && t < cnt;
    const bool whole = first >= start && first + kKvBlock <= start + cnt;

    float x[16] = {}, y[16] = {};
    uint32_t kmax = 0, vmax = 0;
    if (mine) {
        kmax = load16<kBf16>(a.k, b * a.bsk + t * a.ldk + h * DT_HEAD_DIM + c * 16, x);
        vmax = load16<kBf16>(a.v, b * a.bsv + t * a.ldv + h * DT_HEAD_DIM + c * 16, y);
    }
    const auto other = [](uint32_t v, int o) { return static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, 64)); };
    kmax = max(kmax, other(kmax, 1));  // (of the group)
    vmax = max(vmax, other(vmax, 1));
    uint32_t krow = max(kmax, other(kmax, 2)), vrow = max(vmax, other(vmax, 2));
    krow = max(krow, other(krow, 4));
    vrow = max(vrow, other(vrow, 4));
    uint32_t qk[2], qv[2];
    const uint32_t sk = quantise4(x, kmax, krow < kInfBits, qk), sv = quantise4(y, vmax, vrow < kInfBits, qv);
    const uint32_t pv[2] = {other(qv[0], 1), other(qv[1], 1)};

    uint8_t* block = a.c.block<DT_KV_FP4>(rows.slot[b], h, blk);
    uint8_t* vd = block + kTensor;
    if (mine) {
        *reinterpret_cast<uint2*>(block + k_offset<DT_KV_FP4>(c * 16, kk)) = make_uint2(qk[0], qk[1]);
        const int odd = c & 1;
        if (!odd) {
            reinterpret_cast<uint8_t*>(scale_of<DT_KV_FP4>(block, false, kk))[c >> 1] = static_cast<uint8_t>(sk);
            reinterpret_cast<uint8_t*>(scale_of<DT_KV_FP4>(block, true, kk))[c >> 1] = static_cast<uint8_t>(sv);
        }
        // values 8 odd .. 8 odd + 7 of both, the even thread's in the low halves
        const uint32_t low = odd ? pv[1] : qv[0], high = odd ? qv[1] : pv[0];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint8_t v = static_cast<uint8_t>((low >> (4 * i) & 15) | (high >> (4 * i) & 15) << 4);
            const int d = c * 16 + odd * 8 + i;
            if (whole) vbuf[v_lds_offset<DT_KV_FP4>(d, kk)] = v;
            else vd[v_offset<DT_KV_FP4>(d, kk)] = v;
        }
    }
    if (whole) {  // (the same for the whole workgroup)
        __syncthreads();
        if (threadIdx.x < kTensor / 16) {
            const int o = threadIdx.x * 16;
            *reinterpret_cast<uint4*>(vd + o) = *reinterpret_cast<const uint4*>(vbuf + (o >> 10) * kRunLds + (o & (kKvRun - 1)));
        }
    }
}

// Few tokens a sequence: a wave takes one row, 2 values a lane as above. A byte of V has values of lanes 8 apart.
template <bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_append_rows_fp4_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    const int lane = threadIdx.x & 63, unit = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, t = blockIdx.y, h = unit >> 1;
    const bool v = unit & 1;
    if (h >= a.c.heads || t >= rows.cnt[b]) return;
    const int pos = rows.len[b] + t, d = 2 * lane;
    const int64_t at = (v ? b * a.bsv + t * a.ldv : b * a.bsk + t * a.ldk) + h * DT_HEAD_DIM + d;
    const void* src = v ? a.v : a.k;
    float x[2];
    if constexpr (kBf16) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(src) + at);
        x[0] = bf16_lo(w), x[1] = bf16_hi(w);
    } else {
        const float2 w = *reinterpret_cast<const float2*>(static_cast<const float*>(src) + at);
        x[0] = w.x, x[1] = w.y;
    }
    uint32_t amax = max(__float_as_uint(x[0]) & 0x7fffffffu, __float_as_uint(x[1]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), o, 64)));
    uint32_t q[1];
    const uint32_t s = quantise4<2>(x, amax, !__any(amax >= kInfBits), q);
    const int kk = pos & (kKvBlock - 1);
    uint8_t* block = a.c.block<DT_KV_FP4>(rows.slot[b], h, pos / kKvBlock);
    if ((lane & 15) == 0) reinterpret_cast<uint8_t*>(scale_of<DT_KV_FP4>(block, v, kk))[lane >> 4] = static_cast<uint8_t>(s);
    if (!v) {
        block[k_offset<DT_KV_FP4>(d, kk)] = static_cast<uint8_t>(q[0]);
    } else {
        const uint32_t p = static_cast<uint32_t>(__shfl_xor(static_cast<int>(q[0]), 8, 64));
        const int odd = lane >> 3 & 1;  // which of the two this lane has, and which of its two values' bytes it writes
        const uint32_t low = odd ? p : q[0], high = odd ? q[0] : p;
        block[kv_tensor_bytes(DT_KV_FP4) + v_offset<DT_KV_FP4>(d + odd, kk)] = static_cast<uint8_t>((low >> (4 * odd) & 15) | (high >> (4 * odd) & 15) << 4);
    }
}

template <bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_read_fp4_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    constexpr int kTensor = kv_tensor_bytes(DT_KV_FP4);
    __shared__ __align__(16) uint8_t vbuf[kTensor / kKvRun * kRunLds];
    const int b = blockIdx.z, h = blockIdx.y;
    const int start = rows.len[b], cnt = rows.cnt[b];
    const int blk = start / kKvBlock + static_cast<int>(blockIdx.x);
    const int first = blk * kKvBlock;
    if (first >= start + cnt) return;
    const int kk = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int t = first + kk - start;
    const bool mine = t >= 0 && t < cnt;
    uint8_t* block = a.c.block<DT_KV_FP4>(rows.slot[b], h, blk);
    if (threadIdx.x < kTensor / 16) {
        const int o = threadIdx.x * 16;
        *reinterpret_cast<uint4*>(vbuf + (o >> 10) * kRunLds + (o & (kKvRun - 1))) = *reinterpret_cast<const uint4*>(block + kTensor + o);
    }
    const auto scale = [&](bool v) { return reinterpret_cast<const uint8_t*>(scale_of<DT_KV_FP4>(block, v, kk))[c >> 1]; };
    float x[16];
    if (mine) {
        const uint2 w = *reinterpret_cast<const uint2*>(block + k_offset<DT_KV_FP4>(c * 16, kk));
        dequantise4(w.x, scale(false), x);
        dequantise4(w.y, scale(false), x + 8);
        store16<kBf16>(a.k, b * a.bsk + t * a.ldk + h * DT_HEAD_DIM + c * 16, x);
    }
    __syncthreads();
    if (mine) {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w[i >> 3] |= (static_cast<uint32_t>(vbuf[v_lds_offset<DT_KV_FP4>(c * 16 + i, kk)]) >> (4 * (c & 1)) & 15) << (4 * (i & 7));
        dequantise4(w[0], scale(true), x);
        dequantise4(w[1], scale(true), x + 8);
        store16<kBf16>(a.v, b * a.bsv + t * a.ldv + h * DT_HEAD_DIM + c * 16, x);
    }
}

template <int kFormat, bool kBf16, int kRows>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvMoveArgs a, KvRowsOf<kRows> rows) {
    constexpr int kEs = kv_elem_bytes(kFormat), kWords = 4 * kEs, kTensor = kv_tensor_bytes(kFormat);
    __shared__ __align__(16) uint8_t vbuf[kTensor / kKvRun * kRunLds];
    const int b = blockIdx.z, h = blockIdx.y;
    const int start = rows.len[b], cnt = rows.cnt[b];
    const int blk = start / kKvBlock + static_cast<int>(blockIdx.x);
    const int first = blk * kKvBlock;
    if (first >= start + cnt) return;
    const int kk = threadIdx.x >> 3, c = threadIdx.x & 7;
    const int t = first + kk - start;
    const bool mine = t >= 0 && t < cnt;
    uint8_t* block = a.c.block<kFormat>(rows.slot[b], h, blk);

#pragma unroll
    for (int i = 0; i < kEs; ++i) {
        const int o = (i * kThreads + threadIdx.x) * 16;
        *reinterpret_cast<uint4*>(vbuf + (o >> 10) * kRunLds + (o & (kKvRun - 1))) = *reinterpret_cast<const uint4*>(block + kTensor + o);
    }
    float x[16];
    uint32_t w[kWords];
    if (mine) {
#pragma unroll
        for (int i = 0; i < kEs; ++i) {
            const uint4 u = *k_piece<kFormat>(block, c, kk, i);
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
        dequantise<kFormat>(w, *scale_of<kFormat>(block, false, kk), x);
        store16<kBf16>(a.k, b * a.bsk + t * a.ldk + h * DT_HEAD_DIM + c * 16, x);
    }
    __syncthreads();
    if (mine) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int o = v_lds_offset<kFormat>(c * 16 + i, kk);
            if constexpr (kEs == 2) w[i >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(vbuf + o)) << (16 * (i & 1));
            else w[i >> 2] |= static_cast<uint32_t>(vbuf[o]) << (8 * (i & 3));
        }
        dequantise<kFormat>(w, *scale_of<kFormat>(block, true, kk), x);
        store16<kBf16>(a.v, b * a.bsv + t * a.ldv + h * DT_HEAD_DIM + c * 16, x);
    }
}

template <bool kAppend, int kRows>
int launch_rows(const KvMoveArgs& a, const KvRowsOf<kRows>& rows, int B, int format, int dtype, hipStream_t s) {
    int blocks = 0, tokens = 0;  // of the batch row that touches most
    for (int b = 0; b < B; ++b)
        if (rows.cnt[b] > 0) {
            blocks = std::max(blocks, (rows.len[b] + rows.cnt[b] - 1) / kKvBlock - rows.len[b] / kKvBlock + 1);
            tokens = std::max(tokens, rows.cnt[b]);
        }
    if (blocks == 0) return DT_OK;
    // up to kFewTokens a wave a row: one token of 64 sequences (16 heads, int8) 6.3 us by blocks, 3.7 by rows, of 256 13.8 and 6.4;
    // sixteen of eight sequences 4.5 by blocks
    constexpr int kFewTokens = 8;
    const bool few = kAppend && tokens <= kFewTokens;
    const dim3 grid = few ? dim3((2 * a.c.heads + 3) / 4, tokens, B) : dim3(blocks, a.c.heads, B), block(kThreads);
    const bool bf16 = dtype == DT_BF16;
#define DT_KV_GO(F, M)                                                                                            \
    do {                                                                                                         \
        if constexpr (kAppend) {                                                                                 \
            if (few) hipLaunchKernelGGL((kv_append_rows_kernel<F, M, kRows>), grid, block, 0, s, a, rows);              \
            else hipLaunchKernelGGL((kv_append_kernel<F, M, kRows>), grid, block, 0, s, a, rows);                       \
        } else {                                                                                                 \
            hipLaunchKernelGGL((kv_read_kernel<F, M, kRows>), grid, block, 0, s, a, rows);                              \
        }                                                                                                        \
    } while (0)
#define DT_KV_GO2(F)                                                                                             \
    do {                                                                                                         \
        if (bf16) DT_KV_GO(F, true);                                                                             \
        else DT_KV_GO(F, false);                                                                                 \
    } while (0)
    if (format == DT_KV_FP4) {
#define DT_KV_GO4(M)                                                                                                       \
    do {                                                                                                                   \
        if constexpr (kAppend) {                                                                                           \
            if (few) hipLaunchKernelGGL((kv_append_rows_fp4_kernel<M, kRows>), grid, block, 0, s, a, rows);               \
            else hipLaunchKernelGGL((kv_append_fp4_kernel<M, kRows>), grid, block, 0, s, a, rows);                        \
        } else {                                                                                                           \
            hipLaunchKernelGGL((kv_read_fp4_kernel<M, kRows>), grid, block, 0, s, a, rows);                               \
        }                                                                                                                  \
    } while (0)
        if (bf16) DT_KV_GO4(true);
        else DT_KV_GO4(false);
#undef DT_KV_GO4
    } else if (format == DT_KV_INT8) DT_KV_GO2(DT_KV_INT8);
    else if (format == DT_KV_FP8) DT_KV_GO2(DT_KV_FP8);
    else DT_KV_GO2(DT_KV_BF16);
#undef DT_KV_GO2
#undef DT_KV_GO
    DT_HIP_TRY(hipGetLastError());
    return DT_OK;
}

template <bool kAppend>
int launch_move(const KvMoveArgs& a, const KvRows& rows, int B, int format, int dtype, hipStream_t s) {
    if (B > kFewRows) return launch_rows<kAppend>(a, rows, B, format, dtype, s);
    KvRowsOf<kFewRows> few;
    std::copy_n(rows.slot, kFewRows, few.slot);
    std::copy_n(rows.len, kFewRows, few.len);
    std::copy_n(rows.cnt, kFewRows, few.cnt);
    return launch_rows<kAppend>(a, few, B, format, dtype, s);
}

void free_cache(dt_kv_cache* c) {
    if (c->data) (void)hipFree(c->data);
    delete c;
}

int check_common(int B, int T, int dtype, int mem) {
    if (B < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d must be >= 1", B);
    if (B > kMaxRaggedBatch) return set_error(DT_ERR_UNSUPPORTED, "B=%d > %d", B, kMaxRaggedBatch);
    if (T < 1 || T > kMaxCacheTokens)
        return set_error(DT_ERR_INVALID_ARG, "%d tokens outside [1, %d]", T, kMaxCacheTokens);
    if (dtype != DT_FP32_EXACT && dtype != DT_BF16) return set_error(DT_ERR_INVALID_ARG, "unknown dtype %d", dtype);
    if (mem != DT_MEM_DEVICE && mem != DT_MEM_HOST) return set_error(DT_ERR_INVALID_ARG, "unknown mem %d", mem);
    return DT_OK;
}

}  // namespace

int kv_check_slots(const dt_kv_cache* c, int B, const int32_t* slots, bool distinct, KvRows* rows) {
    if (!slots && B > c->slots) return set_error(DT_ERR_INVALID_ARG, "B=%d exceeds the cache's %d slots", B, c->slots);
    for (int b = 0; b < B; ++b) {
        const int s = slots ? slots[b] : b;
        if (s < 0 || s >= c->slots) return set_error(DT_ERR_INVALID_ARG, "slots[%d]=%d outside [0, %d)", b, s, c->slots);
        rows->slot[b] = s;
    }
    if (slots && distinct)
        for (int b = 1; b < B; ++b)
            for (int a = 0; a < b; ++a)
                if (slots[a] == slots[b])
                    return set_error(DT_ERR_INVALID_ARG, "slots[%d] and slots[%d] are both %d", a, b, slots[a]);
    return DT_OK;
}

int kv_check_counts(int B, int T, const int32_t* counts, KvRows* rows) {
    for (int b = 0; b < B; ++b) {
        const int n = counts ? counts[b] : T;
        if (n < 0 || n > T) return set_error(DT_ERR_INVALID_ARG, "counts[%d]=%d outside [0, T=%d]", b, n, T);
        rows->cnt[b] = n;
    }
    return DT_OK;
}

}  // namespace dt

using namespace dt;

extern "C" {

int dt_kv_cache_create(dt_ctx* ctx, int slots, int capacity, int n_heads, int D, int format, dt_kv_cache** out) {
    clear_error();
    if (!out) return set_error(DT_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (D != DT_HEAD_DIM) return set_error(DT_ERR_UNSUPPORTED, "head_dim D=%d, kernels are built for D=%d", D, DT_HEAD_DIM);
    if (slots < 1 || slots > 65535) return set_error(DT_ERR_INVALID_ARG, "slots=%d outside [1, 65535]", slots);
    if (capacity < 1 || capacity > kMaxCacheTokens)
        return set_error(DT_ERR_INVALID_ARG, "capacity=%d outside [1, %d]", capacity, kMaxCacheTokens);
    if (n_heads < 1 || n_heads > kMaxCacheHeads)
        return set_error(DT_ERR_INVALID_ARG, "n_heads=%d outside [1, %d]", n_heads, kMaxCacheHeads);
    if (format != DT_KV_INT8 && format != DT_KV_FP8 && format != DT_KV_BF16 && format != DT_KV_FP4)
        return set_error(DT_ERR_INVALID_ARG, "unknown cache format %d", format);
    if (!ctx) return set_error(DT_ERR_INVALID_ARG, "ctx is NULL");
    DeviceScope scope;
    DT_TRY(scope.enter(ctx->device));
    dt_kv_cache* c = new (std::nothrow) dt_kv_cache;
    if (!c) return set_error(DT_ERR_INVALID_ARG, "out of host memory");
    c->ctx = ctx;
    c->device = ctx->device;
    c->slots = slots;
    c->capacity = capacity;
    c->heads = n_heads;
    c->format = format;
    c->blocks = (capacity + kKvBlock - 1) / kKvBlock;
    try {
        c->len.assign(slots, 0);
    } catch (const std::bad_alloc&) {
        free_cache(c);
        return set_error(DT_ERR_INVALID_ARG, "out of host memory");
    }
    const size_t bytes = static_cast<size_t>(slots) * n_heads * c->blocks * kv_block_bytes(format);
    hipError_t e = hipMalloc(&c->data, bytes);
    if (e == hipSuccess) e = hipMemset(c->data, 0, bytes);
    // the clearing is done before the call returns: streams that do not wait for the null stream may use the cache
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        free_cache(c);
        return set_error(DT_ERR_HIP, "a cache of %.1f GiB cannot be had: %s",
                         static_cast<double>(bytes) / (1u << 30), hipGetErrorString(e));
    }
    *out = c;
    return DT_OK;
}

int dt_kv_cache_destroy(dt_kv_cache* cache) {
    clear_error();
    if (!cache) return DT_OK;
    DeviceScope scope;
    DT_TRY(scope.enter(cache->device));
    free_cache(cache);  // (hipFree waits for the device)
    return DT_OK;
}

int dt_kv_cache_lengths(const dt_kv_cache* cache, int32_t* lengths) {
    clear_error();
    if (!cache) return set_error(DT_ERR_INVALID_ARG, "cache is NULL");
    if (!lengths) return set_error(DT_ERR_INVALID_ARG, "lengths is NULL");
    std::copy(cache->len.begin(), cache->len.end(), lengths);
    return DT_OK;
}

int dt_kv_cache_truncate(dt_kv_cache* cache, int B, const int32_t* slots, const int32_t* lengths) {
    clear_error();
    if (!lengths) return set_error(DT_ERR_INVALID_ARG, "lengths is NULL");
    if (B < 1) return set_error(DT_ERR_INVALID_ARG, "B=%d must be >= 1", B);
    if (!cache) return set_error(DT_ERR_INVALID_ARG, "cache is NULL");
    if (!slots && B > cache->slots)
        return set_error(DT_ERR_INVALID_ARG, "B=%d exceeds the cache's %d slots", B, cache->slots);
    for (int b = 0; b < B; ++b) {
        const int s = slots ? slots[b] : b;
        if (s < 0 || s >= cache->slots)
            return set_error(DT_ERR_INVALID_ARG, "slots[%d]=%d outside [0, %d)", b, s, cache->slots);
        if (lengths[b] < 0 || lengths[b] > cache->len[s])
            return set_error(DT_ERR_INVALID_ARG, "lengths[%d]=%d outside [0, %d], what slot %d holds", b, lengths[b],
                             cache->len[s], s);
    }
    for (int b = 0; b < B; ++b) {  // (a slot named twice keeps the least)
        int32_t& n = cache->len[slots ? slots[b] : b];
        n = std::min(n, lengths[b]);
    }
    return DT_OK;
}

int dt_kv_cache_append(dt_kv_cache* cache, const void* k, const void* v, int B, int T, int64_t ldk, int64_t ldv,
                       const int32_t* slots, const int32_t* counts, int dtype, int mem, void* stream) {
    clear_error();
    if (!k || !v) return set_error(DT_ERR_INVALID_ARG, "k and v must be non-NULL");
    DT_TRY(check_common(B, T, dtype, mem));
    const size_t esz = dtype == DT_BF16 ? 2 : 4;
    if (mem == DT_MEM_DEVICE && (!aligned16(k) || !aligned16(v) || ldk * esz % 16 || ldv * esz % 16))
        return set_error(DT_ERR_INVALID_ARG, "device k/v and their row strides must be 16-byte aligned");
    if (!cache) return set_error(DT_ERR_INVALID_ARG, "cache is NULL");
    const int64_t dm = static_cast<int64_t>(cache->heads) * DT_HEAD_DIM;
    if (ldk < dm || ldv < dm)
        return set_error(DT_ERR_INVALID_ARG, "row strides %lld, %lld are below %lld", (long long)ldk, (long long)ldv, (long long)dm);
    KvRows rows{};
    DT_TRY(kv_check_slots(cache, B, slots, true, &rows));
    DT_TRY(kv_check_counts(B, T, counts, &rows));
    for (int b = 0; b < B; ++b) {
        rows.len[b] = cache->len[rows.slot[b]];
        if (rows.cnt[b] > cache->capacity - rows.len[b])
            return set_error(DT_ERR_INVALID_ARG, "slot %d holds %d of %d tokens: %d more do not fit", rows.slot[b],
                             rows.len[b], cache->capacity, rows.cnt[b]);
    }
    DeviceScope scope;
    DT_TRY(scope.enter(cache->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    KvMoveArgs a{cache->view(), const_cast<void*>(k), const_cast<void*>(v), ldk, ldv, T * ldk, T * ldv};
    if (mem == DT_MEM_HOST) {
        const size_t rowb = dm * esz;
        for (int i = 0; i < 2; ++i) {
            DT_TRY(cache->ctx->stage[i].ensure(rowb * B * T));
            DT_HIP_TRY(hipMemcpy2DAsync(cache->ctx->stage[i].ptr, rowb, i ? v : k, (i ? ldv : ldk) * esz, rowb,
                                        static_cast<size_t>(B) * T, hipMemcpyHostToDevice, s));
        }
        a.k = cache->ctx->stage[0].ptr;
        a.v = cache->ctx->stage[1].ptr;
        a.ldk = a.ldv = dm;
        a.bsk = a.bsv = T * dm;
    }
    DT_TRY(launch_move<true>(a, rows, B, cache->format, dtype, s));
    if (mem == DT_MEM_HOST) DT_HIP_TRY(hipStreamSynchronize(s));
    for (int b = 0; b < B; ++b) cache->len[rows.slot[b]] += rows.cnt[b];
    return DT_OK;
}

int dt_kv_cache_read(dt_kv_cache* cache, void* k, void* v, int B, int T, const int32_t* slots, const int32_t* starts,
                     int dtype, int mem, void* stream) {
    clear_error();
    if (!k || !v) return set_error(DT_ERR_INVALID_ARG, "k and v must be non-NULL");
    DT_TRY(check_common(B, T, dtype, mem));
    if (mem == DT_MEM_DEVICE && (!aligned16(k) || !aligned16(v)))
        return set_error(DT_ERR_INVALID_ARG, "device k/v must be 16-byte aligned");
    if (!cache) return set_error(DT_ERR_INVALID_ARG, "cache is NULL");
    KvRows rows{};
    DT_TRY(kv_check_slots(cache, B, slots, false, &rows));
    for (int b = 0; b < B; ++b) {
        rows.len[b] = starts ? starts[b] : 0;
        rows.cnt[b] = T;
        const int held = cache->len[rows.slot[b]];
        if (rows.len[b] < 0 || rows.len[b] > held || T > held - rows.len[b])
            return set_error(DT_ERR_INVALID_ARG, "%d tokens from %d on: slot %d holds %d", T, rows.len[b], rows.slot[b], held);
    }
    DeviceScope scope;
    DT_TRY(scope.enter(cache->device));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t dm = static_cast<int64_t>(cache->heads) * DT_HEAD_DIM;
    KvMoveArgs a{cache->view(), k, v, dm, dm, T * dm, T * dm};
    const size_t bytes = static_cast<size_t>(B) * T * dm * (dtype == DT_BF16 ? 2 : 4);
    if (mem == DT_MEM_HOST) {
        for (int i = 0; i < 2; ++i) DT_TRY(cache->ctx->stage[i].ensure(bytes));
        a.k = cache->ctx->stage[0].ptr;
        a.v = cache->ctx->stage[1].ptr;
    }
    DT_TRY(launch_move<false>(a, rows, B, cache->format, dtype, s));
    if (mem == DT_MEM_HOST) {
        DT_HIP_TRY(hipMemcpyAsync(k, a.k, bytes, hipMemcpyDeviceToHost, s));
        DT_HIP_TRY(hipMemcpyAsync(v, a.v, bytes, hipMemcpyDeviceToHost, s));
        DT_HIP_TRY(hipStreamSynchronize(s));
    }
    return DT_OK;
}

}  // extern "C"
