// The key/value cache's layout in device memory, shared by the kernels that write it, read it back and attend
// over it (kv_cache.hip, cached_attn.hip).
//
// A row is the 128 values of one (slot, head, token). It is held as 128 values of the cache's format and one
// fp32 scale; what it stands for is value * scale:
//   int8  scale = amax / 127, value = x / scale to the nearest whole number, ties to even
//   fp8   scale = the smallest power of two (at least 2^-126) with amax / scale <= 448, value = x / scale as
//         e4m3, ties to even: a power of two leaves the division exact, and e4m3's relative step does not gain from
//         a finer scale; where the value would stand for more than fp32's range, the largest that does not
//   bf16  value = x as bf16, scale 1
// A row that holds an infinity or a NaN (in bf16 also one that rounding makes infinite) has value 0 and scale
// NaN: it reads back as NaN, and no held value is ever infinite or NaN. A masked key may then go through the
// matrix instructions with probability 0 (0 times a held value is 0).
//
// Per (slot, head), keys in blocks of 32 (the k extent of one v_mfma_f32_16x16x32_bf16):
//   K       [key][128 values], row-major: the A operand of S^T = K Q^T has 8 consecutive values a lane
//   V       each block in the order in which the A operand of O^T = V^T P^T reads it, so a lane's fragment is one
//           16-byte load: see v_offset
//   scales  [key] for K and V each
// All of it is zeroed when the cache is made, and the block that a length ends in lies whole in the buffer.
#pragma once

#include "dt_internal.h"

namespace dt {

constexpr int kKvBlock = 32;
constexpr int kMaxCacheTokens = 1 << 20;
constexpr int kMaxCacheHeads = 1024;

// Which slot and how many tokens a call's batch rows take, by value in the kernel's arguments.
struct KvRows {
    int32_t slot[kMaxRaggedBatch];
    int32_t len[kMaxRaggedBatch];  // tokens held (attention), or the first position (append, read)
    int32_t cnt[kMaxRaggedBatch];  // tokens of this call
};

__host__ __device__ constexpr int kv_elem_bytes(int format) { return format == DT_KV_BF16 ? 2 : 1; }

// Byte offset of value d (0..127) of key kk (0..31) in a block of V. The A operand of the 16x16x32 product takes
// 16 values d (lane & 15) and 32 keys, 8 a lane group g = lane >> 4; which keys those are may be chosen freely as
// long as P's fragment has the same order. P comes out of S^T's accumulators, where group g holds keys 4g..4g+3
// of each 16-key tile: so slots 0..3 are those of the first tile, 4..7 those of the second.
template <int kFormat>
__device__ __forceinline__ int v_offset(int d, int kk) {
    const int g = (kk & 15) >> 2, j = (kk >> 4) * 4 + (kk & 3);
    const int mt = d >> 4, lane = g * 16 + (d & 15);
    if constexpr (kFormat == DT_KV_BF16) return mt * 1024 + lane * 16 + j * 2;
    return (mt >> 1) * 1024 + lane * 16 + (mt & 1) * 8 + j;
}

struct KvView {
    uint8_t* k;
    uint8_t* v;
    float* ks;
    float* vs;
    int64_t keys;  // keys allocated per (slot, head), a multiple of kKvBlock
    int heads;
};

}  // namespace dt

struct dt_kv_cache {
    dt_ctx* ctx = nullptr;
    int slots = 0, capacity = 0, heads = 0, format = 0;
    int64_t keys = 0;
    void* k = nullptr;
    void* v = nullptr;
    float* ks = nullptr;
    float* vs = nullptr;
    std::vector<int32_t> len;  // tokens held by each slot
    dt::KvView view() const {
        return {static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), ks, vs, keys, heads};
    }
};

namespace dt {
// the batch rows' slots (NULL: 0 .. B-1): in range, and, for a call that writes them, each once
int kv_check_slots(const dt_kv_cache* c, int B, const int32_t* slots, bool distinct, KvRows* rows);
// tokens of each batch row (NULL: T each), in [0, T]
int kv_check_counts(int B, int T, const int32_t* counts, KvRows* rows);
}  // namespace dt
