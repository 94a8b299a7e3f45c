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
//   fp4   four scales, one for each 32 values: the smallest power of two (at least 2^-120) with amax / scale <= 6, as its
//         exponent + 127 in a byte each of the row's 32 bits; value = x / scale as e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), ties to
//         even; where it would stand for more than fp32's range, the largest that does not
// A row that holds an infinity or a NaN (in bf16 also one that rounding makes infinite) has value 0 and scale
// NaN (fp4: bytes of 255): it reads back as NaN, and no held value is ever infinite or NaN. A masked key may then go through the
// matrix instructions with probability 0 (0 times a held value is 0).
//
// Per (slot, head), keys in blocks of 32 (the k extent of one v_mfma_f32_16x16x32_bf16), a block's K, V and scales behind
// each other, so a reader streams one run of memory:
//   K       32 x 128 values in the order in which the A operand of S^T = K Q^T reads them
//   V       32 x 128 values in the order of the A operand of O^T = V^T P^T
//   scales  of K [32], of V [32]
// A lane's fragment is one 16-byte load and a wave's load one run of 1 KB: see k_offset and v_offset. All of it is zeroed
// when the cache is made, and the block that a length ends in lies whole in the buffer.
#pragma once

#include "dt_internal.h"

namespace dt {

constexpr int kKvBlock = 32;
constexpr int kMaxCacheTokens = 1 << 20;
constexpr int kMaxCacheHeads = 1024;

// Which slot and how many tokens a call's batch rows take, by value in the kernel's arguments: places for kFewRows where these are
// enough, as each launch copies its arguments (eager calls on 8 rows: append 8.3 and 8.0 us, read 8.2 and 7.9).
constexpr int kFewRows = 32;
template <int kN>
struct KvRowsOf {
    int32_t slot[kN];
    int32_t len[kN];  // tokens held (attention), or the first position (append, read)
    int32_t cnt[kN];  // tokens of this call
};
using KvRows = KvRowsOf<kMaxRaggedBatch>;

__host__ __device__ constexpr int kv_elem_bits(int format) { return format == DT_KV_BF16 ? 16 : format == DT_KV_FP4 ? 4 : 8; }
__host__ __device__ constexpr int kv_elem_bytes(int format) { return kv_elem_bits(format) / 8; }  // (of formats that have whole ones)

constexpr int kKvRun = 1024;  // bytes of a wave's load
constexpr int kKvGroup = 32;  // fp4: values of a scale
constexpr uint32_t kKvNoScale = 255;  // fp4: the scale of a row that is none
__host__ __device__ constexpr int kv_tensor_bytes(int format) { return kKvBlock * DT_HEAD_DIM * kv_elem_bits(format) / 8; }
__host__ __device__ constexpr int kv_scale_at(int format) { return 2 * kv_tensor_bytes(format); }  // K's; V's behind
__host__ __device__ constexpr int kv_block_bytes(int format) { return kv_scale_at(format) + 2 * kKvBlock * 4; }

// Byte offset of value d (0..127) of key kk (0..31) in a block's K. The A operand of the 16x16x32 product takes 16 keys
// (lane & 15) and 32 values d, 8 a lane group g = lane >> 4; which those are may be chosen freely as long as Q's fragment has the
// same order. A 16-byte piece has 16 (8 bits) or 8 (bf16) consecutive ones: two steps, or one. In fp4
// it has 32, all four steps of the lane group, which share a scale; the offset is that of the byte, an even d in its low half.
template <int kFormat>
__host__ __device__ __forceinline__ int k_offset(int d, int kk) {
    const int tile = kk >> 4, m = kk & 15;
    if constexpr (kFormat == DT_KV_BF16) return tile * 4096 + (d >> 5) * kKvRun + ((d >> 3 & 3) * 16 + m) * 16 + (d & 7) * 2;
    if constexpr (kFormat == DT_KV_FP4) return tile * kKvRun + ((d >> 5) * 16 + m) * 16 + ((d & 31) >> 1);
    return tile * 2048 + (d >> 6) * kKvRun + ((d >> 4 & 3) * 16 + m) * 16 + (d & 15);
}

// Byte offset of value d of key kk in a block's V. The operand takes 16 values d (lane & 15) and 32 keys, 8 a lane group.
// P comes out of S^T's accumulators, where group g holds keys 4g..4g+3 of each 16-key tile: so slots 0..3 are those of the
// first tile, 4..7 those of the second. In fp4 a byte has
// the values d and d + 16 of a key, which share a scale: one instruction makes bf16 of both.
template <int kFormat>
__host__ __device__ __forceinline__ int v_offset(int d, int kk) {
    const int g = (kk & 15) >> 2, j = (kk >> 4) * 4 + (kk & 3);
    const int mt = d >> 4, lane = g * 16 + (d & 15);
    if constexpr (kFormat == DT_KV_BF16) return mt * kKvRun + lane * 16 + j * 2;
    if constexpr (kFormat == DT_KV_FP4) return (mt >> 2) * kKvRun + lane * 16 + (mt >> 1 & 1) * 8 + j;
    return (mt >> 1) * kKvRun + lane * 16 + (mt & 1) * 8 + j;
}

struct KvView {
    uint8_t* data;
    int blocks;  // allocated per (slot, head)
    int heads;
    template <int kFormat>
    __device__ __forceinline__ uint8_t* block(int slot, int head, int blk) const {
        return data + ((static_cast<int64_t>(slot) * heads + head) * blocks + blk) * kv_block_bytes(kFormat);
    }
};

}  // namespace dt

struct dt_kv_cache {
    dt_ctx* ctx = nullptr;
    int device = 0, slots = 0, capacity = 0, heads = 0, format = 0;
    int blocks = 0;  // of 32 tokens per (slot, head)
    void* data = nullptr;
    std::vector<int32_t> len;  // tokens held by each slot
    dt::KvView view() const { return {static_cast<uint8_t*>(data), blocks, heads}; }
};

namespace dt {
// the batch rows' slots (NULL: 0 .. B-1): in range, and, for a call that writes them, each once
int kv_check_slots(const dt_kv_cache* c, int B, const int32_t* slots, bool distinct, KvRows* rows);
// tokens of each batch row (NULL: T each), in [0, T]
int kv_check_counts(int B, int T, const int32_t* counts, KvRows* rows);
}  // namespace dt
