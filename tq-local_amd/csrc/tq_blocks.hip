// tq_blocks.hip -- bounds of the keys of every 64 tokens, and the blocks that a query chooses by them (gfx950).
//
// A block's keys lie between lo and hi, channel by channel, so no key of it gives the query q a larger product than
//   sum_d max(q_d lo_d, q_d hi_d).
// lo and hi are whole numbers of a step of the block's own, rounded outward to 8 bits, and q is rounded to whole numbers too: the sum is
// a whole number below 2^22, the step a power of two, and so every score is exact in fp32, whatever the order of its sum.  The same
// blocks are chosen everywhere, and a block's bounds are the same however its keys arrived.
//
//   bounds_kernel  a block per wave, 16 bytes of four keys a lane and load, all of a block's loads in flight together.  Bound by memory:
//                  8 sequences of 32768 tokens of 8 KV heads (537 MB) take 94 to 99 us, 5.4 to 5.7 TB/s; one of 131072 43 us, 6.3 TB/s
//                  (part of it from the last-level cache); a block of each of 64 KV heads 4 us, first bytes and launch
//   select_kernel  a KV head's whole choice per workgroup: scores by v_mfma_i32_16x16x64_i8, a column for a block, then the keep-th
//                  largest by radix and the chosen numbers in order.  Bound by the steps that wait for one another: 32 of 129 blocks
//                  for 8 KV heads take 6.3 us, 64 of 512 for 64 KV heads 10
//   score_kernel   the scores of longer histories, spread over the CUs; the choice then reads 4 bytes of a block instead of 260.  128 of
//                  2048 blocks for 32 KV heads take 14.5 us, the scores 6 of them (17 MB, 2.8 TB/s) and the choice 7

#include <algorithm>

#include "tq_common.h"

namespace {

constexpr int D = TQ_DIM, BT = TQ_BLOCK_TOKENS;
constexpr int MAX_EXP = 100;  // a step is from 2^-MAX_EXP to 2^MAX_EXP

typedef int i32x4 __attribute__((ext_vector_type(4)));

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The exponent of the least step whose 127-fold is not below a number, from the bits of its absolute value (fp32, infinities and NaN
// as such): 127 = 1.984375 2^6.
__device__ __forceinline__ int step_exponent(uint32_t bits) {
    const int e = (int)(bits >> 23) - 127 - 6 + ((bits & 0x7FFFFFu) > 0x7E0000u);
    return std::min(std::max(e, -MAX_EXP), MAX_EXP);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// ------------------------------------------------------------------ bounds

// Two bf16 numbers as int16 whose order is theirs (NaN beyond the infinity of its sign), and back.
__device__ __forceinline__ uint32_t ordered(uint32_t x) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const s16x2 sign = __builtin_bit_cast(s16x2, x) >> 15;
    return x ^ (__builtin_bit_cast(uint32_t, sign) & 0x7FFF7FFFu);
}
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, a), __builtin_bit_cast(s16x2, b)));
}

// fp32 bits as an integer whose order is theirs (NaN as above), and back.
__device__ __forceinline__ int ordered(float x) {
    const int b = __float_as_int(x);
    return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ uint32_t unordered(int x) { return (uint32_t)(x ^ ((x >> 31) & 0x7FFFFFFF)); }

struct BoundsArgs {
    const void* k;
    int heads;
    int64_t tokens, k_sb, k_sh, k_st;
    int8_t* lohi;
    float* step;
    int64_t cap, first, per_head, all;  // blocks to a head, and of all heads
    // whether neighbouring waves have a block's heads, or a head's blocks: what is next to one another in memory.  The 8 sequences above, us,
    // a head's blocks and a block's heads: rows of a token together 99 and 94, rows of a head together 97 and 108
    int heads_next;
};

// Whole numbers outward of eight channels' least or largest keys (fp32 bits) over a step (times `down`), four to a word.
__device__ __forceinline__ uint2 outward8(const uint32_t* bits, bool upper, float down) {
    uint32_t out[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // an infinity for NaN too
        const float v = __uint_as_float((bits[j] & 0x80000000u) | std::min(bits[j] & 0x7FFFFFFFu, 0x7F800000u)) * down;
        float r = fminf(fmaxf(upper ? __builtin_ceilf(v) : __builtin_floorf(v), -127.0f), 127.0f);
        // a number less than 2^-149 of a step gives the product 0, and is rounded outward all the same
        if (r == 0.0f && (bits[j] << 1) != 0u && upper != (bool)(bits[j] >> 31)) r = upper ? 1.0f : -1.0f;
        out[j >> 2] |= ((uint32_t)(int)r & 0xFFu) << (8 * (j & 3));
    }
    return make_uint2(out[0], out[1]);
}

// TYPE: of the keys, 0: bf16, 1: fp32, 2: fp16.  16-bit keys are compared two at a time as they are; a bf16 or fp16 number is an fp32 one, so
// the bounds are of the keys as given whatever their type.  fp32 keys are twice the bytes: the 8 sequences
// above 190 to 194 us, 5.6 TB/s.
constexpr int BOUNDS_WAVES = 4;
template <int TYPE>
__global__ __launch_bounds__(64 * BOUNDS_WAVES) void bounds_kernel(BoundsArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = (int64_t)blockIdx.x * BOUNDS_WAVES + wave;
    if (at >= a.all) return;
    int64_t group, block;
    if (a.heads_next) {
        const int64_t place = at / a.heads, b = place / a.per_head;
        block = place - b * a.per_head, group = b * a.heads + (at - place * a.heads);
    } else {
        group = at / a.per_head, block = at - group * a.per_head;
    }
    const int64_t b = group / a.heads, h = group - b * a.heads, first = b * a.k_sb + h * a.k_sh + block * BT * a.k_st;
    const int left = (int)std::min<int64_t>(a.tokens - block * BT, BT);
    // lane (c = lane % 16, t = lane / 16): channels [8 c, 8 c + 8) of the tokens t, t + 4, ...; past the last it again
    const int c = lane & 15, t = lane >> 4;
    const bool upper = t == 1;  // lanes t = 0 write lo, t = 1 hi
    uint32_t most = 0u;         // the largest absolute value, as fp32 bits
    uint32_t mine[8];           // the lane's eight bounds
    if constexpr (TYPE == 1) {
        const float* const k = static_cast<const float*>(a.k) + first;
        int lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) lo[j] = 0x7FFFFFFF, hi[j] = (int)0x80000000u;
        constexpr int SETS = 2;  // half of a block's loads in flight together, 64 registers
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
            float4 x[BT / 4 / SETS][2];
#pragma unroll
            for (int i = 0; i < BT / 4 / SETS; ++i) {
                const float* const row = k + std::min(4 * (BT / 4 / SETS * s + i) + t, left - 1) * a.k_st + 8 * c;
                x[i][0] = *reinterpret_cast<const float4*>(row), x[i][1] = *reinterpret_cast<const float4*>(row + 4);
            }
#pragma unroll
            for (int i = 0; i < BT / 4 / SETS; ++i) {
                const float w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) lo[j] = std::min(lo[j], ordered(w[j])), hi[j] = std::max(hi[j], ordered(w[j]));
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int d = 16; d < 64; d <<= 1) lo[j] = std::min(lo[j], __shfl_xor(lo[j], d)), hi[j] = std::max(hi[j], __shfl_xor(hi[j], d));
            const uint32_t l = unordered(lo[j]), u = unordered(hi[j]);
            most = std::max(most, std::max(l & 0x7FFFFFFFu, u & 0x7FFFFFFFu));
            mine[j] = upper ? u : l;
        }
    } else {
        const uint16_t* const k = static_cast<const uint16_t*>(a.k) + first;
        uint4 x[BT / 4];
#pragma unroll
        for (int i = 0; i < BT / 4; ++i)
            x[i] = *reinterpret_cast<const uint4*>(k + std::min(4 * i + t, left - 1) * a.k_st + 8 * c);
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = 0x7FFF7FFFu, hi[j] = 0x80008000u;
#pragma unroll
        for (int i = 0; i < BT / 4; ++i) {
            const uint32_t w[4] = {ordered(x[i].x), ordered(x[i].y), ordered(x[i].z), ordered(x[i].w)};
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = min2(lo[j], w[j]), hi[j] = max2(hi[j], w[j]);
        }
        auto fp32 = [](uint32_t half) {
            if constexpr (TYPE == 2) return __float_as_uint(tq::f16_to_f32(half)); else return half << 16;
        };
        uint32_t largest = 0u;  // of two at a time
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int d = 16; d < 64; d <<= 1)
                lo[j] = min2(lo[j], (uint32_t)__shfl_xor((int)lo[j], d)), hi[j] = max2(hi[j], (uint32_t)__shfl_xor((int)hi[j], d));
            lo[j] = ordered(lo[j]), hi[j] = ordered(hi[j]);  // its own inverse
            largest = max2(largest, max2(lo[j] & 0x7FFF7FFFu, hi[j] & 0x7FFF7FFFu));
            const uint32_t w = upper ? hi[j] : lo[j];
            mine[2 * j] = fp32(w & 0xFFFFu), mine[2 * j + 1] = fp32(w >> 16);
        }
        most = fp32(std::max(largest & 0xFFFFu, largest >> 16));
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) most = std::max(most, (uint32_t)__shfl_xor((int)most, d));
    const int e = step_exponent(most);
    const uint2 out = outward8(mine, upper, power_of_two(-e));
    const int64_t to = group * a.cap + a.first + block;
    if (t < 2) *reinterpret_cast<uint2*>(a.lohi + to * (2 * D) + t * D + 8 * c) = out;
    if (lane == 0) a.step[to] = power_of_two(e);
}

// ------------------------------------------------------------------ selection

struct SelectArgs {
    const void* q;
    int q_type, q_heads, kv_heads, group;
    int64_t q_sb, q_sh;
    const int8_t* lohi;
    const float* step;
    int64_t cap, n_blocks, n_tokens;
    const int32_t *starts, *lens;
    int keep, sink, recent;
    int32_t* out;
};

constexpr int ST = 512, SW = ST / 64;  // threads and waves of a workgroup
constexpr int TILE = 16;               // blocks of a matrix instruction
constexpr int AHEAD = 4;               // tiles of a wave whose bounds are on their way together: all that it has of 512 blocks
constexpr uint32_t ALWAYS = 0xFFFFFFFFu;

// The blocks of a row's range: [lo, lo + n).
struct BlockRange {
    int lo, n;
};
__device__ __forceinline__ BlockRange range_of(const SelectArgs& a, int b) {
    const int64_t len = a.lens ? std::min(std::max<int64_t>(a.lens[b], 0), a.n_tokens) : a.n_tokens;
    const int64_t start = a.starts ? std::min(std::max<int64_t>(a.starts[b], 0), len) : 0;
    const int lo = (int)(start / BT);
    return {lo, len > start ? (int)((len + BT - 1) / BT) - lo : 0};
}

// fp32 as an integer whose order is its
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b & 0x80000000u ? 0xFFFFFFFFu : 0x80000000u);
}

// Four elements of a query row as fp32.
__device__ __forceinline__ void load_query4(const SelectArgs& a, int64_t at, float* x) {
    if (a.q_type == 1) {
        __builtin_memcpy(x, static_cast<const float*>(a.q) + at, 16);
        return;
    }
    uint32_t w[2];
    __builtin_memcpy(w, static_cast<const uint16_t*>(a.q) + at, 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[2 * i] = a.q_type == 2 ? tq::f16_to_f32(w[i] & 0xFFFFu) : tq::bf16_to_f32(w[i] & 0xFFFFu);
        x[2 * i + 1] = a.q_type == 2 ? tq::f16_to_f32(w[i] >> 16) : tq::bf16_to_f32(w[i] >> 16);
    }
}
// The largest of their absolute values, as bits; NaN counts as 0.
__device__ __forceinline__ uint32_t largest4(const float* v) {
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        most = std::max(most, bits > 0x7F800000u ? 0u : bits);
    }
    return most;
}

// Scores of the blocks [TILE t, TILE t + TILE) below `known` of a range, for the tiles t0 <= t < tiles, by a workgroup: keys[j] of block j, in
// the order of the scores.  Ends with a barrier.
__device__ __forceinline__ void score_blocks(const SelectArgs& a, int b, int kvh, int lo, int known, int t0, int tiles, uint32_t* keys) {
    __shared__ uint32_t s_most[SW];
    // heads in whole numbers, their negative and their positive parts: 16-byte pieces, swizzled by the head
    __shared__ __align__(16) uint32_t s_q[2][16][D / 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // ---- the queries are asked for, then the first tiles' bounds.  A thread has four dims of one of 16 heads; heads past the last are
    // earlier ones again, which does not change a maximum
    const int64_t q0 = b * a.q_sb + (int64_t)kvh * a.group * a.q_sh;
    const int head = threadIdx.x >> 5, dim = 4 * (threadIdx.x & 31), head_tiles = (a.group + 15) / 16;
    static_assert(ST == 16 * 32, "a thread has four dims of one of 16 heads");
    float x[4];
    auto load_head = [&](int h, float* v) { load_query4(a, q0 + h % a.group * a.q_sh + dim, v); };
    load_head(head, x);

    // bounds: lane (block r of the tile, g) has bytes 64 i + 16 g + (0..15) of its 256, i = 0..3
    const int r = lane & 15, g = lane >> 4;
    const int64_t base = ((int64_t)b * a.kv_heads + kvh) * a.cap + lo;
    i32x4 w[AHEAD][4];
    float step[AHEAD];
    auto load = [&](int tile, int slot) {
        const int64_t at = base + std::min(tile * TILE + r, known - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[slot][i] = *reinterpret_cast<const i32x4*>(a.lohi + at * (2 * D) + 64 * i + 16 * g);
        step[slot] = a.step[at];
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (t0 + wave + i * SW < tiles) load(t0 + wave + i * SW, i);

    // ---- the heads' common step
    uint32_t most = largest4(x);
    for (int h = 16; h < a.group; h += 16) {
        float y[4];
        load_head(h + head, y);
        most = std::max(most, largest4(y));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = std::max(most, (uint32_t)__shfl_xor((int)most, d));
    if (lane == 0) s_most[wave] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SW; ++i) most = std::max(most, s_most[i]);
    const float down = power_of_two(-step_exponent(most));

    for (int ht = 0; ht < head_tiles; ++ht) {
        if (ht) {
            load_head(16 * ht + head, x);
            __syncthreads();
        }
        uint32_t neg = 0u, pos = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = x[e] == x[e] ? x[e] : 0.0f;
            const int z = (int)fminf(fmaxf(__builtin_rintf(y * down), -127.0f), 127.0f);
            neg |= ((uint32_t)std::min(z, 0) & 0xFFu) << (8 * e), pos |= (uint32_t)std::max(z, 0) << (8 * e);
        }
        const int at = (((dim >> 4) ^ (head & 7)) << 2) + (dim >> 2 & 3);
        s_q[0][head][at] = neg, s_q[1][head][at] = pos;
        __syncthreads();
        // lane (head r, g): dims 64 i + 16 g + (0..15), i = 0, 1
        i32x4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const i32x4*>(&s_q[i >> 1][r][((4 * (i & 1) + g) ^ (r & 7)) << 2]);
        for (int t = t0 + wave; t < tiles; t += AHEAD * SW) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int tile = t + i * SW, next = tile + AHEAD * SW;
                if (tile < tiles) {
                    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(q[k], w[i][k], acc, 0, 0, 0);
                    int u = std::max(std::max(acc[0], acc[1]), std::max(acc[2], acc[3]));
                    u = std::max(u, __shfl_xor(u, 16));
                    u = std::max(u, __shfl_xor(u, 32));
                    const int j = tile * TILE + r;
                    if (g == 0 && j < known) {
                        const uint32_t key = order_of((float)u * step[i]);
                        keys[j] = ht ? std::max(keys[j], key) : key;
                    }
                }
                // the next tiles, and the first ones again for the next heads
                if (next < tiles) load(next, i);
                else if (ht + 1 < head_tiles && t0 + wave + i * SW < tiles) load(t0 + wave + i * SW, i);
            }
        }
    }
    __syncthreads();
}
__device__ __forceinline__ int tiles_of(int known) { return known > 0 ? (known + TILE - 1) / TILE : 0; }

// `per` tiles of a KV head's range to a workgroup, into keys [KV head of the batch][most].
__global__ __launch_bounds__(ST) void score_kernel(SelectArgs a, uint32_t* keys, int most, int per) {
    const int group = blockIdx.y, b = group / a.kv_heads, kvh = group - b * a.kv_heads;
    const BlockRange range = range_of(a, b);
    const int known = (int)std::min<int64_t>(a.n_blocks - range.lo, range.n), tiles = tiles_of(known), t0 = blockIdx.x * per;
    if (range.n <= a.keep || t0 >= tiles) return;
    score_blocks(a, b, kvh, range.lo, known, t0, std::min(t0 + per, tiles), keys + (int64_t)group * most);
}

// A KV head's choice.  FUSED: its scores too; else they are in `keys`.
template <bool FUSED>
__global__ __launch_bounds__(ST) void select_kernel(SelectArgs a, const uint32_t* keys, int most) {
    extern __shared__ uint32_t s_key[];  // a block's score, by its number in the range
    __shared__ __align__(16) uint32_t s_hist[4][256];
    __shared__ int2 s_wave[SW];
    __shared__ uint2 s_bits[SW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.kv_heads, kvh = blockIdx.x - b * a.kv_heads;
    const BlockRange range = range_of(a, b);
    const int lo = range.lo, n = range.n, known = (int)std::min<int64_t>(a.n_blocks - lo, n);
    int32_t* const out = a.out + (int64_t)blockIdx.x * a.keep;
    if (n <= a.keep) {  // all of them
        for (int i = threadIdx.x; i < a.keep; i += ST) out[i] = i < n ? lo + i : -1;
        return;
    }
    for (int i = threadIdx.x; i < 4 * 256; i += ST) (&s_hist[0][0])[i] = 0u;
    if (FUSED) score_blocks(a, b, kvh, lo, known, 0, tiles_of(known), s_key);

    // ---- in between the first and the last blocks, which are always chosen, the choice is by score; blocks without come last.  What the
    // keys there have in common needs no looking at
    const int first = a.sink, last = n - a.recent;
    uint32_t all = 0xFFFFFFFFu, any = 0u;
    for (int j = threadIdx.x; j < n; j += ST) {
        uint32_t key = 0u;
        if (j < known) key = FUSED ? s_key[j] : keys[(int64_t)blockIdx.x * most + j];
        if (j < first || j >= last) key = ALWAYS;
        else all &= key, any |= key;
        s_key[j] = key;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all &= (uint32_t)__shfl_xor((int)all, d), any |= (uint32_t)__shfl_xor((int)any, d);
    if (lane == 0) s_bits[wave] = make_uint2(all, any);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SW; ++i) all &= s_bits[i].x, any |= s_bits[i].y;
    int rest = a.keep - (n - (last - first));  // of the keys that share the bits found, the `rest` largest are chosen
    int shift = 32 - __builtin_clz((all ^ any) | 1u);  // from the highest bit in which two differ, eight at a time
    uint32_t mask = shift < 32 ? ~0u << shift : 0u, found = all & mask;
    if (rest > 0) {
#pragma unroll 1
        for (int pass = 0; shift > 0; ++pass) {
            const int width = std::min(shift, 8);
            shift -= width;
            uint32_t* const hist = s_hist[pass];
            const uint32_t digits = (1u << width) - 1;
            for (int i = first + threadIdx.x; i < last; i += ST) {
                const uint32_t key = s_key[i];
                if ((key & mask) == found) atomicAdd(&hist[(key >> shift) & digits], 1u);
            }
            __syncthreads();
            // every wave for itself; lane l: the four digits from 252 - 4 l on
            const uint4 c4 = *reinterpret_cast<const uint4*>(&hist[252 - 4 * lane]);
            const int c[4] = {(int)c4.w, (int)c4.z, (int)c4.y, (int)c4.x}, sum = c[0] + c[1] + c[2] + c[3];
            int up = sum;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(up, d);
                if (lane >= d) up += y;
            }
            int above = up - sum, digit = -1, larger = 0, with = 0;  // keys with larger digits, and with this one
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < rest && above + c[i] >= rest) digit = 255 - 4 * lane - i, larger = above, with = c[i];
                above += c[i];
            }
            const int who = __builtin_ctzll(__ballot(digit >= 0));  // one lane has it: there are `rest` keys at least
            found |= (uint32_t)__builtin_amdgcn_readlane(digit, who) << shift, mask |= digits << shift;
            rest -= __builtin_amdgcn_readlane(larger, who);
            if (__builtin_amdgcn_readlane(with, who) == rest) break;  // all of them
        }
    } else {
        mask = found = 0xFFFFFFFFu;  // none
    }

    // ---- what is above it, and the first `rest` of those equal to it, in order
    int before = 0, equal = 0;  // so far
    for (int i0 = 0; i0 < n; i0 += ST) {
        const int i = i0 + threadIdx.x;
        const bool always = i < first || i >= last;
        const uint32_t key = i < n ? s_key[i] & mask : 0u;
        const bool is_above = i < n && (always || key > found), is_equal = i < n && !always && key == found;
        const uint64_t above = __ballot(is_above), same = __ballot(is_equal), below = (1ull << lane) - 1;
        if (i0) __syncthreads();
        if (lane == 0) s_wave[wave] = make_int2(__popcll(above), __popcll(same));
        __syncthreads();
        int a0 = before, e0 = equal;
#pragma unroll
        for (int v = 0; v < SW; ++v) {
            const int2 c = s_wave[v];
            if (v < wave) a0 += c.x, e0 += c.y;
            before += c.x, equal += c.y;
        }
        a0 += __popcll(above & below), e0 += __popcll(same & below);
        if (is_above || (is_equal && e0 < rest)) out[a0 + std::min(e0, std::max(rest, 0))] = lo + i;
    }
}

// One workgroup for a KV head's whole choice up to here, else its scores in a launch of their own, spread over the CUs: a workgroup alone takes
// its bounds at about 36 GB/s, but a launch more is 4 us of the host.  In graphs, us, in one and in two launches: 128 blocks 6.5 and 8.0, 256
// 7.4 and 8.1, 512 9.7 and 8.5 (from the host 13.4 and 17; for 256 KV heads 12.5 and 14.8), 1024 14.5 and 9.3, 2048 22.7 and 11.3.
constexpr int FUSED_BLOCKS = 512;

}  // namespace

extern "C" int tq_block_bounds_typed(const void* k, int k_type, int batch, int heads, int64_t tokens, int dim, int64_t k_sb, int64_t k_sh,
                                     int64_t k_st, int8_t* lohi, float* step, int64_t cap, int64_t first, void* stream) {
    if (!k || k_type < 0 || k_type > 2 || !lohi || !step || batch < 1 || heads < 1 || tokens < 1 || first < 0) return TQ_ERR_INVALID_ARGUMENT;
    const int64_t per_head = (tokens - 1) / BT + 1;
    if (first > cap - per_head) return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D || !aligned16(k) || !aligned16(lohi) || ((k_sb | k_sh | k_st) & (k_type == 1 ? 3 : 7))) return TQ_ERR_UNSUPPORTED;
    const int64_t groups = (int64_t)batch * heads;
    if (per_head >= (int64_t)1 << 31 || groups * per_head >= (int64_t)1 << 31) return TQ_ERR_UNSUPPORTED;
    const BoundsArgs a{k, heads, tokens, k_sb, k_sh, k_st, lohi, step, cap, first, per_head, groups * per_head, k_sh < k_st};
    const dim3 grid((unsigned)((a.all + BOUNDS_WAVES - 1) / BOUNDS_WAVES)), threads(64 * BOUNDS_WAVES);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (k_type == 0) hipLaunchKernelGGL(bounds_kernel<0>, grid, threads, 0, s, a);
    else if (k_type == 1) hipLaunchKernelGGL(bounds_kernel<1>, grid, threads, 0, s, a);
    else hipLaunchKernelGGL(bounds_kernel<2>, grid, threads, 0, s, a);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}

extern "C" int tq_block_bounds(const uint16_t* k, int batch, int heads, int64_t tokens, int dim, int64_t k_sb, int64_t k_sh,
                               int64_t k_st, int8_t* lohi, float* step, int64_t cap, int64_t first, void* stream) {
    return tq_block_bounds_typed(k, 0, batch, heads, tokens, dim, k_sb, k_sh, k_st, lohi, step, cap, first, stream);
}

extern "C" size_t tq_select_blocks_workspace_bytes(int batch, int kv_heads, int64_t n_tokens) {
    if (batch < 1 || kv_heads < 1 || n_tokens < 0 || n_tokens > (int64_t)TQ_MAX_SCORED * BT) return 0;
    const int64_t most = (n_tokens + BT - 1) / BT;
    return most <= FUSED_BLOCKS ? 0 : (size_t)batch * kv_heads * most * 4;
}

extern "C" int tq_select_blocks(const void* q, int q_type, int batch, int q_heads, int kv_heads, int dim, int64_t q_sb, int64_t q_sh,
                                const int8_t* lohi, const float* step, int64_t cap, int64_t n_blocks, int64_t n_tokens,
                                const int32_t* seq_starts, const int32_t* seq_lens, int keep, int sink, int recent, int32_t* out,
                                void* workspace, size_t workspace_bytes, void* stream) {
    if (!q || q_type < 0 || q_type > 2 || batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || n_blocks < 0 ||
        n_blocks > cap || n_tokens < 0 || (n_blocks > 0 && (!lohi || !step)) || keep < 1 || sink < 0 || recent < 0 || sink > keep ||
        recent > keep - sink || !out)
        return TQ_ERR_INVALID_ARGUMENT;
    const int64_t groups = (int64_t)batch * kv_heads;
    if (dim != D || keep > TQ_MAX_BLOCKS || n_tokens > (int64_t)TQ_MAX_SCORED * BT || (lohi && !aligned16(lohi)) ||
        groups >= (int64_t)1 << 31)
        return TQ_ERR_UNSUPPORTED;
    const size_t need = tq_select_blocks_workspace_bytes(batch, kv_heads, n_tokens);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return TQ_ERR_WORKSPACE;
    const SelectArgs a{q, q_type, q_heads, kv_heads, q_heads / kv_heads, q_sb, q_sh, lohi, step, cap, n_blocks, n_tokens,
                       seq_starts, seq_lens, keep, sink, recent, out};
    const int most = (int)((n_tokens + BT - 1) / BT);  // blocks of a range
    const size_t lds = (size_t)std::max(most, 1) * 4;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (!need) {
        hipLaunchKernelGGL(select_kernel<true>, dim3((unsigned)groups), dim3(ST), lds, s, a, nullptr, most);
        TQ_CHECK_LAUNCH();
        return TQ_OK;
    }
    if (groups > 65535) return TQ_ERR_UNSUPPORTED;
    uint32_t* const keys = static_cast<uint32_t*>(workspace);
    const int64_t tiles = (most + TILE - 1) / TILE;
    const int per = (int)((tiles * groups + 256 * SW - 1) / (256 * SW) * SW);
    hipLaunchKernelGGL(score_kernel, dim3((unsigned)((tiles + per - 1) / per), (unsigned)groups), dim3(ST), 0, s, a, keys, most, per);
    TQ_CHECK_LAUNCH();
    hipLaunchKernelGGL(select_kernel<false>, dim3((unsigned)groups), dim3(ST), lds, s, a, keys, most);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
