// tq_blocks.hip -- bounds of the keys of every 64 tokens, and the blocks that a query chooses by them (gfx950).
//
// A block's keys lie between lo and hi, channel by channel, so no key of it gives the query q a larger product than
//   sum_d max(q_d lo_d, q_d hi_d).
// lo and hi are whole numbers of a step of the block's own, rounded outward to 8 bits, and q is rounded to whole numbers too: the sum is
// a whole number below 2^22, the step a power of two, and so every score is exact in fp32, whatever the order of its sum.  The same
// blocks are chosen everywhere, and a block's bounds are the same however its keys arrived.
//
//   bounds_kernel  a block per wave, 16 bytes of four keys a lane and load, all of a block's loads in flight together
//   select_kernel  a KV head's whole choice per workgroup: scores by v_mfma_i32_16x16x64_i8, a column for a block, then the keep-th
//                  largest by radix and the chosen numbers in order

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

struct BoundsArgs {
    const uint16_t* k;
    int heads;
    int64_t tokens, k_sb, k_sh, k_st;
    int8_t* lohi;
    float* step;
    int64_t cap, first, per_head, all;  // blocks to a head, and of all heads
};

constexpr int BOUNDS_WAVES = 4;
__global__ __launch_bounds__(64 * BOUNDS_WAVES) void bounds_kernel(BoundsArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = (int64_t)blockIdx.x * BOUNDS_WAVES + wave;
    if (at >= a.all) return;
    const int64_t group = at / a.per_head, block = at - group * a.per_head, b = group / a.heads, h = group - b * a.heads;
    const uint16_t* const k = a.k + b * a.k_sb + h * a.k_sh + block * BT * a.k_st;
    const int left = (int)std::min<int64_t>(a.tokens - block * BT, BT);
    // lane (c = lane % 16, t = lane / 16): channels [8 c, 8 c + 8) of the tokens t, t + 4, ...; past the last it again
    const int c = lane & 15, t = lane >> 4;
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
    uint32_t most = 0u;  // the largest absolute value, as fp32 bits
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int d = 16; d < 64; d <<= 1)
            lo[j] = min2(lo[j], (uint32_t)__shfl_xor((int)lo[j], d)), hi[j] = max2(hi[j], (uint32_t)__shfl_xor((int)hi[j], d));
        lo[j] = ordered(lo[j]), hi[j] = ordered(hi[j]);  // its own inverse
        const uint32_t l = lo[j] & 0x7FFF7FFFu, u = hi[j] & 0x7FFF7FFFu;
        most = std::max(most, std::max(std::max(l << 16, l & 0x7FFF0000u), std::max(u << 16, u & 0x7FFF0000u)));
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) most = std::max(most, (uint32_t)__shfl_xor((int)most, d));
    const int e = step_exponent(most);
    const float down = power_of_two(-e);
    // lanes t = 0 write lo, t = 1 hi
    const bool upper = t == 1;
    uint32_t out[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t w = upper ? hi[j >> 1] : lo[j >> 1], bits = j & 1 ? w & 0xFFFF0000u : w << 16;
        // an infinity for NaN too
        const float v = __uint_as_float((bits & 0x80000000u) | std::min(bits & 0x7FFFFFFFu, 0x7F800000u)) * down;
        const float r = fminf(fmaxf(upper ? __builtin_ceilf(v) : __builtin_floorf(v), -127.0f), 127.0f);
        out[j >> 2] |= ((uint32_t)(int)r & 0xFFu) << (8 * (j & 3));
    }
    const int64_t to = group * a.cap + a.first + block;
    if (t < 2) *reinterpret_cast<uint2*>(a.lohi + to * (2 * D) + t * D + 8 * c) = make_uint2(out[0], out[1]);
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

constexpr int ST = 1024, SW = ST / 64;  // threads and waves of a workgroup
constexpr int TILE = 16;                // blocks of a matrix instruction
constexpr uint32_t ALWAYS = 0xFFFFFFFFu;

// fp32 as an integer whose order is its
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (b & 0x80000000u ? 0xFFFFFFFFu : 0x80000000u);
}

// Eight elements of a query row as fp32.
__device__ __forceinline__ void load_query8(const SelectArgs& a, int64_t at, float* x) {
    if (a.q_type == 1) {
        __builtin_memcpy(x, static_cast<const float*>(a.q) + at, 32);
        return;
    }
    uint32_t w[4];
    __builtin_memcpy(w, static_cast<const uint16_t*>(a.q) + at, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = a.q_type == 2 ? tq::f16_to_f32(w[i] & 0xFFFFu) : tq::bf16_to_f32(w[i] & 0xFFFFu);
        x[2 * i + 1] = a.q_type == 2 ? tq::f16_to_f32(w[i] >> 16) : tq::bf16_to_f32(w[i] >> 16);
    }
}

__global__ __launch_bounds__(ST) void select_kernel(SelectArgs a) {
    extern __shared__ uint32_t s_key[];  // a block's score, by its number in the range
    __shared__ uint32_t s_hist[256];
    __shared__ int s_digit, s_above;
    __shared__ int2 s_wave[SW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.x / a.kv_heads, kvh = blockIdx.x - b * a.kv_heads;
    const int64_t len = a.lens ? std::min(std::max<int64_t>(a.lens[b], 0), a.n_tokens) : a.n_tokens;
    const int64_t start = a.starts ? std::min(std::max<int64_t>(a.starts[b], 0), len) : 0;
    const int lo = (int)(start / BT), n = len > start ? (int)((len + BT - 1) / BT) - lo : 0;  // the range's blocks
    int32_t* const out = a.out + (int64_t)blockIdx.x * a.keep;
    if (n <= a.keep) {  // all of them
        for (int i = threadIdx.x; i < a.keep; i += ST) out[i] = i < n ? lo + i : -1;
        return;
    }

    // ---- the queries: lane (r = lane % 16, g = lane / 16) has head r's dims 64 i + 16 g + (0..15), i = 0, 1, as its A operands; heads
    // past the last are earlier ones again, which does not change a maximum
    const int r = lane & 15, g = lane >> 4;
    const int64_t q0 = b * a.q_sb + (int64_t)kvh * a.group * a.q_sh + 16 * g;
    auto load = [&](int h, float* x) {
        const int64_t at = q0 + (h % a.group) * a.q_sh;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_query8(a, at + 64 * (i >> 1) + 8 * (i & 1), x + 8 * i);
    };
    const int head_tiles = (a.group + 15) / 16;
    uint32_t most = 0u;
    float x[32];
    for (int ht = head_tiles - 1; ht >= 0; --ht) {
        load(16 * ht + r, x);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t bits = __float_as_uint(x[i]) & 0x7FFFFFFFu;
            most = std::max(most, bits > 0x7F800000u ? 0u : bits);  // NaN counts as 0
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = std::max(most, (uint32_t)__shfl_xor((int)most, d));
    const float down = power_of_two(-step_exponent(most));
    i32x4 neg[2], pos[2];
    auto operands = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t n4 = 0u, p4 = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = x[16 * i + 4 * w + e], y = v == v ? v : 0.0f;
                    const int z = (int)fminf(fmaxf(__builtin_rintf(y * down), -127.0f), 127.0f);
                    n4 |= ((uint32_t)std::min(z, 0) & 0xFFu) << (8 * e), p4 |= (uint32_t)std::max(z, 0) << (8 * e);
                }
                neg[i][w] = (int)n4, pos[i][w] = (int)p4;
            }
    };
    operands();  // of the first 16 heads

    // ---- scores: lane (block r of the tile, g) has bytes 64 i + 16 g + (0..15) of its 256
    const int first = a.sink, last = n - a.recent;  // in between the choice is by score
    const int64_t base = (int64_t)blockIdx.x * a.cap + lo;
    for (int ht = 0; ht < head_tiles; ++ht) {
        if (ht) load(16 * ht + r, x), operands();
        for (int t0 = wave * TILE; t0 < n; t0 += SW * TILE) {
            const int j = t0 + r, known = std::min(j, (int)std::min<int64_t>(a.n_blocks - 1 - lo, n - 1));
            uint32_t key = 0u;
            if (known >= 0) {
                const int8_t* const p = a.lohi + (base + known) * (2 * D) + 16 * g;
                i32x4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const i32x4*>(p + 64 * i);
                const float step = a.step[base + known];
                i32x4 acc = {0, 0, 0, 0};
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(neg[0], w[0], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(neg[1], w[1], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(pos[0], w[2], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(pos[1], w[3], acc, 0, 0, 0);
                int u = std::max(std::max(acc[0], acc[1]), std::max(acc[2], acc[3]));
                u = std::max(u, __shfl_xor(u, 16));
                u = std::max(u, __shfl_xor(u, 32));
                key = known == j ? order_of((float)u * step) : 0u;
            }
            if (j < first || j >= last) key = ALWAYS;
            if (g == 0 && j < n) s_key[j] = ht ? std::max(s_key[j], key) : key;
        }
    }
    __syncthreads();

    // ---- the keep-th largest, eight bits at a time
    uint32_t found = 0u, mask = 0u;
    int rest = a.keep;  // of the keys that share the bits found, the `rest` largest are chosen
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) s_hist[threadIdx.x] = 0u;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += ST) {
            const uint32_t key = s_key[i];
            if ((key & mask) == found) atomicAdd(&s_hist[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {  // lane l: the four digits from 252 - 4 l on
            uint32_t c[4], sum = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = s_hist[255 - 4 * lane - i], sum += c[i];
            uint32_t up = sum;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = (uint32_t)__shfl_up((int)up, d);
                if (lane >= d) up += y;
            }
            int above = (int)(up - sum);  // keys with larger digits
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < rest && above + (int)c[i] >= rest) s_digit = 255 - 4 * lane - i, s_above = above;
                above += (int)c[i];
            }
        }
        __syncthreads();
        found |= (uint32_t)s_digit << shift, mask |= 255u << shift, rest -= s_above;
    }

    // ---- what is above it, and the first `rest` of those equal to it, in order
    int before = 0, equal = 0;  // so far
    for (int i0 = 0; i0 < n; i0 += ST) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < n ? s_key[i] : 0u;
        const bool is_above = i < n && key > found, is_equal = i < n && key == found;
        const uint64_t above = __ballot(is_above), same = __ballot(is_equal), below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) s_wave[wave] = make_int2(__popcll(above), __popcll(same));
        __syncthreads();
        int a0 = before, e0 = equal;
#pragma unroll
        for (int w = 0; w < SW; ++w) {
            const int2 c = s_wave[w];
            if (w < wave) a0 += c.x, e0 += c.y;
            before += c.x, equal += c.y;
        }
        a0 += __popcll(above & below), e0 += __popcll(same & below);
        if (is_above || (is_equal && e0 < rest)) out[a0 + std::min(e0, rest)] = lo + i;
    }
}

}  // namespace

extern "C" int tq_block_bounds(const uint16_t* k, int batch, int heads, int64_t tokens, int dim, int64_t k_sb, int64_t k_sh,
                               int64_t k_st, int8_t* lohi, float* step, int64_t cap, int64_t first, void* stream) {
    if (!k || !lohi || !step || batch < 1 || heads < 1 || tokens < 1 || first < 0) return TQ_ERR_INVALID_ARGUMENT;
    const int64_t per_head = (tokens - 1) / BT + 1;
    if (first > cap - per_head) return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D || !aligned16(k) || !aligned16(lohi) || ((k_sb | k_sh | k_st) & 7)) return TQ_ERR_UNSUPPORTED;
    const int64_t groups = (int64_t)batch * heads;
    if (per_head >= (int64_t)1 << 31 || groups * per_head >= (int64_t)1 << 31) return TQ_ERR_UNSUPPORTED;
    const BoundsArgs a{k, heads, tokens, k_sb, k_sh, k_st, lohi, step, cap, first, per_head, groups * per_head};
    hipLaunchKernelGGL(bounds_kernel, dim3((unsigned)((a.all + BOUNDS_WAVES - 1) / BOUNDS_WAVES)), dim3(64 * BOUNDS_WAVES), 0,
                       static_cast<hipStream_t>(stream), a);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}

extern "C" int tq_select_blocks(const void* q, int q_type, int batch, int q_heads, int kv_heads, int dim, int64_t q_sb, int64_t q_sh,
                                const int8_t* lohi, const float* step, int64_t cap, int64_t n_blocks, int64_t n_tokens,
                                const int32_t* seq_starts, const int32_t* seq_lens, int keep, int sink, int recent, int32_t* out,
                                void* stream) {
    if (!q || q_type < 0 || q_type > 2 || batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || n_blocks < 0 ||
        n_blocks > cap || n_tokens < 0 || (n_blocks > 0 && (!lohi || !step)) || keep < 1 || sink < 0 || recent < 0 || sink > keep ||
        recent > keep - sink || !out)
        return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D || keep > TQ_MAX_BLOCKS || n_tokens > (int64_t)TQ_MAX_SCORED * BT || (lohi && !aligned16(lohi)) ||
        (int64_t)batch * kv_heads >= (int64_t)1 << 31)
        return TQ_ERR_UNSUPPORTED;
    const SelectArgs a{q, q_type, q_heads, kv_heads, q_heads / kv_heads, q_sb, q_sh, lohi, step, cap, n_blocks, n_tokens,
                       seq_starts, seq_lens, keep, sink, recent, out};
    const int64_t most = (n_tokens + BT - 1) / BT;  // blocks of a range
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)(batch * kv_heads)), dim3(ST), (size_t)std::max<int64_t>(most, 1) * 4,
                       static_cast<hipStream_t>(stream), a);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
