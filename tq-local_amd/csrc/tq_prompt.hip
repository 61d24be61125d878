// tq_prompt.hip -- causal attention over whole prompts for gfx950: grouped query heads, padded batches,
// and prompts of different lengths packed behind one another.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = 2^(c q_i . k_j - m_i),   c = scale log2(e)
//
// j over the sequence of row i.  One pass over the keys with a running reference m_i of each row.
//
// Layout.  A workgroup of eight waves owns 256 consecutive rows of one sequence and query head (KS = 1), or 128 (KS = 2),
// a wave 32 of them, and the waves walk the keys in tiles of 64 tokens.
//   S^T = K Q^T   v_mfma_f32_32x32x16, A = 32 tokens x 16 dims, B = 16 dims x 32 rows: lane (r = l % 32,
//                 h = l / 32) ends with row r's scores of the tokens 8 j + 4 h + (0..3) of a block of 32
//   O^T = V^T P^T A = 32 dims x 16 tokens, B = 16 tokens x 32 rows.  The order of the 16 tokens along k
//                 is free: it is the order the scores come back in, so a lane's weights become its B
//                 operand as they are, and ds_read_b64_tr_b16 takes V^T out of row-major rows in that
//                 order (16 lanes read 4 tokens x 16 dims and each ends with one dim's 4 tokens).
// K and V go from memory to LDS without passing registers (16 bytes a lane), double-buffered, their chunks swizzled by the token.
//
// Cost.  Bound by the matrix pipe and the softmax beside it: a tile of 64 tokens and 32 rows is 32 products of 32 cycles
// and about 430 cycles of exponentials, maxima, sums and roundings, on a SIMD that holds two waves.  The waves' halves therefore
// take turns (below).  1 x 32/8 heads of 8192 tokens take 480 to 525 us by the clock of the card = 1145 to 1050 TFLOP/s of
// counted work, where a large product of matrices reaches 1326, and 16384 tokens 1.88 to 1.99 ms = 1170 to 1105; four waves that each do one thing
// after the other took 662 us when these took 584, and eight without the operands read ahead 595 when they took 544 with
// them.  The clock gives way under this load (1.6 to 1.9 GHz of 2.4), so cycles won come back in part only.  64 rows to a wave
// (512 registers) took longer: its sums move between the two register files.  Short sequences are bound by a block's
// start and end, 4 to 5 us of loads and stores that nothing hides: eight packed prompts of 1 to 2811 tokens take 105 us,
// of which 59 are the products, one of 2048 tokens 49, of which 26.  The smallest calls are bound by latency, 13 us at 300 tokens.
//
// Rounding.  Scores, weights, sums and outputs are fp32; the weights are rounded to the values' type for
// their product, once and to nearest: off by at most half a step (relative 2^-8 in bf16, 2^-11 in fp16), as much as the
// output's own rounding, and independently from weight to weight.  Fp16 weights below 2^-25 of their row's reference, which
// is one of its larger scores, are off by up to 2^-36 of it instead: 16384 of them by 2^-22 of their values, where an fp16 output
// of that size has steps of 2^-24 and more.  The sum of a row's weights is of the unrounded ones.

#include <algorithm>
#include <type_traits>

#include "tq_rows16.h"

namespace {

using namespace tqr;

constexpr int D = TQ_DIM;
constexpr int TK = 64;  // tokens per tile
constexpr float LOG2E = 1.44269504f;
// A score may exceed its row's reference by LAZY (log2), and weights are in units of 2^-LIFT.  Fp16 weights reach up to 2^15 and
// keep their 11 bits down to 2^-25 of the reference's; references that rise more often for it cost nothing with logits of a
// standard deviation of 1 (1 x 32/8 heads of 8192 tokens take 525 us, and 527 with a LAZY of 8), and 2% with one of 4 (554, 542).  A
// LAZY of 2 takes 532 and 564
template <bool F16>
constexpr float LAZY = F16 ? 4.0f : 8.0f;
template <bool F16>
constexpr float LIFT = F16 ? 15.0f - LAZY<F16> : 0.0f;

#define INLINE __attribute__((always_inline))
constexpr int MFMA = 0x8, DS_READ = 0x100;  // kinds of instructions for the scheduler
constexpr int AHEAD = 4;                    // products whose operands are on their way

template <bool F16>
__device__ __forceinline__ f32x16 mfma_32(const Frag& a, const Frag& b, f32x16 c) {
    if constexpr (F16) return mfma_f16(a, b, c);
    else return mfma_bf16(a, b, c);
}
// two fp32 values to the element type
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (F16) return pack_f16(a, b);
    else return pack_bf16(a, b);
}
// Byte offset in a tile of a lane's 16 bytes of key row r in step ks (plus 32 rows for the second block of tokens); values'
// in value_offset, plus 16 rows per step.
__device__ __forceinline__ int key_offset(int ks, int lane) {
    return (lane & 31) * 256 + (((2 * ks + (lane >> 5)) ^ swizzle(lane & 31)) << 4);
}
struct PromptArgs {
    const uint16_t *q, *k, *v;
    uint16_t* out;
    float* lse;
    int batch, q_heads, kv_heads, tokens;
    int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st;
    const int32_t* cu;  // packed sequences: n_seqs + 1 ascending offsets
    int n_seqs;
    const int32_t *starts, *ends;
    int zero_outside;
    float scale;
    int row_blocks;
};

// Rows [lo, hi) are the sequence that the block's rows [row0, row0 + BM) belong to; only those of [w_lo, w_hi)
// are the block's to write.
struct Block {
    int b, lo, hi, row0, w_lo, w_hi;
};

// Block `blk` of packed sequences: sequence by sequence, longest-running rows first, then the rows that
// belong to none (before the first offset, behind the last), which have no keys.
__device__ __forceinline__ Block find_packed(const PromptArgs& a, int blk, int BM) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const int i = base + lane;
        int lo = 0, hi = 0;
        if (i < a.n_seqs) {
            lo = std::max(a.cu[i], 0);
            hi = std::min(a.cu[i + 1], a.tokens);
        }
        const int n = hi > lo ? (hi - lo + BM - 1) / BM : 0;
        int sum = n;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const int t = __shfl_up(sum, k);
            if (lane >= k) sum += t;
        }
        const uint64_t hit = __ballot(before + sum > blk);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            lo = __shfl(lo, src), hi = __shfl(hi, src);
            const int j = blk - before - (__shfl(sum, src) - __shfl(n, src));
            const int row0 = lo + (__shfl(n, src) - 1 - j) * BM;
            return {0, lo, hi, row0, row0, std::min(row0 + BM, hi)};
        }
        before += __shfl(sum, 63);
    }
    int j = blk - before;  // rows outside
    const int head = std::min(std::max(a.cu[0], 0), a.tokens), head_blocks = (head + BM - 1) / BM;
    if (j < head_blocks) return {0, 0, 0, j * BM, j * BM, std::min(j * BM + BM, head)};
    const int64_t row0 = (int64_t)std::max(a.cu[a.n_seqs], 0) + (int64_t)(j - head_blocks) * BM;
    if (row0 >= a.tokens) return {0, 0, 0, a.tokens, a.tokens, a.tokens};
    return {0, 0, 0, (int)row0, (int)row0, (int)std::min<int64_t>(row0 + BM, a.tokens)};
}

// The wait of a wave for its own reads of LDS, and the barrier, with nothing moved across either.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight waves, two to a SIMD, in two halves of four.  KS = 1: 256 rows, 32 to a wave, and every wave walks all tiles.
// KS = 2: 128 rows, and the halves walk every other tile of the same rows, their sums meet at the end: half the steps where
// there are few blocks.
template <bool F16, int KS>
__global__ __launch_bounds__(512, 2) void prompt_kernel(PromptArgs a) {
    constexpr int T = 512, BM = 256 / KS;
    constexpr int TL = T / KS;           // threads that bring in a tile
    constexpr int CH = TK * 16 / TL;     // 16-byte chunks of K, and of V, each of them
    __shared__ uint4 s_k[KS][2][TK * 16];
    __shared__ uint4 s_v[KS][2][TK * 16];
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // in a scalar register, and what follows from it
    const bool second = wave >= 4;
    const int part = KS == 2 && second ? 1 : 0;
    // workgroups of one KV head share an XCD's L2 where their number divides by the eight XCDs.  Ragged batches move on by a
    // batch row with every head and block: an XCD hands its workgroups to its four groups of CUs in turn, and one long
    // row of 1500 tokens among four (40 heads), on one group of CUs all along, took 106 us, and 47 spread over them
    const int n_kv = (a.cu ? 1 : a.batch) * a.kv_heads, group = a.q_heads / a.kv_heads;
    const int item = blockIdx.x / n_kv;
    int kv = blockIdx.x % n_kv;
    if (a.starts || a.ends) kv = (int)((kv + (int64_t)item * a.kv_heads) % n_kv);
    const int kvh = kv % a.kv_heads, hq = kvh * group + item % group;
    int blk = item / group;
    Block w;
    if (a.cu) {
        w = find_packed(a, blk, BM);
        if (w.w_lo >= w.w_hi) return;
    } else {
        blk = a.row_blocks - 1 - blk;  // the longest first
        const int b = kv / a.kv_heads;
        const int lo = a.starts ? std::min(std::max(a.starts[b], 0), a.tokens) : 0;
        const int hi = a.ends ? std::min(std::max(a.ends[b], lo), a.tokens) : a.tokens;
        w = {b, lo, hi, blk * BM, blk * BM, (int)std::min<int64_t>((int64_t)blk * BM + BM, a.tokens)};
    }
    // the same in every lane
    w.lo = __builtin_amdgcn_readfirstlane(w.lo), w.hi = __builtin_amdgcn_readfirstlane(w.hi);
    w.row0 = __builtin_amdgcn_readfirstlane(w.row0), w.b = __builtin_amdgcn_readfirstlane(w.b);
    uint16_t* const ob = a.out + w.b * a.o_sb + hq * a.o_sh;
    const int64_t lse_row = ((int64_t)w.b * a.q_heads + hq) * a.tokens;
    if (w.lo >= w.hi || w.row0 >= w.hi || w.row0 + BM <= w.lo) {  // no row of a sequence
        if (w.hi > w.lo || !a.cu || a.zero_outside) {
            for (int i = threadIdx.x; i < (w.w_hi - w.w_lo) * 16; i += T)
                *reinterpret_cast<uint4*>(ob + (w.w_lo + (i >> 4)) * a.o_st + 8 * (i & 15)) = make_uint4(0, 0, 0, 0);
            if (a.lse)
                for (int i = w.w_lo + threadIdx.x; i < w.w_hi; i += T) a.lse[lse_row + i] = -__builtin_inff();
        }
        return;
    }

    const uint16_t* const kb = a.k + w.b * a.k_sb + kvh * a.k_sh;
    const uint16_t* const vb = a.v + w.b * a.v_sb + kvh * a.v_sh;
    const int k_end = (int)std::min<int64_t>(w.hi, (int64_t)w.row0 + BM);
    const int n = (k_end - w.lo + TK - 1) / TK, steps = (n + KS - 1) / KS, last = KS * steps;  // tiles, and each half's

    // ---- tiles to LDS; those of a half of KS = 2 are part, part + 2, ...
    // (a thread has a chunk of every TL / 16-th row, at the same place of its row: TL / 16 is a multiple of the swizzle's 16;
    // tokens past the last are copies of it, left out by the mask)
    const int tid = threadIdx.x % TL, lds_wave = KS == 2 ? wave & 3 : wave;
    const uint32_t in_row = 16 * ((tid & 15) ^ swizzle(tid >> 4));
    const uint32_t k_st2 = (uint32_t)a.k_st * 2, v_st2 = (uint32_t)a.v_st * 2, k_off = (tid >> 4) * k_st2, v_off = (tid >> 4) * v_st2;
    auto load = [&](const uint16_t* base, int64_t st, uint32_t st2, uint32_t off, int tile, uint4* dst) INLINE {
        if (tile >= last) return;
        const int t0 = std::min(w.lo + tile * TK, k_end - 1);
        const char* const rows = reinterpret_cast<const char*>(base + (int64_t)t0 * st);
        const uint32_t most = (uint32_t)std::min(k_end - 1 - t0, TK - 1) * st2;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            load_lds16(rows + (std::min(off + i * (TL / 16) * st2, most) + in_row), dst + i * TL + lds_wave * 64);
    };
    auto load_k = [&](int j) INLINE { load(kb, a.k_st, k_st2, k_off, KS * j + part, s_k[part][j & 1]); };
    auto load_v = [&](int j) INLINE { load(vb, a.v_st, v_st2, v_off, KS * j + part, s_v[part][j & 1]); };
    load_k(0);

    // ---- the wave's query rows: dims 16 s + 8 h + (0..7) of row r
    const int wrow = w.row0 + 32 * (KS == 2 ? wave & 3 : wave), row = wrow + r;
    const bool live = row >= w.lo && row < w.hi;
    Frag q[8];
    {
        const uint16_t* p = a.q + w.b * a.q_sb + hq * a.q_sh + (int64_t)(live ? row : w.lo) * a.q_st;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            q[s].q = reinterpret_cast<const uint4*>(p)[2 * s + h];
            if (!live) q[s].q = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const float c2 = a.scale * LOG2E;
    f32x16 o[4], s[2];
    Frag p[4];
    float top, sum;  // reference of the row's weights in log2, this lane's share of their sum
    float lift = LIFT<F16>;
    auto start = [&]() INLINE {
        top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    };
    start();

    // S^T of a tile of keys and (or) the last weights' sums of a tile of values.  The operands are asked for some products
    // ahead: left to itself the compiler reads two, waits and multiplies (595 us against 544 at 8192 tokens).  `between`
    // is called when all operands are read and AHEAD products are left.
    auto products = [&](const uint4* k, const uint4* v, f32x16* out, auto qk, auto pv, auto between) INLINE {
        const uint8_t *const k8 = reinterpret_cast<const uint8_t*>(k), *const v8 = reinterpret_cast<const uint8_t*>(v);
        Frag last[AHEAD];
        auto value_operand = [&](int i) INLINE {
            Frag f;
#pragma unroll
            for (int e = 0; e < 2; ++e) f.t[e] = read_tr(v8 + value_offset(i & 3, e, lane) + 16 * 256 * (i >> 2));
            return f;
        };
        auto key_operand = [&](int i) INLINE {
            Frag f;
            f.q = *reinterpret_cast<const uint4*>(k8 + key_offset(i >> 1, lane) + 32 * 256 * (i & 1));
            return f;
        };
        if constexpr (pv) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const Frag f = value_operand(i);
                if (!qk && i >= 16 - AHEAD) last[i - (16 - AHEAD)] = f;
                else out[i & 3] = mfma_32<F16>(f, p[i >> 2], out[i & 3]);
            }
        }
        if constexpr (qk) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const Frag f = key_operand(i);
                if (i >= 16 - AHEAD) last[i - (16 - AHEAD)] = f;
                else s[i & 1] = mfma_32<F16>(f, q[i >> 1], s[i & 1]);
            }
        }
        if constexpr (pv) {
            __builtin_amdgcn_sched_group_barrier(DS_READ, 2 * AHEAD, 0);
#pragma unroll
            for (int i = 0; i < 16 - AHEAD; ++i) {
                __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
                __builtin_amdgcn_sched_group_barrier(DS_READ, 2, 0);
            }
        } else {
            __builtin_amdgcn_sched_group_barrier(DS_READ, AHEAD, 0);
        }
        if constexpr (qk) {
#pragma unroll
            for (int i = 0; i < (pv ? 16 : 16 - AHEAD); ++i) {
                __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
                __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
            }
        }
        between();
#pragma unroll
        for (int i = 16 - AHEAD; i < 16; ++i) {
            const Frag f = last[i - (16 - AHEAD)];
            if constexpr (qk) s[i & 1] = mfma_32<F16>(f, q[i >> 1], s[i & 1]);
            else out[i & 3] = mfma_32<F16>(f, p[i >> 2], out[i & 3]);
        }
    };
    // weights of the scores of tile t0, in their B-operand order
    auto softmax = [&](int t0) INLINE {
        if (t0 + TK > wrow + 1) {  // some row leaves out some token
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > row) s[t][i] = -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
        // the reference is raised when some score is more than LAZY above it; -inf and NaN do not raise it
        if (__any(__builtin_fmaf(mx, c2, -top) > LAZY<F16>)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * c2;
            const float ref = mx > top ? mx : top;
            const float corr = top == ref ? 1.0f : exp2_(top - ref);
            top = ref;
            sum *= corr;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= corr;
        }
        const float base = (top == -__builtin_inff() ? 0.0f : top) - lift;
        float added = 0.0f;  // a tile's weights first: one by one, small ones lose their last bits to a large sum
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = 8 * x + 2 * k;
                    s[t][i] = exp2_(__builtin_fmaf(s[t][i], c2, -base));
                    s[t][i + 1] = exp2_(__builtin_fmaf(s[t][i + 1], c2, -base));
                    added += s[t][i];
                    added += s[t][i + 1];
                    p[2 * t + x].u[k] = pack2<F16>(s[t][i], s[t][i + 1]);
                }
        sum += added;
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};

    // ---- The halves take turns: while one does its products, QK of its tile j and PV of its tile j - 1, the other does the
    // softmax of its scores.  In time slots with a barrier between them:
    //   slot 2 j      first half: products of j      second half: softmax of j - 1
    //   slot 2 j + 1  first half: softmax of j       second half: products of j
    // With KS = 1, K of tile j and V of tile j - 1 are read in slots 2 j and 2 j + 1, and those of the next step come in
    // meanwhile.  Tiles that leave a wave's rows out whole take their turns like the others, with weights of 0.
    {
        wait_loads();
        barrier();
        if (second) {
            load_k(1);
            load_v(0);
            barrier();
        }
        auto turn = [&](int j, auto qk, auto pv) INLINE {
            int half = wave >> 2;
            asm volatile("" : "+s"(half));  // one copy of the loop, not one for each half
            const bool later = half != 0;
            // the other half may begin when the operands are read: it has its own to wait for.  The loads come behind the
            // reads, since the compiler has every read of LDS wait for the loads to it ahead of it
            auto between = [&]() INLINE {
                wait_reads();
                if (later) {
                    wait_loads();
                } else {
                    load_k(j + 1);
                    load_v(j);
                }
                barrier();
            };
            __builtin_amdgcn_s_setprio(1);
            products(s_k[part][j & 1], s_v[part][(j - 1) & 1], o, qk, pv, between);
            __builtin_amdgcn_s_setprio(0);
            if (later) {
                load_k(j + 2);
                load_v(j + 1);
            }
            if constexpr (qk) softmax(w.lo + (KS * j + part) * TK);
            if (!later) wait_loads();
            barrier();
        };
        turn(0, yes, no);
        for (int j = 1; j < steps; ++j) turn(j, yes, yes);
        turn(steps, no, yes);
        if (!second) barrier();
    }

    // ---- A left-out token's weight is 0, which makes NaN of a value that is not finite.  A workgroup that ends with a sum
    // that is not finite walks its tiles once more, with care: such values are taken out of the tile and added apart, and
    // bf16 weights are in units of 2^32, so that no number of finite values adds up to an infinity.
    uint32_t most = 0u;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = std::max(most, __float_as_uint(o[d][i]) & 0x7FFFFFFFu);
    if (__syncthreads_or(most >= 0x7F800000u)) {
        start();
        if constexpr (!F16) lift = -32.0f;
        uint4 *const ck = s_k[0][0], *const cv = s_v[0][0];
        constexpr int CC = TK * 16 / T;
#pragma unroll 1
        for (int t0 = w.lo; t0 < k_end; t0 += TK) {
            const bool some = part == 0 && t0 < wrow + 32;  // the wave's rows attend to some token of the tile
            __syncthreads();
            // values that are not finite as 0, and again as counts: +inf 1, -inf 128, NaN 16384, at most 64 of each
#pragma unroll 1
            for (int round = 0; round < 2; ++round) {
#pragma unroll 1
                for (int i = 0; i < CC; ++i) {
                    const int id = i * T + threadIdx.x, tok = id >> 4, c = (id & 15) ^ swizzle(tok);
                    const int64_t t = std::min(t0 + tok, k_end - 1);
                    if (round == 0) ck[id] = *reinterpret_cast<const uint4*>(kb + t * a.k_st + 8 * c);
                    uint4 x = *reinterpret_cast<const uint4*>(vb + t * a.v_st + 8 * c);
                    const uint32_t inf = F16 ? 0x7C00u : 0x7F80u;
                    for (uint32_t* u : {&x.x, &x.y, &x.z, &x.w}) {
                        uint32_t f[2];
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t y = (*u >> (16 * e)) & 0xFFFFu, z = y & 0x7FFFu;
                            const float count = z < inf ? 0.0f : z > inf ? 16384.0f : y == inf ? 1.0f : 128.0f;
                            f[e] = round ? pack2<F16>(count, 0.0f) : z < inf ? y : 0u;
                        }
                        *u = f[0] | f[1] << 16;
                    }
                    cv[id] = x;
                }
                __syncthreads();
                if (some && round == 0) {
                    products(ck, nullptr, nullptr, yes, no, [] {});
                    softmax(t0);
                    products(nullptr, cv, o, no, yes, [] {});
                } else if (some) {
                    f32x16 counts[4];
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) counts[d][i] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            p[ks].u[k] = pack2<F16>(s[ks >> 1][8 * (ks & 1) + 2 * k] > 0.0f ? 1.0f : 0.0f,
                                                    s[ks >> 1][8 * (ks & 1) + 2 * k + 1] > 0.0f ? 1.0f : 0.0f);
                    products(nullptr, cv, counts, no, yes, [] {});
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int x = (int)counts[d][i];
                            if (x & 127) o[d][i] += __builtin_inff();
                            if (x >> 7 & 127) o[d][i] -= __builtin_inff();
                            if (x >> 14) o[d][i] = __builtin_nanf("");
                        }
                }
                __syncthreads();
            }
        }
    }

    float total = sum + __shfl_xor(sum, 32), inv;
    if constexpr (KS == 2) {  // the halves' sums meet
        float* const meet = reinterpret_cast<float*>(s_k);
        float2* const ms = reinterpret_cast<float2*>(s_v);
        __syncthreads();
        if (second) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) meet[((wave & 3) * 64 + 16 * d + i) * 64 + lane] = o[d][i];
            ms[(wave & 3) * 64 + lane] = make_float2(top, total);
        }
        __syncthreads();
        if (second) return;
        const float2 m = ms[wave * 64 + lane];
        const float best = fmaxf(top, m.x), safe = best == -__builtin_inff() ? 0.0f : best;
        float w0 = exp2_(top - safe), w1 = exp2_(m.x - safe);
        total = total * w0 + m.y * w1;
        top = best;
        // divided first: two finite sums may add up to an infinity
        w0 /= total == 0.0f ? 1.0f : total, w1 /= total == 0.0f ? 1.0f : total, inv = 1.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                o[d][i] = o[d][i] * w0 + (w1 == 0.0f ? 0.0f : meet[(wave * 64 + 16 * d + i) * 64 + lane] * w1);
    } else {
        inv = 1.0f / (total == 0.0f ? 1.0f : total);
    }

    // ---- rows out: two lanes hold a row's dims 8 j + 4 h + (0..3); pairs of j are exchanged for 16-byte stores
    const bool mine = row >= w.w_lo && row < w.w_hi;
    if (a.lse && mine && h == 0)
        a.lse[lse_row + row] = !live || total == 0.0f ? -__builtin_inff() : (top - lift) / LOG2E + __builtin_logf(total);
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
            uint32_t x[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int i = 4 * (2 * jj + e) + 2 * k;
                    x[e][k] = live ? pack2<F16>(o[d][i] * inv, o[d][i + 1] * inv) : 0u;
                }
            const auto lo = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
            const auto hi = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
            if (mine)
                *reinterpret_cast<uint4*>(ob + row * a.o_st + 32 * d + 8 * (2 * jj + h)) =
                    make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
}

template <bool F16, int KS>
void launch(PromptArgs& a, unsigned grid_kv, hipStream_t s) {
    constexpr int BM = 256 / KS;
    a.row_blocks = (a.tokens + BM - 1) / BM + (a.cu ? a.n_seqs + 2 : 0);
    hipLaunchKernelGGL((prompt_kernel<F16, KS>), dim3(grid_kv * (unsigned)a.row_blocks), dim3(512), 0, s, a);
}

}  // namespace

extern "C" int tq_prompt_attention(const void* q, const void* k, const void* v, void* out, float* lse, int is_f16,
                                   int batch, int q_heads, int kv_heads, int64_t tokens, int dim, int64_t q_sb,
                                   int64_t q_sh, int64_t q_st, int64_t k_sb, int64_t k_sh, int64_t k_st, int64_t v_sb,
                                   int64_t v_sh, int64_t v_st, int64_t o_sb, int64_t o_sh, int64_t o_st,
                                   const int32_t* cu_seqlens, int n_seqs, const int32_t* seq_starts,
                                   const int32_t* seq_ends, int zero_outside, float scale, void* stream) {
    if (!q || !k || !v || !out || batch < 1 || q_heads < 1 || kv_heads < 1 || tokens < 1 || q_heads % kv_heads ||
        !(scale > 0.0f) || scale == __builtin_inff() ||
        (cu_seqlens && (batch != 1 || n_seqs < 1 || seq_starts || seq_ends)))
        return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D) return TQ_ERR_UNSUPPORTED;
    for (int64_t s : {q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st})
        if (s % 8) return TQ_ERR_UNSUPPORTED;
    // offsets inside a tile of 64 keys are 32 bits wide
    for (int64_t s : {k_st, v_st})
        if (s < 0 || s >= (int64_t)1 << 25) return TQ_ERR_UNSUPPORTED;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return TQ_ERR_UNSUPPORTED;
    // rows are counted in 32 bits, and threads: 512 to a block
    const int64_t blocks = (tokens + 127) / 128 + (cu_seqlens ? (int64_t)n_seqs + 2 : 0);
    if (tokens > (int64_t)1 << 30 || blocks * batch * q_heads >= (int64_t)1 << 23) return TQ_ERR_UNSUPPORTED;
    PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                 static_cast<uint16_t*>(out), lse, batch, q_heads, kv_heads, (int)tokens, q_sb, q_sh, q_st, k_sb, k_sh,
                 k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st, cu_seqlens, n_seqs, seq_starts, seq_ends, zero_outside != 0,
                 scale, 0};
    const unsigned grid_kv = (unsigned)(batch * q_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    // KS = 2 while its blocks of 128 rows are at most two for each of the 256 CUs (one fits a CU at a time): 1 x 32 heads of 1024
    // tokens take 24 us with it and 32 with KS = 1, of 2048 54 and 61; past that a CU has blocks to go on with, and its merge
    // and its smaller blocks cost more than they save: 2400 tokens take 81 and 77 us, 8192 625 and 584.
    const bool wide = blocks * batch * q_heads > 512;
    if (is_f16) wide ? launch<true, 1>(a, grid_kv, s) : launch<true, 2>(a, grid_kv, s);
    else wide ? launch<false, 1>(a, grid_kv, s) : launch<false, 2>(a, grid_kv, s);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
