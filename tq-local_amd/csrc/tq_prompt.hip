// tq_prompt.hip -- causal attention over whole prompts for gfx950: grouped query heads, padded batches,
// and prompts of different lengths packed behind one another.
//
//   o_i = sum_{j <= i} p_ij v_j / sum_{j <= i} p_ij,   p_ij = 2^(c q_i . k_j - m_i),   c = scale log2(e)
//
// j over the sequence of row i.  One pass over the keys with a running reference m_i of each row.
//
// Layout.  A workgroup owns 32 RB W consecutive rows of one sequence and query head, a wave 32 RB of
// them, and all waves walk the keys in tiles of 64 tokens.
//   S^T = K Q^T   v_mfma_f32_32x32x16, A = 32 tokens x 16 dims, B = 16 dims x 32 rows: lane (r = l % 32,
//                 h = l / 32) ends with row r's scores of the tokens 8 j + 4 h + (0..3) of a block of 32
//   O^T = V^T P^T A = 32 dims x 16 tokens, B = 16 tokens x 32 rows.  The order of the 16 tokens along k
//                 is free: it is the order the scores come back in, so a lane's weights become its B
//                 operand as they are, and ds_read_b64_tr_b16 takes V^T out of row-major rows in that
//                 order (16 lanes read 4 tokens x 16 dims and each ends with one dim's 4 tokens).
// K and V go from memory to LDS without passing registers (16 bytes a lane); a row's 16-byte chunk c is at
// slot c ^ f(token), f taking the token's low four bits to the slot with the bits 0-1 on top, so that
// the 16 rows of a K read and the 4 x 2 rows of a V read both meet every bank once.
//
// Rounding.  Scores, weights, sums and outputs are fp32; the weights are rounded to the values' type for
// their product, once and to nearest: relative 2^-9 (bf16), as much as the output's own rounding, and
// independent from weight to weight.  The sum of a row's weights is of the unrounded ones.

#include <algorithm>
#include <type_traits>

#include "tq_common.h"

namespace {

constexpr int D = TQ_DIM;
constexpr int TK = 64;  // tokens per tile
constexpr float LOG2E = 1.44269504f;
constexpr float LAZY = 8.0f;  // log2 that a score may exceed its row's reference by

constexpr int MFMA = 0x8, DS_READ = 0x100;  // kinds of instructions for the scheduler

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
union Frag {
    uint32_t u[4];
    uint4 q;
    s16x4 t[2];
    bf16x8 b;
    f16x8 f;
};

template <bool F16>
__device__ __forceinline__ f32x16 mfma_32(const Frag& a, const Frag& b, f32x16 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.f, b.f, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
}
// two fp32 values to the element type, nearest even
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 p = {a, b};
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
// 2^x (v_exp_f32, 1 ulp; 2^-inf = 0)
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int swizzle(int token) { return ((token & 3) << 2) | ((token >> 2) & 3); }

__device__ __forceinline__ void load_lds16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)g,
                                     (__attribute__((address_space(3))) uint32_t*)l, 16, 0, 0);
}
__device__ __forceinline__ s16x4 read_tr(const uint8_t* l) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)l);
}
// Byte offsets in a tile: a lane's 16 bytes of key row r in step ks (plus 32 rows for the second block of tokens), and what it
// gives ds_read_b64_tr_b16 for dims 32 d + (0..31) of the tokens 8 e + 4 h + (0..3) (plus 16 rows per step).
__device__ __forceinline__ int key_offset(int ks, int lane) {
    return (lane & 31) * 256 + (((2 * ks + (lane >> 5)) ^ swizzle(lane & 31)) << 4);
}
__device__ __forceinline__ int value_offset(int d, int e, int lane) {
    const int tok = 8 * e + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int chunk = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return tok * 256 + ((chunk ^ swizzle(tok)) << 4) + 8 * (lane & 1);
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

// Waits of a wave for its own loads to LDS, and the barrier, with nothing moved across either.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

template <bool F16, int W>
__global__ __launch_bounds__(64 * W, 2) void prompt_kernel(PromptArgs a) {
    constexpr int T = 64 * W, BM = 32 * W;
    constexpr int CH = TK * 16 / T;  // 16-byte chunks of K, and of V, a thread brings in per tile
    constexpr int BUF = W == 8 ? 2 : 1;
    __shared__ uint4 s_k[BUF][TK * 16];
    __shared__ uint4 s_v[BUF][TK * 16];
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // in a scalar register, and what follows from it
    // workgroups of one KV head share an XCD's L2 where their number divides by the eight XCDs
    const int n_kv = (a.cu ? 1 : a.batch) * a.kv_heads, group = a.q_heads / a.kv_heads;
    const int kv = blockIdx.x % n_kv, item = blockIdx.x / n_kv;
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

    // ---- the wave's query rows: dims 16 s + 8 h + (0..7) of row r
    const int wrow = w.row0 + 32 * wave, row = wrow + r;
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
    const uint16_t* const kb = a.k + w.b * a.k_sb + kvh * a.k_sh;
    const uint16_t* const vb = a.v + w.b * a.v_sb + kvh * a.v_sh;
    const int k_end = (int)std::min<int64_t>(w.hi, (int64_t)w.row0 + BM);

    // a tile's rows to LDS; tokens past the last are copies of it, left out by the mask
    auto load_rows = [&](const uint16_t* base, int64_t st, uint4* dst, int t0) {
        const uint16_t* const tile = base + (int64_t)t0 * st;  // scalar
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * T + threadIdx.x, tok = id >> 4, c = (id & 15) ^ swizzle(tok);
            load_lds16(tile + std::min(tok, k_end - 1 - t0) * st + 8 * c, dst + i * T + wave * 64);
        }
    };

    const float c2 = a.scale * LOG2E;
    f32x16 o[4], s[2];
    Frag p[4];
    float top = -__builtin_inff(), sum = 0.0f;  // reference of the row's weights in log2, this lane's share of their sum
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;

    auto products_qk = [&](const uint4* k) {
        const uint8_t* const k8 = reinterpret_cast<const uint8_t*>(k);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag kf;
                kf.q = *reinterpret_cast<const uint4*>(k8 + key_offset(ks, lane) + 32 * 256 * t);
                s[t] = mfma_32<F16>(kf, q[ks], s[t]);
            }
        // operands on their way six products ahead
        __builtin_amdgcn_sched_group_barrier(DS_READ, 6, 0);
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
            __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(MFMA, 6, 0);
    };
    auto products_pv = [&](const uint4* v, const Frag* weights, f32x16* out) {
        const uint8_t* const v8 = reinterpret_cast<const uint8_t*>(v);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                Frag vf;
#pragma unroll
                for (int e = 0; e < 2; ++e) vf.t[e] = read_tr(v8 + value_offset(d, e, lane) + 16 * 256 * ks);
                out[d] = mfma_32<F16>(vf, weights[ks], out[d]);
            }
        __builtin_amdgcn_sched_group_barrier(DS_READ, 8, 0);
#pragma unroll
        for (int i = 0; i < 12; ++i) {
            __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
            __builtin_amdgcn_sched_group_barrier(DS_READ, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(MFMA, 4, 0);
    };
    // weights of the scores of tile t0, in their B-operand order
    auto softmax = [&](int t0, auto edge) {
        if constexpr (edge) {
            if (t0 + TK > wrow + 1) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > row) s[t][i] = -__builtin_inff();
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
        // the reference is raised when some score is more than 2^LAZY above it; -inf and NaN do not raise it
        if (__any(__builtin_fmaf(mx, c2, -top) > LAZY)) {
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
        const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = 8 * x + 2 * k;
                    s[t][i] = exp2_(__builtin_fmaf(s[t][i], c2, -base));
                    s[t][i + 1] = exp2_(__builtin_fmaf(s[t][i + 1], c2, -base));
                    sum += s[t][i];
                    sum += s[t][i + 1];
                    p[2 * t + x].u[k] = pack2<F16>(s[t][i], s[t][i + 1]);
                }
    };

    int t0 = w.lo;
    if constexpr (W == 8) {
        // ---- tiles that every row attends to whole.  Waves 0-3 and 4-7 share the SIMDs two by two and take turns: while the
        // one half does its products, QK of tile j and PV of tile j - 1, the other does the softmax of its scores.  In time
        // slots with a barrier between them:
        //   slot 2 j      first half: products of j      second half: softmax of j - 1
        //   slot 2 j + 1  first half: softmax of j       second half: products of j
        // K of tile j and V of tile j - 1 are read in slots 2 j and 2 j + 1, those of the next step come in meanwhile.
        const int n = w.row0 >= w.lo ? (w.row0 + 1 - w.lo) / TK : 0;
        if (n > 0) {
            const bool second = wave >= 4;
            // this thread's chunks of the next K and V tile
            const uint16_t *kp[CH], *vp[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const int id = i * T + threadIdx.x, tok = id >> 4, c = (id & 15) ^ swizzle(tok);
                kp[i] = kb + (int64_t)(w.lo + tok) * a.k_st + 8 * c;
                vp[i] = vb + (int64_t)(w.lo + tok) * a.v_st + 8 * c;
            }
            const int64_t k_step = TK * a.k_st, v_step = TK * a.v_st;
            auto load_k = [&](int j) {
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    load_lds16(kp[i], s_k[j & 1] + i * T + wave * 64);
                    kp[i] += k_step;
                }
            };
            auto load = [&](int j) {  // K of tile j + 1 and V of tile j
                if (j + 1 < n) load_k(j + 1);
                if (j < n) {
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        load_lds16(vp[i], s_v[j & 1] + i * T + wave * 64);
                        vp[i] += v_step;
                    }
                }
            };
            load_k(0);
            wait_loads();
            barrier();
            if (second) {
                load(0);
                barrier();
            }
            for (int j = 0; j <= n; ++j) {
                if (!second) load(j);
                __builtin_amdgcn_s_setprio(1);
                if (j > 0) products_pv(s_v[(j - 1) & 1], p, o);
                if (j < n) products_qk(s_k[j & 1]);
                __builtin_amdgcn_s_setprio(0);
                if (second) wait_loads();
                barrier();
                if (second) load(j + 1);
                if (j < n) softmax(w.lo + j * TK, std::false_type{});
                if (!second) wait_loads();
                barrier();
            }
            if (!second) barrier();
            t0 = w.lo + n * TK;
        }
    }

    // ---- tiles with tokens that some row leaves out
    for (; t0 < k_end; t0 += TK) {
        __syncthreads();
        load_rows(kb, a.k_st, s_k[0], t0);
        load_rows(vb, a.v_st, s_v[0], t0);
        wait_loads();
        __syncthreads();
        bool special = false;
        if (t0 + TK > w.row0 + 1) {
            // a left-out token's weight is 0, which makes NaN of a value that is not finite: such values
            // are taken out of the tile and added apart
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint4 x = s_v[0][i * T + threadIdx.x];
                const uint32_t e = F16 ? 0x7C00u : 0x7F80u;
                for (uint32_t u : {x.x, x.y, x.z, x.w})
                    special |= (u & e) == e || ((u >> 16) & e) == e;
            }
            special = __syncthreads_or(special);
        }
        if (special) {
#pragma unroll 1
            for (int i = 0; i < CH; ++i) {
                uint4 x = s_v[0][i * T + threadIdx.x];
                const uint32_t e = F16 ? 0x7C00u : 0x7F80u;
                for (uint32_t* u : {&x.x, &x.y, &x.z, &x.w}) {
                    if ((*u & e) == e) *u &= 0xFFFF0000u;
                    if (((*u >> 16) & e) == e) *u &= 0x0000FFFFu;
                }
                s_v[0][i * T + threadIdx.x] = x;
            }
            __syncthreads();
        }
        const bool some = t0 < wrow + 32;  // the wave's rows attend to some token of the tile
        if (some) {
            products_qk(s_k[0]);
            softmax(t0, std::true_type{});
            products_pv(s_v[0], p, o);
        }
        if (special) {
            // what was taken out, counted apart for every row and dim that gives it weight: +inf as 1, -inf as
            // 128, NaN as 16384, at most 64 of each
            __syncthreads();
#pragma unroll 1
            for (int i = 0; i < CH; ++i) {
                const int id = i * T + threadIdx.x, tok = id >> 4, c = (id & 15) ^ swizzle(tok);
                const int64_t t = std::min(t0 + tok, k_end - 1);
                uint4 x = *reinterpret_cast<const uint4*>(vb + t * a.v_st + 8 * c);
                const uint32_t inf = F16 ? 0x7C00u : 0x7F80u;
                for (uint32_t* u : {&x.x, &x.y, &x.z, &x.w}) {
                    uint32_t f[2];
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t y = (*u >> (16 * e)) & 0xFFFFu;
                        const float n = (y & 0x7FFFu) < inf ? 0.0f : (y & 0x7FFFu) > inf ? 16384.0f : y == inf ? 1.0f : 128.0f;
                        f[e] = pack2<F16>(n, 0.0f);
                    }
                    *u = f[0] | f[1] << 16;
                }
                s_v[0][id] = x;
            }
            __syncthreads();
            if (some) {
                f32x16 n[4];
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) n[d][i] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        p[ks].u[k] = pack2<F16>(s[ks >> 1][8 * (ks & 1) + 2 * k] > 0.0f ? 1.0f : 0.0f,
                                                s[ks >> 1][8 * (ks & 1) + 2 * k + 1] > 0.0f ? 1.0f : 0.0f);
                products_pv(s_v[0], p, n);
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int x = (int)n[d][i];
                        if (x & 127) o[d][i] += __builtin_inff();
                        if (x >> 7 & 127) o[d][i] -= __builtin_inff();
                        if (x >> 14) o[d][i] = __builtin_nanf("");
                    }
            }
        }
    }

    // ---- rows out: two lanes hold a row's dims 8 j + 4 h + (0..3); pairs of j are exchanged for 16-byte stores
    const float total = sum + __shfl_xor(sum, 32);
    const float inv = live ? 1.0f / (total == 0.0f ? 1.0f : total) : 0.0f;
    const bool mine = row >= w.w_lo && row < w.w_hi;
    if (a.lse && mine && h == 0)
        a.lse[lse_row + row] = !live || total == 0.0f ? -__builtin_inff() : top / LOG2E + __builtin_logf(total);
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <bool F16, int W>
void launch(PromptArgs& a, unsigned grid_kv, hipStream_t s) {
    constexpr int BM = 32 * W;
    a.row_blocks = (a.tokens + BM - 1) / BM + (a.cu ? a.n_seqs + 2 : 0);
    hipLaunchKernelGGL((prompt_kernel<F16, W>), dim3(grid_kv * (unsigned)a.row_blocks), dim3(64 * W), 0, s, a);
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
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return TQ_ERR_UNSUPPORTED;
    // rows and blocks are counted in 32 bits
    const int64_t blocks = (tokens + 127) / 128 + (cu_seqlens ? (int64_t)n_seqs + 2 : 0);
    if (tokens > (int64_t)1 << 30 || blocks * batch * q_heads >= (int64_t)1 << 24) return TQ_ERR_UNSUPPORTED;
    PromptArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                 static_cast<uint16_t*>(out), lse, batch, q_heads, kv_heads, (int)tokens, q_sb, q_sh, q_st, k_sb, k_sh,
                 k_st, v_sb, v_sh, v_st, o_sb, o_sh, o_st, cu_seqlens, n_seqs, seq_starts, seq_ends, zero_outside != 0,
                 scale, 0};
    const unsigned grid_kv = (unsigned)(batch * q_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool wide = tokens * batch * q_heads >= (int64_t)256 * 256;
    if (is_f16) wide ? launch<true, 8>(a, grid_kv, s) : launch<true, 4>(a, grid_kv, s);
    else wide ? launch<false, 8>(a, grid_kv, s) : launch<false, 4>(a, grid_kv, s);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
