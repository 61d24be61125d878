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

#include "tq_common.h"

namespace {

constexpr int D = TQ_DIM;
constexpr int TK = 64;  // tokens per tile
constexpr float LOG2E = 1.44269504f;

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
__device__ __forceinline__ s16x4 read_tr(const uint16_t* l) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)l);
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

template <bool F16, int RB, int W>
__global__ __launch_bounds__(64 * W, RB == 1 ? 2 : 1) void prompt_kernel(PromptArgs a) {
    constexpr int T = 64 * W, BM = 32 * RB * W;
    constexpr int CH = TK * 16 / T;  // 16-byte chunks of K, and of V, a thread brings in per tile
    __shared__ uint4 s_k[TK * 16];
    __shared__ uint4 s_v[TK * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, h = lane >> 5;
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

    // ---- the wave's query rows: dims 16 s + 8 h + (0..7) of row r of each block of 32
    const int wrow = w.row0 + wave * 32 * RB;
    Frag q[RB][8];
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        const int row = wrow + 32 * m + r;
        const bool live = row >= w.lo && row < w.hi;
        const uint16_t* p = a.q + w.b * a.q_sb + hq * a.q_sh + (int64_t)(live ? row : w.lo) * a.q_st;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            q[m][s].q = reinterpret_cast<const uint4*>(p)[2 * s + h];
            if (!live) q[m][s].q = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    const uint16_t* const kb = a.k + w.b * a.k_sb + kvh * a.k_sh;
    const uint16_t* const vb = a.v + w.b * a.v_sb + kvh * a.v_sh;
    const int k_end = (int)std::min<int64_t>(w.hi, (int64_t)w.row0 + BM);

    // a tile to LDS; tokens past the last are copies of it, left out by the mask
    auto load_tile = [&](int t0) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int id = i * T + threadIdx.x, tok = id >> 4, c = (id & 15) ^ swizzle(tok);
            const int64_t t = std::min(t0 + tok, k_end - 1);
            load_lds16(kb + t * a.k_st + 8 * c, s_k + i * T + wave * 64);
            load_lds16(vb + t * a.v_st + 8 * c, s_v + i * T + wave * 64);
        }
    };

    const float c2 = a.scale * LOG2E;
    f32x16 o[RB][4];
    float top[RB], sum[RB];  // reference of a row's weights, in units of q . k, and this lane's share of their sum
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        top[m] = -__builtin_inff(), sum[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[m][d][i] = 0.0f;
    }
    const uint16_t* const v16 = reinterpret_cast<const uint16_t*>(s_v);

    for (int t0 = w.lo; t0 < k_end; t0 += TK) {
        __syncthreads();
        load_tile(t0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // of this wave's part, ahead of the barrier
        __syncthreads();
        const bool edge = t0 + TK > w.row0 + 1;  // some row leaves out some token
        bool special = false;
        if (edge) {
            // a left-out token's weight is 0, which makes NaN of a value that is not finite: such values
            // are taken out of the tile and added apart
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint4 x = s_v[i * T + threadIdx.x];
                const uint32_t e = F16 ? 0x7C00u : 0x7F80u;
                for (uint32_t u : {x.x, x.y, x.z, x.w})
                    special |= (u & e) == e || ((u >> 16) & e) == e;
            }
            special = __syncthreads_or(special);
        }
        if (special) {
#pragma unroll 1
            for (int i = 0; i < CH; ++i) {
                uint4 x = s_v[i * T + threadIdx.x];
                const uint32_t e = F16 ? 0x7C00u : 0x7F80u;
                for (uint32_t* u : {&x.x, &x.y, &x.z, &x.w}) {
                    if ((*u & e) == e) *u &= 0xFFFF0000u;
                    if (((*u >> 16) & e) == e) *u &= 0x0000FFFFu;
                }
                s_v[i * T + threadIdx.x] = x;
            }
            __syncthreads();
        }

        f32x16 s[RB][2];
#pragma unroll
        for (int m = 0; m < RB; ++m)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[m][t][i] = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                Frag kf;
                const int tok = 32 * t + r;
                kf.q = s_k[tok * 16 + ((2 * ks + h) ^ swizzle(tok))];
#pragma unroll
                for (int m = 0; m < RB; ++m) s[m][t] = mfma_32<F16>(kf, q[m][ks], s[m][t]);
            }
        Frag p[RB][4];
#pragma unroll
        for (int m = 0; m < RB; ++m) {
            const int row = wrow + 32 * m + r;
            if (edge) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > row) s[m][t][i] = -__builtin_inff();
            }
            float mx = top[m];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[m][t][i]);
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float safe = mx == -__builtin_inff() ? 0.0f : mx;
            if (__any(mx > top[m])) {
                const float corr = exp2_(__builtin_fmaf(top[m], c2, -safe * c2));
                sum[m] *= corr;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[m][d][i] *= corr;
            }
            top[m] = mx;
            const float base = safe * c2;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[m][t][i] = exp2_(__builtin_fmaf(s[m][t][i], c2, -base));
                    sum[m] += s[m][t][i];
                }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        p[m][2 * t + x].u[k] = pack2<F16>(s[m][t][8 * x + 2 * k], s[m][t][8 * x + 2 * k + 1]);
        }
        // V^T of 16 tokens: lane (r, h) takes dim 32 d + r of tokens 4 h + (0..3) and 8 + 4 h + (0..3)
        auto v_frag = [&](int ks, int d) {
            Frag vf;
            const int cl = 4 * d + 2 * (r >> 4) + ((lane & 3) >> 1);  // 16-byte chunk of this lane's 4 dims
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int tok = 16 * ks + 8 * e + 4 * h + ((lane & 15) >> 2);
                vf.t[e] = read_tr(v16 + (tok * 16 + (cl ^ swizzle(tok))) * 8 + 4 * (lane & 1));
            }
            return vf;
        };
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const Frag vf = v_frag(ks, d);
#pragma unroll
                for (int m = 0; m < RB; ++m) o[m][d] = mfma_32<F16>(vf, p[m][ks], o[m][d]);
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
                s_v[id] = x;
            }
            __syncthreads();
#pragma unroll
            for (int m = 0; m < RB; ++m) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        p[m][ks].u[k] = pack2<F16>(s[m][ks >> 1][8 * (ks & 1) + 2 * k] > 0.0f ? 1.0f : 0.0f,
                                                   s[m][ks >> 1][8 * (ks & 1) + 2 * k + 1] > 0.0f ? 1.0f : 0.0f);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    f32x16 n;
#pragma unroll
                    for (int i = 0; i < 16; ++i) n[i] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) n = mfma_32<F16>(v_frag(ks, d), p[m][ks], n);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int x = (int)n[i];
                        if (x & 127) o[m][d][i] += __builtin_inff();
                        if (x >> 7 & 127) o[m][d][i] -= __builtin_inff();
                        if (x >> 14) o[m][d][i] = __builtin_nanf("");
                    }
                }
            }
        }
    }

    // ---- rows out: two lanes hold a row's dims 8 j + 4 h + (0..3); pairs of j are exchanged for 16-byte stores
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        const int row = wrow + 32 * m + r;
        float total = sum[m] + __shfl_xor(sum[m], 32);
        const bool live = row >= w.lo && row < w.hi;
        const float inv = live ? 1.0f / (total == 0.0f ? 1.0f : total) : 0.0f;
        const bool mine = row >= w.w_lo && row < w.w_hi;
        if (a.lse && mine && h == 0) {
            a.lse[lse_row + row] = !live || total == 0.0f ? -__builtin_inff()
                                                          : top[m] * a.scale + __builtin_logf(total);
        }
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
                        x[e][k] = live ? pack2<F16>(o[m][d][i] * inv, o[m][d][i + 1] * inv) : 0u;
                    }
                const auto lo = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
                const auto hi = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
                if (mine)
                    *reinterpret_cast<uint4*>(ob + row * a.o_st + 32 * d + 8 * (2 * jj + h)) =
                        make_uint4(lo[0], hi[0], lo[1], hi[1]);
            }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <bool F16, int RB, int W>
void launch(PromptArgs& a, unsigned grid_kv, hipStream_t s) {
    constexpr int BM = 32 * RB * W;
    a.row_blocks = (a.tokens + BM - 1) / BM + (a.cu ? a.n_seqs + 2 : 0);
    hipLaunchKernelGGL((prompt_kernel<F16, RB, W>), dim3(grid_kv * (unsigned)a.row_blocks), dim3(64 * W), 0, s, a);
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
    if (is_f16) launch<true, 1, 4>(a, grid_kv, s);
    else launch<false, 1, 4>(a, grid_kv, s);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
