// tq_tiles.h -- attention of up to 64 query rows at a time over tiles of 32 packed tokens (gfx950), shared by the attention of drafted
// trees and the attention behind shared prompts.
//
//   logit_t = scale (|k_t| <q R_k^T, C_k[kidx_t]> + sqrt(pi/2)/D |r_t| <q S^T, s_t>)
//   out     = (sum_t softmax_t |v_t| C_v[vidx_t]) R_v
// Keys and values are never rotated: the queries are, once, and the sums are rotated back, once.  attend_tiles() gives a workgroup's
// partial sums; which rows they are, which tiles the workgroup takes and who attends to what of them its Source says.  merge_rows()
// weighs and adds the partials of the splits and rotates them back.
//
// Codes to fp16.  Keys become A operands in registers, a lane's token and half of its dims: a byte lookup (v_perm_b32) of the
// centroid's two halves for four codes at once.  Which four codes meet in a register follows from the packing (those at the
// same bits of neighbouring bytes), so each bit width has an order of the 128 dims of its own, which the queries are
// written in (position_of).  Signs stay where they are, as the lowest mantissa bits of fp16 numbers.  Values are looked up in LDS, two
// codes at a time (PairTable), and turned around by ds_read_b64_tr_b16.
//
// Rounding.  Rotated queries and centroids are rounded once to fp16, by at most 2^-11 of each, 2^-11 / sqrt(3) root mean square (with
// |q| = 11 and |k| = 20 a logit moves by 7e-4; the queries' part of it goes with LO, most of the centroids' where the caller gives them times a
// factor that fp16 holds them well with, and the rotation divided by it), value centroids too (their sum's errors are kept from adding up
// by the codebook, see tq_value_codebook_f16, or that factor), weights times norm p |v| once: to 11 bits down to 2^-25 of the largest norm's, of the tiles that
// the row attends to any of, at the row's reference, and by up to 2^-36 of it below.  Logits, maxima, weights, sums and outputs are
// fp32.

#pragma once

#include <algorithm>
#include <type_traits>

#include "tq_rows16.h"

namespace tqt {

using namespace tqr;

constexpr int D = TQ_DIM;
constexpr int TK = 32;         // tokens per tile
constexpr int MIN_TILES = 8;   // tiles of a split
constexpr int MAX_SPLIT = 64;  // partials a merge wave weighs with one lane each
constexpr float LOG2E = 1.44269504f;
// Log2 that a score may exceed its row's reference by, and of the largest weight times norm at the reference: 15 together, what fp16
// holds.  The less a score may exceed it the smaller the weights that keep their bits, and the more often references rise: trees of 16
// nodes of 4 heads over 8 sequences of 32768 tokens (8 KV heads, 4-bit Q_prod), and of 64 nodes of 7 heads over 4 of 8192 (4 KV heads, 3-bit
// Q_mse), take with their merges 159 and 71 us with 4, 156 and 69 with 8, 160 and 72 with 2
constexpr float LAZY = 4.0f;
constexpr int TOP_BIT = 11;
constexpr float QJL_SCALE = 1.2533141373155003f / D;  // sqrt(pi/2) / D

#define INLINE __attribute__((always_inline))

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_amdgcn_perm(hi, lo, sel);
}
// the values of lanes l and l ^ 32 joined, in both
__device__ __forceinline__ float max_of_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float sum_of_halves(float x) {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}

// ------------------------------------------------------------------ codes to fp16 rows

// The fp16 centroids' high and low bytes, four entries to a register.
template <int BITS>
struct Lut {
    static constexpr int N = BITS == 4 ? 4 : 2;
    uint32_t hi[N], lo[N];
    __device__ __forceinline__ void load(const float* centers) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            hi[i] = lo[i] = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * i + e < (1 << BITS)) {
                    const uint32_t x = tq::f32_to_f16(centers[4 * i + e]);
                    hi[i] |= (x >> 8) << (8 * e);
                    lo[i] |= (x & 0xFFu) << (8 * e);
                }
        }
    }
    // four codes, one to a byte: their centroids (0, 1) and (2, 3)
    __device__ __forceinline__ void four(uint32_t code, uint32_t& a, uint32_t& b) const {
        uint32_t h, l;
        if constexpr (BITS < 4) {
            h = perm(hi[1], hi[0], code), l = perm(lo[1], lo[0], code);
        } else {
            const uint32_t sel = code & 0x07070707u, up = perm(0u, 0x0000FF00u, (code >> 3) & 0x01010101u);
            h = (perm(hi[3], hi[2], sel) & up) | (perm(hi[1], hi[0], sel) & ~up);
            l = (perm(lo[3], lo[2], sel) & up) | (perm(lo[1], lo[0], sel) & ~up);
        }
        a = perm(h, l, 0x05010400u), b = perm(h, l, 0x07030602u);
    }
};

// 32 codes (BITS words) one to a byte, in the order of position_of.
template <int BITS>
__device__ __forceinline__ void unpack32(const uint32_t* w, uint32_t* q) {
    if constexpr (BITS == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) q[2 * j] = w[j] & 0x0F0F0F0Fu, q[2 * j + 1] = (w[j] >> 4) & 0x0F0F0F0Fu;
    } else if constexpr (BITS == 3) {
        const uint32_t b0 = perm(w[2], perm(w[1], w[0], 0x0C060300u), 0x05020100u);
        const uint32_t b1 = perm(w[2], perm(w[1], w[0], 0x0C070401u), 0x06020100u);
        const uint32_t b2 = perm(w[2], perm(w[1], w[0], 0x0C0C0502u), 0x07040100u);
        q[0] = b0 & 0x07070707u;
        q[1] = (b0 >> 3) & 0x07070707u;
        q[2] = ((b0 >> 6) & 0x03030303u) | ((b1 << 2) & 0x04040404u);
        q[3] = (b1 >> 1) & 0x07070707u;
        q[4] = (b1 >> 4) & 0x07070707u;
        q[5] = ((b1 >> 7) & 0x01010101u) | ((b2 << 1) & 0x06060606u);
        q[6] = (b2 >> 2) & 0x07070707u;
        q[7] = (b2 >> 5) & 0x07070707u;
    } else if constexpr (BITS == 2) {
#pragma unroll
        for (int p = 0; p < 8; ++p) q[p] = (w[p >> 2] >> (2 * (p & 3))) & 0x03030303u;
    } else {
#pragma unroll
        for (int p = 0; p < 8; ++p) q[p] = (w[0] >> p) & 0x01010101u;
    }
}
// Chunk j of four from them.
template <int BITS>
__device__ __forceinline__ uint4 code_chunk(const uint32_t* q, int j, const Lut<BITS>& lut) {
    uint4 x;
    lut.four(q[2 * j], x.x, x.y);
    lut.four(q[2 * j + 1], x.z, x.w);
    return x;
}

// Chunk j of four from 32 sign bits, left where they are: bits i and i + 16 of the word (or of the word moved down by 8,
// for i = 8..15) as the lowest mantissa bits of two fp16 numbers, 2^(p - 24) with p = i mod 8 for a set bit and 0 for a
// clear one (the matrix cores keep subnormals).  The queries carry the 2^(7 - p), and sum_i s_i x_i = 2 sum_i bit_i x_i -
// sum_i x_i.
__device__ __forceinline__ uint4 sign_chunk(uint32_t w, int j) {
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (j < 2 ? w : w >> 8) & (0x00010001u << ((4 * j + k) & 7));
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// ------------------------------------------------------------------ queries

// fp32 pairs to bf16 terms to nearest: two leave out at most 2^-16 of a number (half a step of each is 2^-8 of what is left)
template <int N>
__device__ __forceinline__ void split_terms(const float* x, Frag* t) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float a = x[2 * k], b = x[2 * k + 1];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const f32x2 p = {a, b};
            t[n].u[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
            a -= __uint_as_float(t[n].u[k] << 16), b -= __uint_as_float(t[n].u[k] & 0xFFFF0000u);
        }
    }
}

// Where dim j stands among a key's 128 operands: 16 chunks of 8 elements, chunk 2 s + h the lanes' operand of step s for
// dims [64 h, 64 h + 64).  What meets in a register follows from the packing: codes of one and of three bits are at the same
// bits of bytes 8 codes apart, of two bits 4 apart, of four bits 2 apart (2^log_st); signs are taken 16 apart.
// Both orders permute the bits of j: the place of j is the sum of those of its parts.
template <int KB>
__device__ __forceinline__ constexpr int position_of(int j) {
    const int log_st = KB == 4 ? 1 : KB == 2 ? 2 : 3, st = 1 << log_st, x = j & 63, y = x & (4 * st - 1), z = y & (st - 1);
    const int s = ((x >> (log_st + 2)) << (log_st - 1)) + (z >> 1);
    return (2 * s + (j >> 6)) * 8 + 4 * (z & 1) + (y >> log_st);
}
__device__ __forceinline__ constexpr int sign_position_of(int j) {
    const int x = j & 63, n = x & 15, s = 4 * (x >> 5) + (n >> 2);
    return (2 * s + (j >> 6)) * 8 + 2 * (n & 3) + ((x >> 4) & 1);
}
// byte offset of a place: chunk p / 8 = 2 s + h is what lane 32 h + r takes in step s
__device__ __forceinline__ constexpr int operand_offset(int p) {
    return (p >> 4) * 1024 + ((p >> 3) & 1) * 512 + 2 * (p & 7);
}
// ------------------------------------------------------------------ attention

// A packed cache: its arrays, groups `cap` slots apart.
struct Cache {
    const uint8_t *k_codes, *k_signs, *v_codes;
    const uint16_t *k_norms, *k_rnorms, *v_norms;
};

// What all tiles share: the codec, the queries and where the partial sums go.
struct Codec {
    const float *key_centers, *value_centers, *rk, *s;
    float c2;  // scale log2(e)
    const void* q;
    int q_type;
    float* part_o;    // [...][row][D]
    float2* part_ms;  // [...][row] (reference of the weights in log2, sum of weights)
};

// A tile's place: its first slot among all of a cache's, and its tokens.
struct Place {
    Cache c;
    int64_t slot;
    int left;
};

// Eight elements of an fp32 or fp16 query row, wherever it stands.
__device__ __forceinline__ void query_elements(const Codec& a, int64_t at, float* y) {
    if (a.q_type == 1) {
        __builtin_memcpy(y, static_cast<const float*>(a.q) + at, 32);
        return;
    }
    uint32_t w[4];
    __builtin_memcpy(w, static_cast<const uint16_t*>(a.q) + at, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[2 * i] = tq::f16_to_f32(w[i] & 0xFFFFu), y[2 * i + 1] = tq::f16_to_f32(w[i] >> 16);
}

// Pairs of value codes looked up in LDS: entry e of the table is the pair (or the two pairs) that the byte e of the
// packed codes holds, 256 bytes to an entry: 32 copies of the first pair, one for each lane of a half wave, so that no two
// lanes meet in a bank, then 32 of the second.  A byte of 3-bit codes is taken as 6-bit windows: bits 0-5, and 2-7.
template <int VB>
struct PairTable {
    static constexpr int SECOND = 128;  // bytes from an entry's first pair to its second
    // `centers` in LDS
    static __device__ __forceinline__ void build(uint32_t* table, const float* centers, int threads) {
        constexpr uint32_t m = (1u << VB) - 1;
        constexpr int sh = VB == 2 ? 4 : 2;
        for (int i = threadIdx.x; i < 256 * 16; i += threads) {
            const uint32_t e = i >> 4, x = e >> ((i & 15) < 8 || VB == 4 ? 0 : sh);
            const uint32_t pair = pack_f16(centers[x & m], centers[(x >> VB) & m]);
            reinterpret_cast<uint4*>(table)[i] = make_uint4(pair, pair, pair, pair);
        }
    }
    // byte k of w as a table address
    static __device__ __forceinline__ uint32_t at(const uint8_t* table, uint32_t w, int k, uint32_t lane4, int second) {
        const uint32_t off = perm(w, lane4, 0x0C0C0000u | (uint32_t)(4 + k) << 8);
        return *reinterpret_cast<const uint32_t*>(table + off + (second ? SECOND : 0));
    }
    // pairs 8 g + (0..7) of 32 codes (VB words), in the order of their dims
    static __device__ __forceinline__ void look_up(const uint8_t* t, const uint32_t* w, uint32_t lane4, int g, uint32_t* out) {
        if constexpr (VB == 3) {
            auto moved = [&](int i) { return i + 1 < VB ? __builtin_amdgcn_alignbit(w[i + 1], w[i], 4) : w[i] >> 4; };
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // 8 codes in 3 bytes
                const int at0 = 3 * (2 * g + k);
                out[4 * k] = at(t, w[at0 >> 2], at0 & 3, lane4, 0);
                out[4 * k + 1] = at(t, moved(at0 >> 2), at0 & 3, lane4, 1);
                out[4 * k + 2] = at(t, moved((at0 + 1) >> 2), (at0 + 1) & 3, lane4, 0);
                out[4 * k + 3] = at(t, w[(at0 + 2) >> 2], (at0 + 2) & 3, lane4, 1);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int n = 8 * g + k;
                if constexpr (VB == 4) out[k] = at(t, w[n >> 2], n & 3, lane4, 0);
                else if constexpr (VB == 2) out[k] = at(t, w[n >> 3], (n >> 1) & 3, lane4, n & 1);
                else out[k] = at(t, n & 2 ? w[n >> 4] >> 4 : w[n >> 4], (n >> 2) & 3, lane4, n & 1);
            }
        }
    }
};

// 32 RB rows of a KV head to a workgroup, all of them in every wave; the waves take the tiles of 32 tokens in turn.  A lane
// is a token and half of its dims: the keys' codes and signs become its A operands in registers; the values' codes go,
// 16 tokens at a time, through 4 KB of LDS of the wave's own.  No barrier until the waves' sums meet at the end.
template <int RB, bool LO = false>
struct Tiles {
    static constexpr int W = 8;
    static constexpr int T = 64 * W;
    // What is read at a lane's place and many constants from there comes first: a read's own offset reaches 64 KB, and behind that every
    // read had an address register to itself
    struct Parts {
        // the rows' operands for the signs and for the codes (these go on to registers with one block of rows; two do not fit)
        uint4 qs[RB][8 * 64], qc[RB][8 * 64];
        uint4 ql[LO ? RB : 1][LO ? 8 * 64 : 1];  // what fp16 leaves of the codes'
        uint16_t kn[W][32], vn[W][32];
        float ratio[W][32];
        uint32_t table[256 * 64];
        uint4 v[W][16 * 16];
    };
    struct Sums {
        float4 o[W][32][32];  // chunks xor-swizzled by the row
        float2 ms[RB][W][32];
        float4 by[RB][32][W / 4];  // what a row's sums of each wave are multiplied by
        float unit[RB][W][32];
    };
    union Lds {
        uint4 m[2 * 128 * 32];
        Parts t;
        Sums s;
    };
};

// A workgroup's partial sums.  The Source, the same in all its waves, has
//   query(row)         where row `row` of the workgroup's stands in a.q, in elements (any place of it for rows past the last)
//   tiles(), whole()   the job's tiles, and how many of them, from the first on, every row attends to in full
//   split(), splits()  which of the job's splits this is: its waves take the tiles 8 split + wave, and every 8 splits-th from there
//   place(tile)        where it stands
//   seen(m, tile)      bit t: whether row 32 m + lane % 32 attends to the tile's token t
//   rows(), partial()  rows whose sums are wanted, and where they go
//   prefetch(), publish(), take_row()  its own loads: asked for, shared in LDS, and taken by a lane for row 32 m + lane % 32
//
// LO: the rotated queries are two fp16 terms for the codes' products (the signs' weigh a tenth of them), which leave out 2^-22 of a
// number, for queries of more bits than bf16 ones.
template <int KB, int VB, bool QJL, int RB, int NQ, bool LO = false, class Source>
__device__ __forceinline__ void attend_tiles(const Codec& a, Source& src, int lane, int wave) {
    using N = Tiles<RB, LO>;
    constexpr int W = N::W;
    __shared__ typename N::Lds lds;
    __shared__ float s_centers[1 << VB];
    __shared__ float s_top[W][32], s_sum[RB][4][32], s_c[RB][32];
    int r = lane & 31, h = lane >> 5;
    // ---- What the queries' rotation takes is asked for first, then a first tile of the cache, then the small things: a workgroup of a
    // short history waits for memory once.  The matrices come by way of LDS: read straight into operands, 32 rows at a time, they
    // were 10000 cycles on their way.  Their 16-byte chunks are xor-swizzled by the row
#pragma unroll
    for (int i = 0; i < (QJL ? 16 : 8); ++i) {  // 64 chunks, two rows, a time
        const int at = (8 * i + wave) * 64 + lane, row = (at >> 5) & 127;
        load_lds16((i < 8 ? a.rk : a.s) + row * D + 4 * ((at & 31) ^ (row & 31)), &lds.m[(8 * i + wave) * 64]);
    }
    Frag x[8][NQ];  // a block's queries: lane (r, h) has row r's dims 16 s + 8 h + (0..7)
    auto load_queries = [&](int m) INLINE {
        const int64_t at = src.query(32 * m + r) + 8 * h;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if constexpr (NQ == 1) {
                __builtin_memcpy(&x[s][0], static_cast<const uint16_t*>(a.q) + at + 16 * s, 16);  // rows past the last: some row
            } else {
                float y[8];
                query_elements(a, at + 16 * s, y);
                split_terms<NQ>(y, x[s]);
            }
        }
    };
    load_queries(0);

    const int64_t tiles = src.tiles();
    const int step_tiles = src.splits() * W;  // tiles in turn, to the waves of all splits

    // a lane's part of a tile, on its way: half of token r's key codes and signs and its norms, and a quarter of the value
    // codes of tokens lane % 16 and lane % 16 + 16.  The arrays are at scalar addresses, a lane's place in them 32-bit
    // offsets; tokens past the last are copies of it, left out by the mask
    uint32_t wk[2 * KB], ws[2], wv[2][VB];
    uint16_t kn, rn = 0, vn;
    auto load_keys = [&](int64_t tile) {
        const Place p = src.place(tile);
        const uint32_t tok = std::min<uint32_t>(r, (uint32_t)p.left - 1);
        __builtin_memcpy(wk, __builtin_assume_aligned(p.c.k_codes + p.slot * (16 * KB) + (tok * (16 * KB) + 8 * KB * h), 8), 8 * KB);
        if constexpr (QJL) {
            __builtin_memcpy(ws, __builtin_assume_aligned(p.c.k_signs + p.slot * 16 + (tok * 16 + 8 * h), 8), 8);
            rn = (p.c.k_rnorms + p.slot)[tok];
        }
        kn = (p.c.k_norms + p.slot)[tok], vn = (p.c.v_norms + p.slot)[tok];
    };
    auto load_values = [&](int64_t tile) {
        const Place p = src.place(tile);
        const uint32_t last = (uint32_t)p.left - 1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t tok = std::min<uint32_t>((lane & 15) + 16 * x, last);
            __builtin_memcpy(wv[x], __builtin_assume_aligned(p.c.v_codes + p.slot * (16 * VB) + (tok * (16 * VB) + 4 * VB * (lane >> 4)), 4),
                             4 * VB);
        }
    };
    int64_t tile = src.split() * W + wave;
    if (RB == 1 && tile < tiles) load_keys(tile), load_values(tile);
    float key_center[1 << KB];
#pragma unroll
    for (int i = 0; i < (1 << KB); ++i) key_center[i] = a.key_centers[i];
    float value_center = 0.0f;
    if (threadIdx.x < (1 << VB)) value_center = a.value_centers[threadIdx.x];
    src.prefetch(wave, lane);
    __builtin_amdgcn_sched_barrier(0);

    wait_loads();
    __syncthreads();
    // a wave has 32 output dims of one of the matrices
    const int mat = wave >> 2, j0 = 32 * (wave & 3);
    const bool works = QJL || mat == 0;
    Frag mt[8][2];
    if (works) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                __builtin_memcpy(&y[4 * e], &lds.m[(128 * mat + j0 + r) * 32 + ((4 * s + 2 * h + e) ^ r)], 16);
            split_terms<2>(y, mt[s]);
        }
    }

    // ---- q R_k^T and q S^T as products of bf16 terms, a bf16 query one, any other two, the matrices two (what is left out,
    // 2^-15 of a product, is 2^-4 of what the rounding to fp16 below may take).  Scaled by a power of two per row, to a largest
    // element in [2^7, 2^8), they go to fp16 operands in LDS
    {
#pragma unroll 1
        for (int m = 0; m < RB; ++m) {
            f32x16 acc = zero16();
            if (works) {
#pragma unroll
                for (int s = 0; s < 8; ++s)
#pragma unroll
                    for (int i = 1; i >= 0; --i)
#pragma unroll
                        for (int j = NQ - 1; j >= 0; --j)
                            if (i + j <= 1) acc = mfma_bf16(mt[s][i], x[s][j], acc);
            }
            if (m + 1 < RB) load_queries(m + 1);
            // this lane: row r's dims j0 + 8 j + 4 h + (0..3)
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (mat) acc[i] *= QJL_SCALE;
                most = fmaxf(most, fabsf(acc[i]));
            }
            most = max_of_halves(most);
            if (h == 0) s_top[wave][r] = most;
            __syncthreads();
            most = 0.0f;
#pragma unroll
            for (int k = 0; k < (QJL ? 8 : 4); ++k) most = fmaxf(most, s_top[k][r]);
            // rows of zeros, and with an infinity, as they are
            int e = 0;
            if (most > 0.0f && most < __builtin_inff()) e = std::min(126, 7 + 127 - (int)((__float_as_uint(most) >> 23) & 0xFF));
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            // what is next to one another goes out together
            if (mat == 0) {
                auto write = [&](uint4* operands) INLINE {
                    uint8_t* const to = reinterpret_cast<uint8_t*>(operands) + operand_offset(position_of<KB>(j0 + 4 * h)) + 16 * r;
                    if constexpr (KB == 3 || KB == 1) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<uint2*>(to + operand_offset(position_of<KB>(e))) =
                                make_uint2(pack_f16(acc[e], acc[4 + e]), pack_f16(acc[8 + e], acc[12 + e]));
                    } else if constexpr (KB == 4) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint32_t*>(to + operand_offset(position_of<KB>(8 * (i >> 1) + (i & 1)))) =
                                pack_f16(acc[4 * (i >> 1) + (i & 1)], acc[4 * (i >> 1) + (i & 1) + 2]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            *reinterpret_cast<uint16_t*>(to + operand_offset(position_of<KB>(8 * (i >> 2) + (i & 3)))) =
                                (uint16_t)tq::f32_to_f16(acc[i]);
                    }
                };
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] *= up;
                write(lds.t.qc[m]);
                if constexpr (LO) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[i] -= tq::f16_to_f32(tq::f32_to_f16(acc[i]));
                    write(lds.t.ql[m]);
                }
            } else if (QJL) {
                uint8_t* const to = reinterpret_cast<uint8_t*>(lds.t.qs[m]) + operand_offset(sign_position_of(j0 + 4 * h)) + 16 * r;
                const _Float16 bit = h ? 8.0f : 128.0f;  // 2^(7 - j mod 8) is this 2^-(i mod 4): the products with it are exact
                float all = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    Frag f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f16x2 y = __builtin_bit_cast(f16x2, pack_f16(acc[4 * n + e] * up, acc[4 * n + 8 + e] * up));
                        all += (float)y[0] + (float)y[1];
                        const _Float16 by = bit * (_Float16)(1.0f / (1 << e));
                        f.u[e] = __builtin_bit_cast(uint32_t, y * f16x2{by, by});
                    }
                    *reinterpret_cast<uint4*>(to + operand_offset(sign_position_of(8 * n))) = f.q;
                }
                all = sum_of_halves(all);
                if (h == 0) s_sum[m][wave & 3][r] = all;
            }
            if (threadIdx.x < 32) s_c[m][r] = a.c2 * __uint_as_float((uint32_t)(127 - e) << 23);
            __syncthreads();
        }
    }
    if (threadIdx.x < (1 << VB)) s_centers[threadIdx.x] = value_center;
    src.publish(wave, lane);
    Lut<KB> klut;
    klut.load(key_center);
    __syncthreads();
    // nothing of the above stays in registers for the loop
    asm volatile("" : "+v"(lane));
    r = lane & 31, h = lane >> 5;
    if (RB > 1 && tile < tiles) load_keys(tile), load_values(tile);
    Frag q[8];  // with one block of rows
    float c[RB], sign0[RB];
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        c[m] = s_c[m][r];
        // what the scores take from the set bits' products, in units of 2^-17, to the signs'
        sign0[m] = QJL ? -0x1p-18f * (s_sum[m][0][r] + s_sum[m][1][r] + s_sum[m][2][r] + s_sum[m][3][r]) : 0.0f;
    }
    if constexpr (RB == 1)
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s].q = lds.t.qc[0][s * 64 + lane];
    PairTable<VB>::build(lds.t.table, s_centers, N::T);
#pragma unroll
    for (int m = 0; m < RB; ++m) src.take_row(m, 32 * m + r);
    __syncthreads();

    f32x16 o[RB][4];
    float top[RB], sum[RB];  // `top` is a weight's reference, raised when a score is more than 2^LAZY above it
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        top[m] = -__builtin_inff(), sum[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[m][d] = zero16();
    }
    // a row's weights and output sums are in units of 2^-shift, 2^-TOP_BIT of a power of two above the largest |v| of the tiles so far
    // that it attends to any of: weights times norm then reach up to 2^(TOP_BIT + LAZY), and fp16 keeps its 11 bits down to 2^-14, 2^-25 of
    // the reference's.  Tiles of others, as another sequence's own tokens, leave a row's unit alone; in whole tiles all rows' are one
    int shift[RB];
#pragma unroll
    for (int m = 0; m < RB; ++m) shift[m] = TOP_BIT + 24;
    int most_shift = TOP_BIT + 24;  // no row's is larger
    const uint32_t lane4 = (lane & 31) * 4;
    const uint8_t* const table = reinterpret_cast<const uint8_t*>(lds.t.table);
    uint8_t* const v8 = reinterpret_cast<uint8_t*>(lds.t.v[wave]);

    // `masked`: not every row attends to every token of the tile
    auto step = [&](int64_t tile, auto masked) {
        const int left = src.place(tile).left;
        const uint32_t norm = !masked || r < left ? vn : 0u;  // tokens past the last weigh nothing
        if (h == 0) {
            // a key's norm that fp16 holds as 0 counts as 2^-24, its least
            const uint16_t k = QJL && (kn & 0x7FFFu) == 0 ? 1 : kn;
            lds.t.kn[wave][r] = k;
            lds.t.vn[wave][r] = (uint16_t)norm;
            // |r| / |k|, in the units of the sign products
            if constexpr (QJL) lds.t.ratio[wave][r] = tq::f16_to_f32(rn) * 0x1p18f / tq::f16_to_f32(k);
        }
        // ---- scores: |k| (<codes> + |r| / |k| <signs>), the sign products' sums going into the codes'.  A step's chunk of the keys is made
        // beside the products of the one before, and what it takes of the queries is on its way from LDS since two steps
        f32x16 x[RB];
#pragma unroll
        for (int m = 0; m < RB; ++m) x[m] = zero16();
        // A code's chunk meets the queries' lower terms, then their higher ones
        constexpr int SIGNS = QJL ? 8 : 0, TERMS = LO ? 2 : 1, STEPS = SIGNS + 8 * TERMS;
        auto chunk_of = [](int i) INLINE { return i < SIGNS ? i : SIGNS + (i - SIGNS) / TERMS; };
        auto lower = [](int i) INLINE { return LO && i >= SIGNS && (i - SIGNS) % TERMS == 0; };
        Frag ring[2][RB];
        auto ask = [&](int i) INLINE {
#pragma unroll
            for (int m = 0; m < RB; ++m) {
                const int c = chunk_of(i) - SIGNS;
                if (i < SIGNS) ring[i % 2][m].q = lds.t.qs[m][i * 64 + lane];
                else if (lower(i)) ring[i % 2][m].q = lds.t.ql[m][c * 64 + lane];
                else if (RB > 1) ring[i % 2][m].q = lds.t.qc[m][c * 64 + lane];
            }
        };
        uint32_t code[8];
        auto chunk = [&](int i) INLINE {
            Frag f;
            if (i < SIGNS) {
                f.q = sign_chunk(ws[i >> 2], i & 3);
            } else {
                if (((i - SIGNS) & 3) == 0) unpack32<KB>(wk + KB * ((i - SIGNS) >> 2), code);
                f.q = code_chunk<KB>(code, (i - SIGNS) & 3, klut);
            }
            return f;
        };
        ask(0);
        Frag now = chunk(0);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (i + 1 < STEPS) ask(i + 1);
            if (QJL && i == SIGNS) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 r4 = *reinterpret_cast<const f32x4*>(&lds.t.ratio[wave][8 * j + 4 * h]);
#pragma unroll
                    for (int m = 0; m < RB; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[m][4 * j + e] = (x[m][4 * j + e] + sign0[m]) * r4[e];
                }
            }
            Frag next;
            const bool turn = i + 1 < STEPS && chunk_of(i + 1) != chunk_of(i);
            if (turn) next = chunk(chunk_of(i + 1));
#pragma unroll
            for (int m = 0; m < RB; ++m)
                x[m] = mfma_f16(now, RB > 1 || i < SIGNS || lower(i) ? ring[i % 2][m] : q[(chunk_of(i) - SIGNS) & 7], x[m]);
            if (turn) now = next;
            if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);  // the registers hold a few operands at a time
        }
        // the largest finite |v| of the tile: its exponent decides the unit (2^(e + 1) is above it)
        const int e5 = (norm >> 10) & 31, ve = e5 == 31 ? 0 : e5;
        bool rise = false;  // uniform: whether units may have to rise, to `limit`
        int limit = 0;
        if (__any(ve > 14 + TOP_BIT - most_shift)) {
            int e = 0;
            uint64_t largest = ~0ull;
#pragma unroll
            for (int k = 4; k >= 0; --k) {
                const uint64_t set = __ballot(ve >> k & 1) & largest;
                if (set) largest = set, e |= 1 << k;
            }
            rise = true, limit = 14 + TOP_BIT - std::max(e, 1);
            if constexpr (!masked) most_shift = limit;
        }
        if (tile + step_tiles < tiles) load_keys(tile + step_tiles);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        Frag pf[RB][2];
#pragma unroll
        for (int m = 0; m < RB; ++m) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x4 k4 = *reinterpret_cast<const f16x4*>(&lds.t.kn[wave][8 * j + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[m][4 * j + e] = __builtin_fmaf((float)k4[e], x[m][4 * j + e], 0.0f);
            }
            int need = 0;  // by how much the row's unit rises
            if (!masked && rise) need = shift[m] - limit;
            if constexpr (masked) {
                const uint32_t seen = src.seen(m, tile), word = seen >> (4 * h);
                if (rise && seen) need = std::max(shift[m] - limit, 0);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(word & (1u << (8 * (i >> 2) + (i & 3))))) x[m][i] = -__builtin_inff();
            }
            float mx = x[m][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[m][i]);
            // neither -inf nor NaN raises the reference
            if (__any(__builtin_fmaf(mx, c[m], -top[m]) > LAZY || need > 0)) {
                mx = max_of_halves(mx) * c[m];
                const float ref = mx > top[m] ? mx : top[m];
                const float corr = exp2_(top[m] == ref ? -(float)need : top[m] - ref - (float)need);
                top[m] = ref;
                shift[m] -= need;
                sum[m] *= corr;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[m][d][i] *= corr;
            }
            const float base = (float)shift[m] - (top[m] == -__builtin_inff() ? 0.0f : top[m]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x4 v4 = *reinterpret_cast<const f16x4*>(&lds.t.vn[wave][8 * j + 4 * h]);
                float p[4], wt[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = exp2_(__builtin_fmaf(x[m][4 * j + e], c[m], base));
                    sum[m] += p[e];
                    wt[e] = __builtin_fmaf((float)v4[e], p[e], 0.0f);
                    if constexpr (masked) wt[e] = p[e] == 0.0f ? 0.0f : wt[e];  // a left-out token's norm may be anything
                }
                pf[m][j >> 1].u[2 * (j & 1)] = pack_f16(wt[0], wt[1]);
                pf[m][j >> 1].u[2 * (j & 1) + 1] = pack_f16(wt[2], wt[3]);
            }
            if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);
        }
        // ---- values, 16 tokens at a time: lane (token lane % 16, quarter lane / 16 of its dims), then V^T
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t y[8];
                PairTable<VB>::look_up(table, wv[ks], lane4, g, y);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    *reinterpret_cast<uint4*>(v8 + (lane & 15) * 256 + (((4 * (lane >> 4) + 2 * g + j) ^ swizzle(lane & 15)) << 4)) =
                        make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (ks == 1 && tile + step_tiles < tiles) load_values(tile + step_tiles);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                Frag vf;
#pragma unroll
                for (int e = 0; e < 2; ++e) vf.t[e] = read_tr(v8 + value_offset(d, e, lane));
#pragma unroll
                for (int m = 0; m < RB; ++m) o[m][d] = mfma_f16(vf, pf[m][ks], o[m][d]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    const int64_t whole = src.whole();
    for (; tile < whole; tile += step_tiles) step(tile, std::false_type{});
    for (; tile < tiles; tile += step_tiles) step(tile, std::true_type{});

    // ---- the waves' sums, one block of rows at a time.  What a wave's sums weigh is found once for a row, beside the sums' way to LDS (by every
    // thread of a row for itself a call took 0.8 us more)
    __syncthreads();
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        const float all = sum_of_halves(sum[m]);
        const float unit = __uint_as_float((uint32_t)(127 - shift[m]) << 23);
        if (h == 0) lds.s.ms[m][wave][r] = make_float2(top[m], all * unit), lds.s.unit[m][wave][r] = unit;
    }
    __syncthreads();
    if (wave == 0 && h < RB) {
        float2 ms[W];
        float best = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < W; ++k) ms[k] = lds.s.ms[h][k][r], best = fmaxf(best, ms[k].x);
        const float safe = best == -__builtin_inff() ? 0.0f : best;
        float den = 0.0f, by[W];
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float w = exp2_(ms[k].x - safe);
            by[k] = w * lds.s.unit[h][k][r];
            den = __builtin_fmaf(w, ms[k].y, den);
        }
#pragma unroll
        for (int k = 0; k < W; k += 4) lds.s.by[h][r][k / 4] = make_float4(by[k], by[k + 1], by[k + 2], by[k + 3]);
        if (32 * h + r < src.rows()) a.part_ms[src.partial() + 32 * h + r] = make_float2(best, den);
    }
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        if (m) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                lds.s.o[wave][r][(8 * d + 2 * j + h) ^ r] =
                    make_float4(o[m][d][4 * j], o[m][d][4 * j + 1], o[m][d][4 * j + 2], o[m][d][4 * j + 3]);
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * 32; i += N::T) {
            const int row = i >> 5, ch = i & 31;
            if (32 * m + row >= src.rows()) continue;
            float by[W];
#pragma unroll
            for (int k = 0; k < W; k += 4) *reinterpret_cast<float4*>(&by[k]) = lds.s.by[m][row][k / 4];
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float4 y = lds.s.o[k][row][ch ^ row];
                x.x = __builtin_fmaf(by[k], y.x, x.x), x.y = __builtin_fmaf(by[k], y.y, x.y);
                x.z = __builtin_fmaf(by[k], y.z, x.z), x.w = __builtin_fmaf(by[k], y.w, x.w);
            }
            reinterpret_cast<float4*>(a.part_o + (src.partial() + 32 * m + row) * D)[ch] = x;
        }
    }
}

// ------------------------------------------------------------------ merge

struct Merge {
    int64_t all_rows;
    const float* part_o;
    const float2* part_ms;
    const float* rv;
    float* out_f32;
    uint16_t* out_16;
    int is_f16;  // what out_16 holds; bf16 otherwise
    float* lse;
};
// A row's partials: split i's stands at `at` + i `step`, for i < n.
struct Part {
    int64_t at, step;
    int n;
};

// ROWS rows per workgroup: their splits weighed and added, then rotated back.  The matrix is read ahead of the partials,
// a quarter of its rows by a thread for its output dim.  `rows` says where a row's partials stand (find) and where its outputs
// go (place).
constexpr int MERGE_ROWS = 16, MERGE_T = 512, PARTS = MERGE_T / D, PART = D / PARTS;
template <int ROWS, class Rows>
__device__ __forceinline__ void merge_rows(const Merge& a, const Rows& rows) {
    __shared__ float s_w[ROWS][MAX_SPLIT];
    __shared__ float s_den[ROWS];
    __shared__ __align__(16) float s_o[ROWS][D];
    __shared__ float s_part[PARTS][ROWS][D];
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = threadIdx.x & 127, quarter = threadIdx.x >> 7;
    float m[PART];
#pragma unroll
    for (int d = 0; d < PART; ++d) m[d] = a.rv[(PART * quarter + d) * D + j];
    // 32 threads to a row and every SHARES-th of its splits, four dims each: the first splits' partials are on their way before the
    // weights are known
    constexpr int SHARES = MERGE_T / 32 / ROWS, AHEAD = 8 / SHARES;
    static_assert(SHARES <= PARTS, "the shares' sums fit s_part");
    const int pk = (threadIdx.x >> 5) / SHARES, share = (threadIdx.x >> 5) % SHARES, pc = threadIdx.x & 31;
    const Part mine = rows.find(std::min(row0 + pk, a.all_rows - 1));
    const float4* const part = reinterpret_cast<const float4*>(a.part_o + mine.at * D) + pc;
    const int64_t step4 = mine.step * (D / 4);
    float4 ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = share + SHARES * i < mine.n ? part[(share + SHARES * i) * step4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int k = wave; k < ROWS; k += MERGE_T / 64) {
        const int64_t row = row0 + k;
        float2 ms = make_float2(-__builtin_inff(), 0.0f);
        if (row < a.all_rows) {
            const Part p = rows.find(row);
            if (lane < p.n) ms = a.part_ms[p.at + lane * p.step];
        }
        float top = ms.x;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float w = exp2_(ms.x - (top == -__builtin_inff() ? 0.0f : top));
        float den = w * ms.y;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) den += __shfl_xor(den, x);
        s_w[k][lane] = w;
        if (lane == 0) {
            s_den[k] = den;
            if (a.lse && row < a.all_rows)
                a.lse[rows.place(row)] = den == 0.0f ? -__builtin_inff() : top * 0.6931471805599453f + __builtin_logf(den);
        }
    }
    __syncthreads();
    {
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](float w, float4 x) INLINE {
            o.x = __builtin_fmaf(w, x.x, o.x), o.y = __builtin_fmaf(w, x.y, o.y);
            o.z = __builtin_fmaf(w, x.z, o.z), o.w = __builtin_fmaf(w, x.w, o.w);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) add(s_w[pk][share + SHARES * i], ahead[i]);  // splits that there are not: 0 times 0
#pragma unroll 8
        for (int i = share + SHARES * AHEAD; i < mine.n; i += SHARES) add(s_w[pk][i], part[i * step4]);
        if constexpr (SHARES > 1) {
            *reinterpret_cast<float4*>(&s_part[share][pk][4 * pc]) = o;
            __syncthreads();
            if (share == 0)
#pragma unroll
                for (int i = 1; i < SHARES; ++i) add(1.0f, *reinterpret_cast<const float4*>(&s_part[i][pk][4 * pc]));
        }
        const float den = s_den[pk] == 0.0f ? 1.0f : s_den[pk];
        if (share == 0) *reinterpret_cast<float4*>(&s_o[pk][4 * pc]) = make_float4(o.x / den, o.y / den, o.z / den, o.w / den);
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < ROWS; ++k) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < PART; d += 4) {
            const float4 o = *reinterpret_cast<const float4*>(&s_o[k][PART * quarter + d]);
            x[0] = __builtin_fmaf(o.x, m[d], x[0]), x[1] = __builtin_fmaf(o.y, m[d + 1], x[1]);
            x[2] = __builtin_fmaf(o.z, m[d + 2], x[2]), x[3] = __builtin_fmaf(o.w, m[d + 3], x[3]);
        }
        s_part[quarter][k][j] = (x[0] + x[1]) + (x[2] + x[3]);
    }
    __syncthreads();
#pragma unroll 1
    for (int k = quarter; k < ROWS; k += PARTS) {
        const int64_t row = row0 + k;
        if (row >= a.all_rows) break;
        const float x = (s_part[0][k][j] + s_part[1][k][j]) + (s_part[2][k][j] + s_part[3][k][j]);
        const int64_t at = rows.place(row) * D + j;
        if (a.out_f32) a.out_f32[at] = x;
        if (a.out_16) a.out_16[at] = (uint16_t)(a.is_f16 ? tq::f32_to_f16(x) : tq::f32_to_bf16(x));
    }
}
}  // namespace tqt
