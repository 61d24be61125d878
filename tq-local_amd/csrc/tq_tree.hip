// tq_tree.hip -- attention of a tree of drafted tokens over the packed TurboQuant cache (gfx950).
//
// T <= 64 drafted tokens (nodes) of each sequence stand packed in the slots behind its history.  Node i
// attends to the history, to its ancestors and to itself:
//   logit_t = scale (|k_t| <q R_k^T, C_k[kidx_t]> + sqrt(pi/2)/D |r_t| <q S^T, s_t>)
//   out     = (sum_t softmax_t |v_t| C_v[vidx_t]) R_v
// so keys and values are never rotated: the queries are, once, and the sums are rotated back, once.
//
//   tree_kernel   a share of the tokens of one KV head per workgroup of eight waves, and 32 query rows (head x node) or 64 of
//                 them, all in every wave.  It rotates its queries first (q R_k^T and q S^T, scaled by a power of two per row, to
//                 fp16 operands), then the waves take tiles of 32 tokens in turn, on their own until their sums meet:
//                 S^T = K Q^T (codes and signs apart: their norms differ) and O^T = V^T P^T with v_mfma_f32_32x32x16_f16.
//                 The splits of a head fill the CUs, with eight tiles at least; batch rows of different lengths share them out
//   merge_kernel  the splits' partials of a row weighed and added, rotated back by R_v
//
// Codes to fp16.  Keys become A operands in registers, a lane's token and half of its dims: a byte lookup (v_perm_b32) of the
// centroid's two halves for four codes at once.  Which four codes meet in a register follows from the packing (those at the
// same bits of neighbouring bytes), so each bit width has an order of the 128 dims of its own, which the queries are
// written in (position_of).  Signs stay where they are, as the lowest mantissa bits of fp16 numbers.  Values are looked up in LDS, two
// codes at a time (PairTable), and turned around by ds_read_b64_tr_b16.
//
// Cost.  The tiles are bound by their decoding and their softmax beside the matrix instructions: 16 nodes x 4 heads of 8
// sequences of 32768 tokens (8 KV heads, 4-bit Q_prod) take 151 us, of which the matrix instructions are 78 at the rate of a
// large product of matrices, the 281 MB of codes 55 at that of a large copy; 64 rows to a workgroup share a tile's decoding
// (the call took 182 us with 32 and 32 when it took 160 with 64).  64 nodes x 7 heads of 4 sequences of 8192 (4 KV heads, 3-bit
// Q_mse) take 67 us.
// Small calls are bound by latency: 8 nodes of one chat of 1037 tokens take 13 us and the merge 7, of which the first bytes
// from memory are 4, and two launches.  Rotating the queries in a kernel of their own took 9 us more a call and saved 5.
//
// Rounding.  Rotated queries and centroids are rounded once to fp16, by at most 2^-11 of each, 2^-11 / sqrt(3) root mean square (with
// |q| = 11 and |k| = 20 a logit moves by 7e-4), value centroids too (their sum's errors are kept from adding up by the
// codebook, see tq_value_codebook_f16), weights times norm p |v| once: to 11 bits down to 2^-25 of the largest norm's at the row's
// reference, and by up to 2^-36 of it below.  Logits, maxima, weights, sums and outputs are fp32.

#include <algorithm>
#include <type_traits>

#include "tq_rows16.h"

namespace {

using namespace tqr;

constexpr int D = TQ_DIM;
constexpr int TK = 32;         // tokens per tile
constexpr int MIN_TILES = 8;   // tiles of a split
constexpr int MAX_SPLIT = 64;  // partials a merge wave weighs with one lane each
constexpr float LOG2E = 1.44269504f;
// Log2 that a score may exceed its row's reference by, and of the largest weight times norm at the reference: 15 together, what fp16
// holds.  The less a score may exceed it the smaller the weights that keep their bits, and the more often references rise: with 4 the
// calls of the header, with their merges, take 159 and 71 us, with 8 156 and 69, with 2 160 and 72
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
__device__ __forceinline__ f32x16 fill16(float x) {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = x;
    return z;
}
__device__ __forceinline__ f32x16 zero16() { return fill16(0.0f); }

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

// Four chunks of 8 elements from 32 codes (BITS words), in the order of position_of.
template <int BITS>
__device__ __forceinline__ void expand32(const uint32_t* w, const Lut<BITS>& lut, uint4* out) {
    uint32_t q[8];
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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lut.four(q[2 * j], out[j].x, out[j].y);
        lut.four(q[2 * j + 1], out[j].z, out[j].w);
    }
}

// Four chunks from 32 sign bits, left where they are: bits i and i + 16 of the word (or of the word moved down by 8,
// for i = 8..15) as the lowest mantissa bits of two fp16 numbers, 2^(p - 24) with p = i mod 8 for a set bit and 0 for a
// clear one (the matrix cores keep subnormals).  The queries carry the 2^(7 - p), and sum_i s_i x_i = 2 sum_i bit_i x_i -
// sum_i x_i.
__device__ __forceinline__ void expand_signs(uint32_t w, uint4* out) {
    const uint32_t v = w >> 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (j < 2 ? w : v) & (0x00010001u << ((4 * j + k) & 7));
        out[j] = make_uint4(x[0], x[1], x[2], x[3]);
    }
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

struct TreeArgs {
    int batch, kv_heads, T, rows;
    const int32_t* parents;
    int64_t parents_sb;
    const int32_t *starts, *lens;
    int64_t n_tokens, cap;
    const uint8_t *k_codes, *k_signs, *v_codes;
    const uint16_t *k_norms, *k_rnorms, *v_norms;
    const float *key_centers, *value_centers;
    const void* q;
    int q_type, group;  // query heads per KV head
    int64_t q_sb, q_sh, q_st;
    const float *rk, *s;
    float c2;  // scale log2(e)
    int n_split, n_slots;  // n_split slots for each batch row, or n_slots dealt out by what the rows have
    float* part_o;         // [slot][kv head][row][D]
    float2* part_ms;       // [slot][kv head][row] (reference of the weights in log2, sum of weights)
    int2* slots;           // [batch] a batch row's first slot and its number of slots, for rows of different lengths
};

// What a batch row attends to: history [lo, end), drafted tokens up to stop.
struct Range {
    int lo, end, stop;
};
// of a row's entries in starts and lens (any number where there are none)
__device__ __forceinline__ Range range_of(const TreeArgs& a, int start, int len) {
    const int nodes = a.parents ? a.T : 0, n = (int)a.n_tokens;
    const int end = std::min(std::max(a.lens ? len : n - nodes, 0), n);
    const int lo = a.starts ? std::min(std::max(start, 0), end) : 0;
    return {lo, end, (int)std::min<int64_t>((int64_t)end + nodes, n)};
}
__device__ __forceinline__ int tiles_of(const Range& r) { return (int)(((int64_t)r.stop - r.lo + TK - 1) / TK); }

// The batch row of a slot, its first slot and its number of slots.  Up to 64 rows of different lengths share the slots in
// proportion to their tiles, each with one at least; what is left over goes unused (b = -1).
struct Slot {
    int b, first, n;
    Range range;
};
// `start`, `len`: the entries of batch row `lane`.
__device__ __forceinline__ Slot find_slot(const TreeArgs& a, int slot, int start, int len) {
    const Range mine = range_of(a, start, len);
    const int tiles = tiles_of(mine);
    int total = 0;
    for (int i = 0; i < a.batch; ++i) total += __builtin_amdgcn_readlane(tiles, i);
    // (the sum of the shares does not pass what there is to share, whatever the roundings: these are far below 1)
    const int share = (int)((float)(a.n_slots - a.batch) * ((float)tiles / (float)std::max(total, 1)));
    const int n = std::min(std::min(1 + share, std::max(1, (tiles + MIN_TILES - 1) / MIN_TILES)), MAX_SPLIT);
    int before = 0;
    for (int i = 0; i < a.batch; ++i) {
        const int own = __builtin_amdgcn_readlane(n, i);
        if (slot < before + own)
            return {i, before, own, {__builtin_amdgcn_readlane(mine.lo, i), __builtin_amdgcn_readlane(mine.end, i),
                                     __builtin_amdgcn_readlane(mine.stop, i)}};
        before += own;
    }
    return {-1, 0, 0, {0, 0, 0}};
}

__device__ __forceinline__ float query_element(const TreeArgs& a, int64_t i) {
    return a.q_type == 1 ? static_cast<const float*>(a.q)[i] : tq::f16_to_f32(static_cast<const uint16_t*>(a.q)[i]);
}

// Bit j of a node's mask: node j is the node itself or one of its ancestors.  A parent that is not an earlier
// node is none.  Called by one whole wave, lane = node, with the node's parent.
__device__ __forceinline__ uint64_t ancestors(int p, int lane) {
    if (p < 0 || p >= lane) p = -1;
    uint64_t mask = 1ull << lane;
#pragma unroll
    for (int k = 0; k < 6; ++k) {  // paths of 2^k steps
        const uint64_t up = __shfl(mask, p < 0 ? 0 : p);
        const int next = __shfl(p, p < 0 ? 0 : p);
        if (p >= 0) mask |= up, p = next;
    }
    return mask;
}

// The tokens of a tile that a node attends to, as bits: those of the history (the first `to_end` of the tile, none
// if it is negative), the nodes behind it that `sees` names, and none from `left` on.
__device__ __forceinline__ uint32_t seen_of_tile(uint64_t sees, int to_end, int left) {
    const uint64_t nodes = to_end >= TK || to_end <= -64 ? 0ull : to_end >= 0 ? sees << to_end : sees >> -to_end;
    const uint64_t history = to_end <= 0 ? 0ull : (1ull << std::min(to_end, TK)) - 1;
    return (uint32_t)((nodes | history) & ((1ull << std::min(left, TK)) - 1));
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
template <int RB>
struct Tree {
    static constexpr int W = 8;
    static constexpr int T = 64 * W;
    struct Tiles {
        uint32_t table[256 * 64];
        uint4 v[W][16 * 16];
        // the rows' operands for the signs and for the codes (these go on to registers with one block of rows; two do not fit)
        uint4 qs[RB][8 * 64], qc[RB][8 * 64];
        uint16_t kn[W][32], vn[W][32];
        float ratio[W][32];
    };
    struct Sums {
        float4 o[W][32][32];  // chunks xor-swizzled by the row
        float2 ms[W][32];
        float unit[W];
    };
    union Lds {
        uint4 m[2 * 128 * 32];
        Tiles t;
        Sums s;
    };
};

template <int KB, int VB, bool QJL, int RB, int NQ>
__global__ __launch_bounds__(Tree<RB>::T, 2) void tree_kernel(TreeArgs a) {
    using N = Tree<RB>;
    constexpr int W = N::W;
    __shared__ typename N::Lds lds;
    __shared__ uint64_t s_anc[64];
    __shared__ float s_centers[1 << VB];
    __shared__ float s_top[W][32], s_sum[RB][4][32], s_c[RB][32];
    int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // in a scalar register, and what follows from it
    const int kvh = blockIdx.y, row_group = RB == 1 ? 0 : blockIdx.x / a.n_slots, slot = blockIdx.x - row_group * a.n_slots;
    // (known before the matrices are asked for: a wait for a load ahead of theirs is one for them all)
    Slot mine;
    if (a.slots) {
        const int entry = std::min(lane, a.batch - 1);
        mine = find_slot(a, slot, a.starts ? a.starts[entry] : 0, a.lens ? a.lens[entry] : 0);
        if (mine.b < 0) return;
    } else {
        using Scalar = const __attribute__((address_space(4))) int32_t*;
        const int b = slot % a.batch;
        mine = {b, 0, a.n_split, range_of(a, a.starts ? ((Scalar)a.starts)[b] : 0, a.lens ? ((Scalar)a.lens)[b] : 0)};
    }
    // ---- What the queries' rotation takes is asked for first, then a first tile of the cache, then the small things: a workgroup of a
    // short history waits for memory once.  The matrices come by way of LDS: read straight into operands, 32 rows at a time, they
    // were 10000 cycles on their way.  Their 16-byte chunks are xor-swizzled by the row
#pragma unroll
    for (int i = 0; i < (QJL ? 16 : 8); ++i) {  // 64 chunks, two rows, a time
        const int at = (8 * i + wave) * 64 + lane, row = (at >> 5) & 127;
        load_lds16((i < 8 ? a.rk : a.s) + row * D + 4 * ((at & 31) ^ (row & 31)), &lds.m[(8 * i + wave) * 64]);
    }
    // without slots of its own a batch row has every batch-th
    const int b = mine.b, kv = b * a.kv_heads + kvh, split = a.slots ? slot - mine.first : slot / a.batch, n_split = mine.n;
    if (a.slots && split == 0 && row_group == 0 && kvh == 0 && threadIdx.x == 0) a.slots[b] = make_int2(mine.first, mine.n);
    Frag x[8][NQ];  // a block's queries: lane (r, h) has row r's dims 16 s + 8 h + (0..7)
    auto load_queries = [&](int m) INLINE {
        const int row = 32 * (row_group * RB + m) + r;
        const bool live = row < a.rows;
        const uint32_t g = live ? (uint32_t)row / (uint32_t)a.T : 0u, t = live ? row - g * a.T : 0u;
        const int64_t at = b * a.q_sb + (int64_t)(kvh * a.group + g) * a.q_sh + t * a.q_st + 8 * h;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if constexpr (NQ == 1) {
                __builtin_memcpy(&x[s][0], static_cast<const uint16_t*>(a.q) + at + 16 * s, 16);  // rows past the last: some row
            } else {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = query_element(a, at + 16 * s + e);
                split_terms<NQ>(y, x[s]);
            }
        }
    };
    load_queries(0);

    const int nodes = a.parents ? a.T : 0;
    const int64_t lo = mine.range.lo, end = mine.range.end, stop = mine.range.stop, tiles = tiles_of(mine.range);
    const int step_tiles = n_split * W;  // tiles in turn, to the waves of all splits

    // a lane's part of a tile, on its way: half of token r's key codes and signs and its norms, and a quarter of the value
    // codes of tokens lane % 16 and lane % 16 + 16.  The arrays are at scalar addresses, a lane's place in them 32-bit
    // offsets; tokens past the last are copies of it, left out by the mask
    uint32_t wk[2 * KB], ws[2], wv[2][VB];
    uint16_t kn, rn = 0, vn;
    auto load_keys = [&](int64_t tile) {
        const int64_t t0 = lo + tile * TK, slot = (int64_t)kv * a.cap + t0;
        const uint32_t tok = std::min<uint32_t>(r, (uint32_t)std::min<int64_t>(stop - t0, TK) - 1);
        __builtin_memcpy(wk, __builtin_assume_aligned(a.k_codes + slot * (16 * KB) + (tok * (16 * KB) + 8 * KB * h), 8), 8 * KB);
        if constexpr (QJL) {
            __builtin_memcpy(ws, __builtin_assume_aligned(a.k_signs + slot * 16 + (tok * 16 + 8 * h), 8), 8);
            rn = (a.k_rnorms + slot)[tok];
        }
        kn = (a.k_norms + slot)[tok], vn = (a.v_norms + slot)[tok];
    };
    auto load_values = [&](int64_t tile) {
        const int64_t t0 = lo + tile * TK, slot = (int64_t)kv * a.cap + t0;
        const uint32_t last = (uint32_t)std::min<int64_t>(stop - t0, TK) - 1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t tok = std::min<uint32_t>((lane & 15) + 16 * x, last);
            __builtin_memcpy(wv[x], __builtin_assume_aligned(a.v_codes + slot * (16 * VB) + (tok * (16 * VB) + 4 * VB * (lane >> 4)), 4),
                             4 * VB);
        }
    };
    int64_t tile = split * W + wave;
    if (RB == 1 && tile < tiles) load_keys(tile), load_values(tile);
    float key_center[1 << KB];
#pragma unroll
    for (int i = 0; i < (1 << KB); ++i) key_center[i] = a.key_centers[i];
    float value_center = 0.0f;
    if (threadIdx.x < (1 << VB)) value_center = a.value_centers[threadIdx.x];
    int parent = -1;
    if (nodes && wave == 0 && lane < a.T) parent = a.parents[b * a.parents_sb + lane];
    __builtin_amdgcn_sched_barrier(0);

    wait_loads();
    __syncthreads();
    // a wave has 32 output dims of one of the matrices
    const int mat = wave >> 2, j0 = 32 * (wave & 3);
    const bool works = QJL || mat == 0;
    float mrow[8][8];
    if (works) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                __builtin_memcpy(&mrow[s][4 * e], &lds.m[(128 * mat + j0 + r) * 32 + ((4 * s + 2 * h + e) ^ r)], 16);
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
                for (int s = 0; s < 8; ++s) {
                    Frag mt[2];
                    split_terms<2>(mrow[s], mt);
#pragma unroll
                    for (int i = 1; i >= 0; --i)
#pragma unroll
                        for (int j = NQ - 1; j >= 0; --j)
                            if (i + j <= 1) acc = mfma_bf16(mt[i], x[s][j], acc);
                }
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
                uint8_t* const to = reinterpret_cast<uint8_t*>(lds.t.qc[m]) + operand_offset(position_of<KB>(j0 + 4 * h)) + 16 * r;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] *= up;
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
    if (nodes && wave == 0) s_anc[lane] = ancestors(parent, lane);
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
    uint64_t sees[RB];
#pragma unroll
    for (int m = 0; m < RB; ++m) sees[m] = nodes ? s_anc[(32 * (row_group * RB + m) + r) % a.T] : 0ull;
    __syncthreads();

    f32x16 o[RB][4];
    float top[RB], sum[RB];  // `top` is a weight's reference, raised when a score is more than 2^LAZY above it
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        top[m] = -__builtin_inff(), sum[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[m][d] = zero16();
    }
    // weights and output sums are in units of 2^-shift, 2^-TOP_BIT of a power of two above the largest |v| so far: weights
    // times norm then reach up to 2^(TOP_BIT + LAZY), and fp16 keeps its 11 bits down to 2^-14, 2^-25 of the reference's
    int shift = TOP_BIT + 24;
    const uint32_t lane4 = (lane & 31) * 4;
    const uint8_t* const table = reinterpret_cast<const uint8_t*>(lds.t.table);
    uint8_t* const v8 = reinterpret_cast<uint8_t*>(lds.t.v[wave]);

    auto step = [&](int64_t tile, auto nodes_here) {
        const int64_t t0 = lo + tile * TK;
        const int left = (int)std::min<int64_t>(stop - t0, TK);
        const uint32_t norm = !nodes_here || r < left ? vn : 0u;  // tokens past the last weigh nothing
        if (h == 0) {
            // a key's norm that fp16 holds as 0 counts as 2^-24, its least
            const uint16_t k = QJL && (kn & 0x7FFFu) == 0 ? 1 : kn;
            lds.t.kn[wave][r] = k;
            lds.t.vn[wave][r] = (uint16_t)norm;
            // |r| / |k|, in the units of the sign products
            if constexpr (QJL) lds.t.ratio[wave][r] = tq::f16_to_f32(rn) * 0x1p18f / tq::f16_to_f32(k);
        }
        // ---- scores: |k| (<codes> + |r| / |k| <signs>), the sign products' sums going into the codes'
        f32x16 x[RB];
#pragma unroll
        for (int m = 0; m < RB; ++m) x[m] = zero16();
        if constexpr (QJL) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint4 f[4];
                expand_signs(ws[u], f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    Frag kf, qf;
                    kf.q = f[j];
#pragma unroll
                    for (int m = 0; m < RB; ++m) {
                        qf.q = lds.t.qs[m][(4 * u + j) * 64 + lane];
                        x[m] = mfma_f16(kf, qf, x[m]);
                    }
                }
                if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);  // the registers hold a few operands at a time
            }
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
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint4 f[4];
            expand32<KB>(wk + KB * u, klut, f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                Frag kf, qf;
                kf.q = f[j];
#pragma unroll
                for (int m = 0; m < RB; ++m) {
                    if constexpr (RB > 1) qf.q = lds.t.qc[m][(4 * u + j) * 64 + lane];
                    x[m] = mfma_f16(kf, RB > 1 ? qf : q[4 * u + j], x[m]);
                }
            }
            if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);
        }
        // the largest finite |v| of the tile: its exponent decides the unit (2^(e + 1) is above it)
        const int e5 = (norm >> 10) & 31, ve = e5 == 31 ? 0 : e5;
        int need = 0;  // uniform: by how much the unit has to rise
        if (__any(ve > 14 + TOP_BIT - shift)) {
            int e = 0;
            uint64_t largest = ~0ull;
#pragma unroll
            for (int k = 4; k >= 0; --k) {
                const uint64_t set = __ballot(ve >> k & 1) & largest;
                if (set) largest = set, e |= 1 << k;
            }
            need = shift - (14 + TOP_BIT - std::max(e, 1));
        }
        shift -= need;
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
            if constexpr (nodes_here) {
                const int to_end = (int)std::max<int64_t>(std::min<int64_t>(end - t0, TK), -64);
                const uint32_t word = seen_of_tile(sees[m], to_end, left) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(word & (1u << (8 * (i >> 2) + (i & 3))))) x[m][i] = -__builtin_inff();
            }
            float mx = x[m][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[m][i]);
            // neither -inf nor NaN raises the reference
            if (__any(__builtin_fmaf(mx, c[m], -top[m]) > LAZY) || need) {
                mx = max_of_halves(mx) * c[m];
                const float ref = mx > top[m] ? mx : top[m];
                const float corr = exp2_(top[m] == ref ? -(float)need : top[m] - ref - (float)need);
                top[m] = ref;
                sum[m] *= corr;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[m][d][i] *= corr;
            }
            const float base = (float)shift - (top[m] == -__builtin_inff() ? 0.0f : top[m]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f16x4 v4 = *reinterpret_cast<const f16x4*>(&lds.t.vn[wave][8 * j + 4 * h]);
                float p[4], wt[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = exp2_(__builtin_fmaf(x[m][4 * j + e], c[m], base));
                    sum[m] += p[e];
                    wt[e] = __builtin_fmaf((float)v4[e], p[e], 0.0f);
                    if constexpr (nodes_here) wt[e] = p[e] == 0.0f ? 0.0f : wt[e];  // a left-out token's norm may be anything
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
    // whole tiles of the history, then those with the end of it or drafted tokens in them
    const int64_t whole = std::min(tiles, (end - lo) / TK);
    for (; tile < whole; tile += step_tiles) step(tile, std::false_type{});
    for (; tile < tiles; tile += step_tiles) step(tile, std::true_type{});

    // ---- the waves' sums, one block of rows at a time
    const float unit = __uint_as_float((uint32_t)(127 - shift) << 23);
#pragma unroll
    for (int m = 0; m < RB; ++m) {
        __syncthreads();
        const float all = sum_of_halves(sum[m]);
        if (h == 0) lds.s.ms[wave][r] = make_float2(top[m], all * unit);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                lds.s.o[wave][r][(8 * d + 2 * j + h) ^ r] =
                    make_float4(o[m][d][4 * j], o[m][d][4 * j + 1], o[m][d][4 * j + 2], o[m][d][4 * j + 3]);
        if (lane == 0) lds.s.unit[wave] = unit;
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * 32; i += N::T) {
            const int row = i >> 5, ch = i & 31, out_row = 32 * (row_group * RB + m) + row;
            if (out_row >= a.rows) continue;
            float best = -__builtin_inff();
#pragma unroll
            for (int k = 0; k < W; ++k) best = fmaxf(best, lds.s.ms[k][row].x);
            const float safe = best == -__builtin_inff() ? 0.0f : best;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float den = 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const float2 ms = lds.s.ms[k][row];
                const float w = exp2_(ms.x - safe), wu = w * lds.s.unit[k];
                const float4 y = lds.s.o[k][row][ch ^ row];
                den = __builtin_fmaf(w, ms.y, den);
                x.x = __builtin_fmaf(wu, y.x, x.x), x.y = __builtin_fmaf(wu, y.y, x.y);
                x.z = __builtin_fmaf(wu, y.z, x.z), x.w = __builtin_fmaf(wu, y.w, x.w);
            }
            const int64_t at = ((int64_t)slot * a.kv_heads + kvh) * a.rows + out_row;
            reinterpret_cast<float4*>(a.part_o + at * D)[ch] = x;
            if (ch == 0) a.part_ms[at] = make_float2(best, den);
        }
    }
}

// ------------------------------------------------------------------ merge

struct MergeArgs {
    int q_heads, kv_heads, T, rows, n_split;
    int64_t all_rows;  // of all KV heads
    const float* part_o;
    const float2* part_ms;
    const int2* slots;  // or n_split for every batch row
    const float* rv;
    float* out_f32;
    uint16_t* out_bf16;
    float* lse;
};

// MERGE_ROWS rows per workgroup: their splits weighed and added, then rotated back.  The matrix is read ahead of the partials,
// a quarter of its rows by a thread for its output dim.
constexpr int MERGE_ROWS = 16, MERGE_T = 512, PARTS = MERGE_T / D, PART = D / PARTS;
__global__ __launch_bounds__(MERGE_T) void merge_kernel(MergeArgs a) {
    __shared__ float s_w[MERGE_ROWS][MAX_SPLIT];
    __shared__ float s_den[MERGE_ROWS];
    __shared__ __align__(16) float s_o[MERGE_ROWS][D];
    __shared__ float s_part[PARTS][MERGE_ROWS][D];
    const int64_t row0 = (int64_t)blockIdx.x * MERGE_ROWS;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = threadIdx.x & 127, quarter = threadIdx.x >> 7;
    float m[PART];
#pragma unroll
    for (int d = 0; d < PART; ++d) m[d] = a.rv[(PART * quarter + d) * D + j];
    // split i of a row is at `at` + i step
    struct Part {
        int64_t at;
        int n;
    };
    const int64_t step = a.slots ? (int64_t)a.kv_heads * a.rows : a.all_rows;
    auto find = [&](int64_t row) INLINE {
        if (!a.slots) return Part{row, a.n_split};
        const uint32_t n = (uint32_t)row, b = n / ((uint32_t)a.kv_heads * (uint32_t)a.rows);
        const int2 slots = a.slots[b];
        return Part{(slots.x - (int64_t)b) * step + row, slots.y};
    };
    // 32 threads to a row, four dims each: the first splits' partials are on their way before the weights are known
    constexpr int AHEAD = 8;
    const int pk = threadIdx.x >> 5, pc = threadIdx.x & 31;
    const Part mine = find(std::min(row0 + pk, a.all_rows - 1));
    const float4* const part = reinterpret_cast<const float4*>(a.part_o + mine.at * D) + pc;
    const int64_t step4 = step * (D / 4);
    float4 ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = i < mine.n ? part[i * step4] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto place = [&](int64_t row) {  // of a row in [batch][q heads][T]
        const uint32_t n = (uint32_t)row, kv = n / (uint32_t)a.rows, in = n - kv * a.rows, g = in / (uint32_t)a.T;
        const uint32_t b = kv / (uint32_t)a.kv_heads, hq = (kv - b * a.kv_heads) * (a.q_heads / a.kv_heads) + g;
        return ((int64_t)b * a.q_heads + hq) * a.T + (in - g * a.T);
    };
#pragma unroll 1
    for (int k = wave; k < MERGE_ROWS; k += MERGE_T / 64) {
        const int64_t row = row0 + k;
        float2 ms = make_float2(-__builtin_inff(), 0.0f);
        if (row < a.all_rows) {
            const Part p = find(row);
            if (lane < p.n) ms = a.part_ms[p.at + lane * step];
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
                a.lse[place(row)] = den == 0.0f ? -__builtin_inff() : top * 0.6931471805599453f + __builtin_logf(den);
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
        for (int i = 0; i < AHEAD; ++i) add(s_w[pk][i], ahead[i]);  // splits that there are not: 0 times 0
#pragma unroll 8
        for (int i = AHEAD; i < mine.n; ++i) add(s_w[pk][i], part[i * step4]);
        const float den = s_den[pk] == 0.0f ? 1.0f : s_den[pk];
        *reinterpret_cast<float4*>(&s_o[pk][4 * pc]) = make_float4(o.x / den, o.y / den, o.z / den, o.w / den);
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < MERGE_ROWS; ++k) {
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
    for (int k = quarter; k < MERGE_ROWS; k += PARTS) {
        const int64_t row = row0 + k;
        if (row >= a.all_rows) break;
        const float x = (s_part[0][k][j] + s_part[1][k][j]) + (s_part[2][k][j] + s_part[3][k][j]);
        const int64_t at = place(row) * D + j;
        if (a.out_f32) a.out_f32[at] = x;
        if (a.out_bf16) a.out_bf16[at] = (uint16_t)tq::f32_to_bf16(x);
    }
}

struct Plan {
    int rows, row_blocks, n_split, n_slots;
    unsigned row_groups;
    int64_t heads;
    size_t ms_bytes, o_bytes, slots_bytes;
    size_t total() const { return ms_bytes + o_bytes + slots_bytes; }
};

// A workgroup fills a CU.  As many splits as fill the CUs, as long as none is left without a tile.
bool make_plan(int batch, int q_heads, int kv_heads, int T, int64_t n_tokens, Plan& p) {
    const int64_t rows = (int64_t)(q_heads / kv_heads) * T;
    p.heads = (int64_t)batch * kv_heads;
    if (p.heads > 65535 || p.heads * rows >= (int64_t)1 << 26 || rows > 65535 * 32) return false;
    p.rows = (int)rows;
    p.row_blocks = (p.rows + 31) / 32;
    p.row_groups = p.row_blocks == 1 ? 1 : (unsigned)(p.row_blocks + 1) / 2;
    const int64_t tiles = std::max<int64_t>(1, (n_tokens + TK - 1) / TK);
    const int64_t most = std::min<int64_t>((tiles + MIN_TILES - 1) / MIN_TILES, MAX_SPLIT);
    p.n_split = (int)std::max<int64_t>(1, std::min<int64_t>(256 / (p.heads * p.row_groups), most));
    // batch rows of different lengths share out what fills the CUs
    p.n_slots = (int)std::max<int64_t>((int64_t)p.n_split * batch,
                                       std::min<int64_t>(256 / (kv_heads * (int64_t)p.row_groups), most * batch));
    p.ms_bytes = ((size_t)p.n_slots * kv_heads * rows * 8 + 15) / 16 * 16;
    p.o_bytes = (size_t)p.n_slots * kv_heads * rows * D * 4;
    p.slots_bytes = ((size_t)batch * 8 + 15) / 16 * 16;
    return true;
}

template <int KB, int VB, bool QJL>
void launch_tree(const TreeArgs& a, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)a.n_slots * p.row_groups, (unsigned)a.kv_heads);
    auto launch = [&](auto rb, auto nq) {
        hipLaunchKernelGGL((tree_kernel<KB, VB, QJL, rb, nq>), grid, dim3(Tree<rb>::T), 0, s, a);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (p.row_blocks == 1) a.q_type == 0 ? launch(One{}, One{}) : launch(One{}, Two{});
    else a.q_type == 0 ? launch(Two{}, One{}) : launch(Two{}, Two{});
}

}  // namespace

extern "C" size_t tq_tree_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int nodes, int dim,
                                                    int64_t n_tokens) {
    Plan p;
    if (batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || nodes < 1 || nodes > TQ_MAX_NODES || dim != D ||
        n_tokens < 0 || !make_plan(batch, q_heads, kv_heads, nodes, n_tokens, p))
        return 0;
    return p.total();
}

extern "C" int tq_tree_attention(const void* q, int q_type, int batch, int q_heads, int kv_heads, int nodes, int dim,
                                 int64_t q_sb, int64_t q_sh, int64_t q_st, const int32_t* parents, int64_t parents_sb,
                                 const int32_t* seq_starts, const int32_t* seq_lens, int64_t n_tokens, int64_t cap,
                                 const uint8_t* k_codes, const uint16_t* k_norms, const uint8_t* k_signs,
                                 const uint16_t* k_rnorms, const uint8_t* v_codes, const uint16_t* v_norms, int key_bits,
                                 int value_bits, int has_qjl, const float* key_rotation, const float* key_centers,
                                 const float* qjl, const float* value_rotation, const float* value_centers, float scale,
                                 float* out_f32, uint16_t* out_bf16, float* lse_out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    if (!q || q_type < 0 || q_type > 2 || batch < 1 || q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || nodes < 1 ||
        n_tokens < 0 || n_tokens > cap || cap < 1 || !k_codes || !k_norms || !v_codes || !v_norms || !key_rotation ||
        !key_centers || !value_rotation || !value_centers || (has_qjl && (!k_signs || !k_rnorms || !qjl)) ||
        (!out_f32 && !out_bf16) || !(scale > 0.0f) || scale == __builtin_inff())
        return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D || nodes > TQ_MAX_NODES || n_tokens >= (int64_t)1 << 31 || value_bits < 1 || value_bits > 4 || key_bits < 1 ||
        key_bits != value_bits - (has_qjl ? 1 : 0))
        return TQ_ERR_UNSUPPORTED;
    if (!aligned16(key_rotation) || !aligned16(k_codes) || !aligned16(v_codes) || (has_qjl && (!aligned16(k_signs) || !aligned16(qjl))))
        return TQ_ERR_UNSUPPORTED;
    Plan p;
    if (!make_plan(batch, q_heads, kv_heads, nodes, n_tokens, p)) return TQ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.total() || !aligned16(workspace)) return TQ_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    float* part_o = reinterpret_cast<float*>(ws);
    float2* part_ms = reinterpret_cast<float2*>(ws + p.o_bytes);
    const bool ragged = batch > 1 && batch <= 64 && p.n_slots > batch && (seq_starts || seq_lens);
    int2* const slots = ragged ? reinterpret_cast<int2*>(ws + p.o_bytes + p.ms_bytes) : nullptr;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const TreeArgs a{batch, kv_heads, nodes, p.rows, parents, parents_sb, seq_starts, seq_lens, n_tokens, cap,
                     k_codes, k_signs, v_codes, k_norms, k_rnorms, v_norms, key_centers, value_centers, q, q_type, q_heads / kv_heads,
                     q_sb, q_sh, q_st, key_rotation, qjl, scale * LOG2E, p.n_split, slots ? p.n_slots : p.n_split * batch, part_o, part_ms,
                     slots};
    if (has_qjl) {
        if (value_bits == 4) launch_tree<3, 4, true>(a, p, s);
        else if (value_bits == 3) launch_tree<2, 3, true>(a, p, s);
        else launch_tree<1, 2, true>(a, p, s);
    } else {
        if (value_bits == 4) launch_tree<4, 4, false>(a, p, s);
        else if (value_bits == 3) launch_tree<3, 3, false>(a, p, s);
        else if (value_bits == 2) launch_tree<2, 2, false>(a, p, s);
        else launch_tree<1, 1, false>(a, p, s);
    }
    TQ_CHECK_LAUNCH();
    const int64_t all = p.heads * p.rows;
    const MergeArgs m{q_heads, kv_heads, nodes, p.rows, p.n_split, all, part_o, part_ms, slots, value_rotation, out_f32, out_bf16,
                      lse_out};
    hipLaunchKernelGGL(merge_kernel, dim3((unsigned)((all + MERGE_ROWS - 1) / MERGE_ROWS)), dim3(MERGE_T), 0, s, m);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
