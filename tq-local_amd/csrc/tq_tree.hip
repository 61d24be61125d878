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
// Cost.  The tiles are bound by their decoding and their softmax beside the matrix instructions: 16 nodes x 4 heads of 8
// sequences of 32768 tokens (8 KV heads, 4-bit Q_prod) take 151 us, of which the matrix instructions are 78 at the rate of a
// large product of matrices, the 281 MB of codes 55 at that of a large copy; 64 rows to a workgroup share a tile's decoding
// (the call took 182 us with 32 and 32 when it took 160 with 64).  64 nodes x 7 heads of 4 sequences of 8192 (4 KV heads, 3-bit
// Q_mse) take 67 us.
// Small calls are bound by latency: 8 nodes of one chat of 1037 tokens take 13 us and the merge 7, of which the first bytes
// from memory are 4, and two launches.  Rotating the queries in a kernel of their own took 9 us more a call and saved 5.

#include "tq_tiles.h"

namespace {

using namespace tqt;

struct TreeArgs {
    int batch, kv_heads, T, rows;
    const int32_t* parents;
    int64_t parents_sb;
    const int32_t *starts, *lens;
    int64_t n_tokens, cap;
    Cache c;
    int group;  // query heads per KV head
    int64_t q_sb, q_sh, q_st;
    int n_split, n_slots;  // n_split slots for each batch row, or n_slots dealt out by what the rows have
    int2* slots;  // [batch] a batch row's first slot and its number of slots, for rows of different lengths
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

// 32 RB rows of a KV head: rows head by head, a head's nodes next to one another.
template <int RB>
struct TreeSource {
    const TreeArgs& a;
    uint64_t* const s_anc;
    const Slot& mine;
    const int slot, kvh, row0, nodes, kv, split_, n_split;
    int parent = -1;
    uint64_t sees[RB];

    __device__ __forceinline__ TreeSource(const TreeArgs& a, uint64_t* s_anc, const Slot& mine, int slot, int kvh, int row_group)
        : a(a), s_anc(s_anc), mine(mine), slot(slot), kvh(kvh), row0(32 * RB * row_group), nodes(a.parents ? a.T : 0),
          // without slots of its own a batch row has every batch-th
          kv(mine.b * a.kv_heads + kvh), split_(a.slots ? slot - mine.first : slot / a.batch), n_split(mine.n) {}
    __device__ __forceinline__ int64_t query(int r) const {
        const int row = row0 + r;
        const bool live = row < a.rows;
        const uint32_t g = live ? (uint32_t)row / (uint32_t)a.T : 0u, t = live ? row - g * a.T : 0u;
        return mine.b * a.q_sb + (int64_t)(kvh * a.group + g) * a.q_sh + t * a.q_st;
    }
    __device__ __forceinline__ int64_t tiles() const { return tiles_of(mine.range); }
    // whole tiles of the history; those with the end of it or drafted tokens in them follow
    __device__ __forceinline__ int64_t whole() const {
        return std::min<int64_t>(tiles(), ((int64_t)mine.range.end - mine.range.lo) / TK);
    }
    __device__ __forceinline__ int split() const { return split_; }
    __device__ __forceinline__ int splits() const { return n_split; }
    __device__ __forceinline__ Place place(int64_t tile) const {
        const int64_t t0 = mine.range.lo + tile * TK;
        return {a.c, (int64_t)kv * a.cap + t0, (int)std::min<int64_t>(mine.range.stop - t0, TK)};
    }
    __device__ __forceinline__ uint32_t seen(int m, int64_t tile) const {
        const int64_t t0 = mine.range.lo + tile * TK;
        const int to_end = (int)std::max<int64_t>(std::min<int64_t>(mine.range.end - t0, TK), -64);
        return seen_of_tile(sees[m], to_end, (int)std::min<int64_t>(mine.range.stop - t0, TK));
    }
    __device__ __forceinline__ int rows() const { return a.rows - row0; }
    __device__ __forceinline__ int64_t partial() const { return ((int64_t)slot * a.kv_heads + kvh) * a.rows + row0; }
    __device__ __forceinline__ void prefetch(int wave, int lane) {
        if (nodes && wave == 0 && lane < a.T) parent = a.parents[mine.b * a.parents_sb + lane];
    }
    __device__ __forceinline__ void publish(int wave, int lane) const {
        if (nodes && wave == 0) s_anc[lane] = ancestors(parent, lane);
    }
    __device__ __forceinline__ void take_row(int m, int r) { sees[m] = nodes ? s_anc[(row0 + r) % a.T] : 0ull; }
};

template <int KB, int VB, bool QJL, int RB, int NQ>
__global__ __launch_bounds__(Tiles<RB>::T, 2) void tree_kernel(TreeArgs a, Codec codec) {
    __shared__ uint64_t s_anc[64];
    const int lane = threadIdx.x & 63;
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
    TreeSource<RB> src(a, s_anc, mine, slot, kvh, row_group);
    if (a.slots && src.split() == 0 && row_group == 0 && kvh == 0 && threadIdx.x == 0) a.slots[mine.b] = make_int2(mine.first, mine.n);
    attend_tiles<KB, VB, QJL, RB, NQ>(codec, src, lane, wave);
}

// Rows of [batch][kv head][head of it][node].
struct TreeRows {
    int q_heads, kv_heads, T, rows, n_split;
    int64_t all_rows;
    const int2* slots;  // or n_split for every batch row

    __device__ __forceinline__ Part find(int64_t row) const {
        if (!slots) return {row, all_rows, n_split};
        const int64_t step = (int64_t)kv_heads * rows;
        const uint32_t n = (uint32_t)row, b = n / ((uint32_t)kv_heads * (uint32_t)rows);
        const int2 s = slots[b];
        return {(s.x - (int64_t)b) * step + row, step, s.y};
    }
    __device__ __forceinline__ int64_t place(int64_t row) const {
        const uint32_t n = (uint32_t)row, kv = n / (uint32_t)rows, in = n - kv * rows, g = in / (uint32_t)T;
        const uint32_t b = kv / (uint32_t)kv_heads, hq = (kv - b * kv_heads) * (q_heads / kv_heads) + g;
        return ((int64_t)b * q_heads + hq) * T + (in - g * T);
    }
};
__global__ __launch_bounds__(MERGE_T) void merge_kernel(Merge a, TreeRows rows) { merge_rows<MERGE_ROWS>(a, rows); }

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
void launch_tree(const TreeArgs& a, const Codec& c, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)a.n_slots * p.row_groups, (unsigned)a.kv_heads);
    auto launch = [&](auto rb, auto nq) {
        hipLaunchKernelGGL((tree_kernel<KB, VB, QJL, rb, nq>), grid, dim3(Tiles<rb>::T), 0, s, a, c);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (p.row_blocks == 1) c.q_type == 0 ? launch(One{}, One{}) : launch(One{}, Two{});
    else c.q_type == 0 ? launch(Two{}, One{}) : launch(Two{}, Two{});
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
                     {k_codes, k_signs, v_codes, k_norms, k_rnorms, v_norms}, q_heads / kv_heads, q_sb, q_sh, q_st,
                     p.n_split, slots ? p.n_slots : p.n_split * batch, slots};
    const Codec c{key_centers, value_centers, key_rotation, qjl, scale * LOG2E, q, q_type, part_o, part_ms};
    if (has_qjl) {
        if (value_bits == 4) launch_tree<3, 4, true>(a, c, p, s);
        else if (value_bits == 3) launch_tree<2, 3, true>(a, c, p, s);
        else launch_tree<1, 2, true>(a, c, p, s);
    } else {
        if (value_bits == 4) launch_tree<4, 4, false>(a, c, p, s);
        else if (value_bits == 3) launch_tree<3, 3, false>(a, c, p, s);
        else if (value_bits == 2) launch_tree<2, 2, false>(a, c, p, s);
        else launch_tree<1, 1, false>(a, c, p, s);
    }
    TQ_CHECK_LAUNCH();
    const int64_t all = p.heads * p.rows;
    const Merge m{all, part_o, part_ms, value_rotation, out_f32, out_bf16, 0, lse_out};
    const TreeRows rows{q_heads, kv_heads, nodes, p.rows, p.n_split, all, slots};
    hipLaunchKernelGGL(merge_kernel, dim3((unsigned)((all + MERGE_ROWS - 1) / MERGE_ROWS)), dim3(MERGE_T), 0, s, m, rows);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
