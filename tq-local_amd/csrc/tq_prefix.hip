// tq_prefix.hip -- attention of one query token per sequence where several sequences continue one packed prompt (gfx950).
//
// The prompt is packed once for all of them, and every sequence has packed tokens of its own behind it; its query attends to both.
// The formulas, the codes' way to the matrix cores and the rounding are those of tq_tiles.h.
//
//   prefix_kernel  a workgroup has up to 32 or 64 query rows of a KV head: `per` sequences of one prompt (an item), all of a sequence's
//                  query heads.  Its tiles are the prompt's, which every row attends to, then the own tokens of its sequences, each of
//                  which only that sequence's rows attend to.  The splits of an item share its tiles
//   merge_kernel   the splits' partials of a row weighed and added, rotated back by R_v
//
// Cost (kernel and merge, in a graph).  Long prompts are bound by the tiles' decoding and softmax beside the matrix instructions, as the
// trees are: three prompts of 131072 tokens with 21, 3 and 8 sequences (8 KV heads of 5 query heads, 4-bit Q_prod) take 319 us, the 458 MB of
// codes at 1.4 TB/s, the products at 0.41 PFLOP/s (0.69 with the rows that fill the blocks up); vector instructions have 59% and matrix instructions 36% of a
// SIMD's time, at the 1.9 GHz that this leaves.  32 sequences behind 32768 tokens (8 of 4 heads) take 60 us, 8 sequences behind each of
// four padded prompts of 8192 tokens (4 of 7 heads, 3-bit Q_mse, fp16) 30.  Small calls are bound by what comes before the first tile
// and after the last: two sequences behind 1037 tokens take 15.6, the kernel 12 (the first bytes from memory, the queries' rotation, the
// table of values, the waves' meeting, 1 to 3 us each) and the merge 4.
// A copy of the prompt for every sequence and tq_decode_attention (8 of 4 heads, 4-bit Q_prod): 16 sequences behind 32768 tokens 114 us,
// here 43; 16 behind 8192 34 and 25; 4 behind 8192 16.4 and 20.5.

#include "tq_tiles.h"

namespace {

using namespace tqt;

struct PrefixArgs {
    int prompts, batch, kv_heads, group;  // query heads per KV head
    int per, items;                       // sequences of an item, and how many items there may be
    const int32_t* cu_rows;               // prompt p's sequences are [cu_rows[p], cu_rows[p + 1]); or `each` to a prompt
    int each;
    const int32_t *starts, *lens, *own_lens;
    int64_t n_prefix, cap_prefix, n_own, cap_own;
    Cache prefix, own;
    int64_t q_sb, q_sh;
    int n_split, n_slots;  // n_split slots for each item, or with `shared` n_slots dealt out by what the items have
    int shared;
    int4* row_slots;  // [batch] a sequence's first slot, its number of slots, their distance, and its place in the item
};

__device__ __forceinline__ int clamp_to(int64_t x, int64_t n) { return (int)std::min(std::max<int64_t>(x, 0), n); }
__device__ __forceinline__ int tiles_of(int tokens) { return (int)(((int64_t)tokens + TK - 1) / TK); }
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Prefix sums and maxima (of numbers >= 0) over the lanes of a wave: within the rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
template <class F>
__device__ __forceinline__ int scan(int x, F join) {
    x = join(x, moved<0x111, 0xF>(x));  // row_shr 1, 2, 4, 8
    x = join(x, moved<0x112, 0xF>(x));
    x = join(x, moved<0x114, 0xF>(x));
    x = join(x, moved<0x118, 0xF>(x));
    x = join(x, moved<0x142, 0xA>(x));  // row_bcast 15 to the second and fourth row, 31 to the upper two
    return join(x, moved<0x143, 0xC>(x));
}
__device__ __forceinline__ int scan_sum(int x) {
    return scan(x, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int scan_max(int x) {
    return scan(x, [](int a, int b) { return std::max(a, b); });
}

// An item's prompt, its first sequence and how many it has (0: there is no such item).
struct Item {
    int p, first, count;
};
// Item `it` (any lane's own), by a whole wave.  Offsets that descend or leave [0, batch] are taken as empty prompts and as the ends of
// the batch; the first prompt begins at sequence 0 and the last ends with the batch, so every sequence is of one item.
__device__ __forceinline__ Item find_item(const PrefixArgs& a, int it, int lane) {
    if (!a.cu_rows) {
        const int of_each = (a.each + a.per - 1) / a.per, p = it / of_each, at = (it - p * of_each) * a.per;
        if (p >= a.prompts) return {0, 0, 0};
        return {p, p * a.each + at, std::min(a.per, a.each - at)};
    }
    Item mine{0, 0, 0};
    int items = 0, rows = 0;  // before these prompts
    for (int p0 = 0; p0 < a.prompts; p0 += 64) {
        const int p = p0 + lane;
        int end = a.batch;
        if (p + 1 < a.prompts) end = clamp_to(a.cu_rows[p + 1], a.batch);
        end = std::max(scan_max(end), rows);
        const int up = __shfl_up(end, 1), begin = lane == 0 ? rows : up;
        const int last = scan_sum((end - begin + a.per - 1) / a.per) + items;
        const int n = std::min(64, a.prompts - p0);
        for (int i = 0; i < n; ++i) {
            const int e = __builtin_amdgcn_readlane(last, i), to = __builtin_amdgcn_readlane(end, i);
            const int at = __builtin_amdgcn_readlane(begin, i) + (it - items) * a.per;
            if (it >= items && it < e) mine = {p0 + i, at, std::min(a.per, to - at)};
            items = e, rows = to;
        }
    }
    return mine;
}

// The prompt's tokens [lo, end).
struct Range {
    int lo, end;
};
__device__ __forceinline__ Range range_of(const PrefixArgs& a, int p) {
    const int end = a.lens ? clamp_to(a.lens[p], a.n_prefix) : (int)a.n_prefix;
    return {a.starts ? clamp_to(a.starts[p], end) : 0, end};
}
__device__ __forceinline__ int own_of(const PrefixArgs& a, int row) {
    return a.own_lens ? clamp_to(a.own_lens[row], a.n_own) : (int)a.n_own;
}

// A slot's item, the first of the item's slots, their number and distance.
struct Slot {
    Item item;
    int first, n, step;
};
// Where lengths may differ, up to 64 items of up to 64 prompts and SHARED_ROWS sequences share the slots in proportion to their tiles, each
// with one at least; what is left over goes unused (count = 0).  Equal numbers of slots and shares, in graphs, us: two sequences behind each of a
// prompt of 32768 tokens and seven of 2000 90 and 38, the three prompts above 339 and 315, eight equal prompts 103 and 105.  All that it reads is asked for together: one wait for memory where a loop over an item's
// sequences had one for each.
constexpr int SHARED_ROWS = 256;
struct Shared {
    int own[SHARED_ROWS / 64];  // of sequence 64 i + lane
    Range range;                // of prompt `lane`
};
__device__ __forceinline__ Slot share_slots(const PrefixArgs& a, int slot, int lane, Shared& s) {
#pragma unroll
    for (int i = 0; i < SHARED_ROWS / 64; ++i) s.own[i] = 64 * i + lane < a.batch ? own_of(a, 64 * i + lane) : 0;
    s.range = lane < a.prompts ? range_of(a, lane) : Range{0, 0};
    const Item mine = find_item(a, lane, lane);
    // tiles of the sequences up to each
    int before = 0, last = mine.first + mine.count - 1, tiles = 0;
#pragma unroll
    for (int i = 0; i < SHARED_ROWS / 64; ++i) {
        if (64 * i >= a.batch) break;
        const int up = scan_sum(tiles_of(s.own[i])) + before;
        const int to = __shfl(up, last & 63), from = __shfl(up, (mine.first - 1) & 63);
        if (last >> 6 == i) tiles += to;
        if (mine.first > 0 && (mine.first - 1) >> 6 == i) tiles -= from;
        before = __builtin_amdgcn_readlane(up, 63);
    }
    tiles = mine.count ? tiles + __shfl(tiles_of(s.range.end - s.range.lo), mine.p) : 0;
    const int total = __builtin_amdgcn_readlane(scan_sum(tiles), 63);
    // (the sum of the shares does not pass what there is to share, whatever the roundings: these are far below 1)
    const int share = (int)((float)(a.n_slots - a.items) * ((float)tiles / (float)std::max(total, 1)));
    const int n = mine.count ? std::min(std::min(1 + share, std::max(1, (tiles + MIN_TILES - 1) / MIN_TILES)), MAX_SPLIT) : 0;
    const int end = scan_sum(n), i = __popcll(__ballot(end <= slot));
    if (i >= 64) return {{0, 0, 0}, 0, 0, 0};
    auto of_item = [&](int x) { return __builtin_amdgcn_readlane(x, i); };
    return {{of_item(mine.p), of_item(mine.first), of_item(mine.count)}, of_item(end - n), of_item(n), 1};
}

// Rows sequence by sequence, a sequence's query heads next to one another.
template <int RB>
struct PrefixSource {
    const PrefixArgs& a;
    const Slot& at;
    const int slot, kvh, lo, end, shared_tiles, own_lens, own_tiles;  // the last two: of sequence `lane`, and with those before it
    int member[RB];

    __device__ __forceinline__ PrefixSource(const PrefixArgs& a, const Slot& at, int slot, int kvh, Range range, int own_len)
        : a(a), at(at), slot(slot), kvh(kvh), lo(scalar(range.lo)), end(scalar(range.end)), shared_tiles(tiles_of(end - lo)),
          own_lens(own_len), own_tiles(scan_sum(tiles_of(own_len))) {}
    __device__ __forceinline__ int64_t query(int r) const {
        const uint32_t m = (uint32_t)r / (uint32_t)a.group, g = r - m * a.group;
        const bool live = (int)m < at.item.count;
        return (int64_t)(at.item.first + (live ? m : 0u)) * a.q_sb + (int64_t)(kvh * a.group + (live ? g : 0u)) * a.q_sh;
    }
    __device__ __forceinline__ int64_t tiles() const { return shared_tiles + __builtin_amdgcn_readlane(own_tiles, 63); }
    __device__ __forceinline__ int64_t whole() const { return (end - lo) / TK; }
    __device__ __forceinline__ int split() const { return (slot - at.first) / at.step; }
    __device__ __forceinline__ int splits() const { return at.n; }
    // whose own tile it is; -1: the prompt's
    __device__ __forceinline__ int owner(int64_t tile) const {
        return tile < shared_tiles ? -1 : __popcll(__ballot(own_tiles <= (int)tile - shared_tiles));
    }
    __device__ __forceinline__ Place place(int64_t tile) const {
        const int s = owner(tile), m = std::max(s, 0);
        const bool mine = s >= 0;
        const int len = __builtin_amdgcn_readlane(own_lens, m), before = __builtin_amdgcn_readlane(own_tiles, m) - tiles_of(len);
        const int t0 = mine ? ((int)tile - shared_tiles - before) * TK : lo + (int)tile * TK;
        const int64_t row = mine ? (int64_t)(at.item.first + m) : (int64_t)at.item.p;
        const Cache &p = a.prefix, &o = a.own;
        return {{mine ? o.k_codes : p.k_codes, mine ? o.k_signs : p.k_signs, mine ? o.v_codes : p.v_codes, mine ? o.k_norms : p.k_norms,
                 mine ? o.k_rnorms : p.k_rnorms, mine ? o.v_norms : p.v_norms},
                (row * a.kv_heads + kvh) * (mine ? a.cap_own : a.cap_prefix) + t0, std::min((mine ? len : end) - t0, TK)};
    }
    __device__ __forceinline__ uint32_t seen(int m, int64_t tile) const {
        const int s = owner(tile), left = place(tile).left;  // by the whole wave, ahead of what differs between lanes
        return s < 0 || s == member[m] ? (uint32_t)((1ull << left) - 1) : 0u;
    }
    __device__ __forceinline__ int rows() const { return at.item.count * a.group; }
    __device__ __forceinline__ int64_t partial() const { return ((int64_t)slot * a.kv_heads + kvh) * (32 * RB); }
    __device__ __forceinline__ void prefetch(int, int) {}
    __device__ __forceinline__ void publish(int, int) const {}
    __device__ __forceinline__ void take_row(int m, int r) { member[m] = r / a.group; }
};

// fp16 and fp32 queries (NQ = 2) keep their bits behind the rotation too, in two fp16 terms (LO): 32 sequences behind 32768 tokens (8 of 4 heads,
// 4-bit Q_prod, fp16) take 68.6 us and 60.2 with one term, the padded prompts above 29.9 and 28.9, and lose 5.4e-4 and 7.1e-4 of an output's
// norm, 2.5e-4 with scaled codebooks as well.
template <int KB, int VB, bool QJL, int RB, int NQ>
__global__ __launch_bounds__(Tiles<RB>::T, 2) void prefix_kernel(PrefixArgs a, Codec codec) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = blockIdx.x, kvh = blockIdx.y;
    Slot at;
    Range range;
    int own_len = 0;  // of the item's sequence `lane`
    if (a.shared) {
        Shared s;
        at = share_slots(a, slot, lane, s);
        if (at.item.count == 0) return;
        range = {__builtin_amdgcn_readlane(s.range.lo, at.item.p), __builtin_amdgcn_readlane(s.range.end, at.item.p)};
        const int row = at.item.first + lane;
#pragma unroll
        for (int i = 0; i < SHARED_ROWS / 64; ++i) {
            const int x = __shfl(s.own[i], row & 63);
            if (row >> 6 == i && lane < at.item.count) own_len = x;
        }
    } else {
        const int it = slot % a.items;
        const Item item = find_item(a, it, lane);
        at = {{scalar(item.p), scalar(item.first), scalar(item.count)}, it, a.n_split, a.items};
        if (at.item.count == 0) return;
        if (lane < at.item.count) own_len = own_of(a, at.item.first + lane);
        range = range_of(a, at.item.p);
    }
    PrefixSource<RB> src(a, at, slot, kvh, range, own_len);
    if (src.split() == 0 && kvh == 0 && (int)threadIdx.x < at.item.count)
        a.row_slots[at.item.first + threadIdx.x] = make_int4(at.first, at.n, at.step, threadIdx.x);
    attend_tiles<KB, VB, QJL, RB, NQ, (NQ > 1)>(codec, src, lane, wave);
}

// Rows of [batch][q head].
struct PrefixRows {
    int q_heads, kv_heads, rows;  // rows of an item
    const int4* slots;

    __device__ __forceinline__ Part find(int64_t row) const {
        const uint32_t n = (uint32_t)row, b = n / (uint32_t)q_heads, hq = n - b * q_heads;
        const uint32_t group = (uint32_t)q_heads / (uint32_t)kv_heads, kvh = hq / group;
        const int4 s = slots[b];
        return {((int64_t)s.x * kv_heads + kvh) * rows + s.w * group + (hq - kvh * group), (int64_t)s.z * kv_heads * rows, s.y};
    }
    __device__ __forceinline__ int64_t place(int64_t row) const { return row; }
};
template <int ROWS>
__global__ __launch_bounds__(MERGE_T) void merge_kernel(Merge a, PrefixRows rows) {
    merge_rows<ROWS>(a, rows);
}

// Rows up to which the merge has 4 of them to a workgroup, which is done with them sooner; 16 beyond, which read the matrix R_v once for
// more.  16 rows always and 4 always, in graphs, us: 64 rows 19.4 and 15.6, 1024 rows 63.3 and 59.8, 1280 rows 323.4 and 320.8.
constexpr int FEW_ROWS = 2048;

struct Plan {
    int row_blocks, per, items, n_split, n_slots;
    size_t o_bytes, ms_bytes, slots_bytes;
    size_t total() const { return o_bytes + ms_bytes + slots_bytes; }
};

// Blocks of 32 rows, or of 64, whose tiles are decoded once for twice the rows.  In graphs, us, 32 and 64 rows: two sequences behind 1037
// tokens 15.6 and 19.1, 56 rows behind each of four times 8192 (3-bit Q_mse) 28.9 and 32.5, 128 behind 32768 63.9 and 59.8, 160 behind
// three times 131072 345 and 321.  A tile of 64 rows takes 5/3 of one of 32, and a workgroup's start and end 46 and 38 tiles of 32
// rows (46 is 8 more, 3 us).  A workgroup fills a CU: as many splits as fill the CUs, as long as none is left without a tile.
bool make_plan(int batch, int q_heads, int kv_heads, int prompts, bool uneven, int max_rows, int64_t n_prefix, int64_t n_own, Plan& p) {
    const int group = q_heads / kv_heads, each = batch / prompts;
    const int most = uneven ? std::min(batch, std::max(max_rows, 1)) : each;
    if (group > 64 || kv_heads > 65535 || (int64_t)batch * q_heads >= (int64_t)1 << 26) return false;
    if (n_prefix + 64 * n_own >= (int64_t)1 << 29) return false;  // sums of 64 items' tiles fit 32 bits
    int64_t useful = 1;
    // the plan for blocks of 32 row_blocks rows; returns what it takes, in thirds of a tile of 32 rows
    auto take = [&](int row_blocks) {
        p.row_blocks = row_blocks;
        p.per = 32 * row_blocks / group;
        p.items = uneven ? (int)std::min<int64_t>(batch, (int64_t)batch / p.per + prompts) : prompts * ((each + p.per - 1) / p.per);
        const int64_t tiles = (n_prefix + TK - 1) / TK + std::min(p.per, batch) * ((n_own + TK - 1) / TK);
        useful = std::min<int64_t>(std::max<int64_t>(1, (tiles + MIN_TILES - 1) / MIN_TILES), MAX_SPLIT);
        p.n_split = (int)std::max<int64_t>(1, std::min<int64_t>(256 / ((int64_t)p.items * kv_heads), useful));
        // (uneven items are taken as full ones: how many there are the device knows)
        const int64_t groups = (int64_t)(uneven ? (batch + p.per - 1) / p.per : p.items) * kv_heads;
        const int64_t split = std::max<int64_t>(1, std::min<int64_t>(256 / groups, useful));
        const int64_t rounds = (groups * split + 255) / 256, each_has = (tiles + split - 1) / split;
        return rounds * (row_blocks == 1 ? 114 + 3 * each_has : 138 + 5 * each_has);
    };
    // (more than 32 query heads take 64 rows, a prompt's few rows 32)
    const bool one = group <= 32, two = (int64_t)most * group > 32;
    const int64_t of_two = two ? take(2) : 0, of_one = one ? take(1) : 0;
    if (two && (!one || of_two < of_one)) take(2);
    p.n_slots = (int)std::max<int64_t>((int64_t)p.n_split * p.items, std::min<int64_t>(256 / kv_heads, useful * p.items));
    const size_t rows = (size_t)p.n_slots * kv_heads * 32 * p.row_blocks;
    p.o_bytes = rows * D * 4, p.ms_bytes = rows * 8, p.slots_bytes = (size_t)batch * 16;
    return true;
}

template <int KB, int VB, bool QJL>
void launch_prefix(const PrefixArgs& a, const Codec& c, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)a.n_slots, (unsigned)a.kv_heads);
    auto launch = [&](auto rb, auto nq) {
        hipLaunchKernelGGL((prefix_kernel<KB, VB, QJL, rb, nq>), grid, dim3(Tiles<rb>::T), 0, s, a, c);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (p.row_blocks == 1) c.q_type == 0 ? launch(One{}, One{}) : launch(One{}, Two{});
    else c.q_type == 0 ? launch(Two{}, One{}) : launch(Two{}, Two{});
}

bool good_shape(int batch, int q_heads, int kv_heads, int prompts, bool uneven, int64_t n_prefix, int64_t n_own) {
    return batch >= 1 && q_heads >= 1 && kv_heads >= 1 && q_heads % kv_heads == 0 && prompts >= 1 && (uneven || batch % prompts == 0) &&
           n_prefix >= 0 && n_own >= 0;
}
// `caches`: k_codes, k_norms, k_signs, k_rnorms, v_codes, v_norms
bool has_arrays(const void* const* c, int64_t n, int has_qjl) {
    return n == 0 || (c && c[0] && c[1] && c[4] && c[5] && (!has_qjl || (c[2] && c[3])));
}
bool has_alignment(const void* const* c, int64_t n, int has_qjl) {
    return n == 0 || (aligned16(c[0]) && aligned16(c[4]) && (!has_qjl || aligned16(c[2])));
}
Cache cache_of(const void* const* c, int64_t n) {
    if (n == 0) return Cache{};
    auto u8 = [&](int i) { return static_cast<const uint8_t*>(c[i]); };
    auto u16 = [&](int i) { return static_cast<const uint16_t*>(c[i]); };
    return {u8(0), u8(2), u8(4), u16(1), u16(3), u16(5)};
}

}  // namespace

extern "C" size_t tq_prefix_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int dim, int prompts, int uneven,
                                                      int max_rows, int64_t n_prefix, int64_t n_own) {
    Plan p;
    if (!good_shape(batch, q_heads, kv_heads, prompts, uneven != 0, n_prefix, n_own) || dim != D ||
        !make_plan(batch, q_heads, kv_heads, prompts, uneven != 0, max_rows, n_prefix, n_own, p))
        return 0;
    return p.total();
}

extern "C" int tq_prefix_attention(const void* q, int q_type, int batch, int q_heads, int kv_heads, int dim, int64_t q_sb, int64_t q_sh,
                                   int prompts, const int32_t* cu_rows, int max_rows, const int32_t* prefix_starts,
                                   const int32_t* prefix_lens, int64_t n_prefix, int64_t cap_prefix, const void* const* prefix,
                                   const int32_t* own_lens, int64_t n_own, int64_t cap_own, const void* const* own, int key_bits,
                                   int value_bits, int has_qjl, const float* key_rotation, const float* key_centers, const float* qjl,
                                   const float* value_rotation, const float* value_centers, float scale, float* out_f32,
                                   uint16_t* out_16, float* lse_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!q || q_type < 0 || q_type > 2 || !good_shape(batch, q_heads, kv_heads, prompts, cu_rows != nullptr, n_prefix, n_own) ||
        n_prefix > cap_prefix || n_own > cap_own || !has_arrays(prefix, n_prefix, has_qjl) || !has_arrays(own, n_own, has_qjl) ||
        !key_rotation || !key_centers || !value_rotation || !value_centers || (has_qjl && !qjl) || (!out_f32 && !out_16) ||
        !(scale > 0.0f) || scale == __builtin_inff())
        return TQ_ERR_INVALID_ARGUMENT;
    if (dim != D || n_prefix >= (int64_t)1 << 31 || n_own >= (int64_t)1 << 31 || value_bits < 1 || value_bits > 4 || key_bits < 1 ||
        key_bits != value_bits - (has_qjl ? 1 : 0))
        return TQ_ERR_UNSUPPORTED;
    if (!aligned16(key_rotation) || (has_qjl && !aligned16(qjl)) || !has_alignment(prefix, n_prefix, has_qjl) ||
        !has_alignment(own, n_own, has_qjl))
        return TQ_ERR_UNSUPPORTED;
    Plan p;
    if (!make_plan(batch, q_heads, kv_heads, prompts, cu_rows != nullptr, max_rows, n_prefix, n_own, p)) return TQ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.total() || !aligned16(workspace)) return TQ_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int4* const row_slots = reinterpret_cast<int4*>(ws + p.o_bytes + p.ms_bytes);
    const int shared = (cu_rows || prefix_starts || prefix_lens || own_lens) && p.items <= 64 && prompts <= 64 && batch <= SHARED_ROWS &&
                       p.n_slots > p.items;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const PrefixArgs a{prompts, batch, kv_heads, q_heads / kv_heads, p.per, p.items, cu_rows, batch / prompts,
                       prefix_starts, prefix_lens, own_lens, n_prefix, cap_prefix, n_own, cap_own,
                       cache_of(prefix, n_prefix), cache_of(own, n_own), q_sb, q_sh, p.n_split,
                       shared ? p.n_slots : p.n_split * p.items, shared, row_slots};
    const Codec c{key_centers, value_centers, key_rotation, qjl, scale * LOG2E, q, q_type, reinterpret_cast<float*>(ws),
                  reinterpret_cast<float2*>(ws + p.o_bytes)};
    if (has_qjl) {
        if (value_bits == 4) launch_prefix<3, 4, true>(a, c, p, s);
        else if (value_bits == 3) launch_prefix<2, 3, true>(a, c, p, s);
        else launch_prefix<1, 2, true>(a, c, p, s);
    } else {
        if (value_bits == 4) launch_prefix<4, 4, false>(a, c, p, s);
        else if (value_bits == 3) launch_prefix<3, 3, false>(a, c, p, s);
        else if (value_bits == 2) launch_prefix<2, 2, false>(a, c, p, s);
        else launch_prefix<1, 1, false>(a, c, p, s);
    }
    TQ_CHECK_LAUNCH();
    const Merge m{(int64_t)batch * q_heads, c.part_o, c.part_ms, value_rotation, out_f32, out_16, q_type == 2, lse_out};
    const PrefixRows rows{q_heads, kv_heads, 32 * p.row_blocks, row_slots};
    if (m.all_rows <= FEW_ROWS)
        hipLaunchKernelGGL(merge_kernel<4>, dim3((unsigned)((m.all_rows + 3) / 4)), dim3(MERGE_T), 0, s, m, rows);
    else
        hipLaunchKernelGGL(merge_kernel<MERGE_ROWS>, dim3((unsigned)((m.all_rows + MERGE_ROWS - 1) / MERGE_ROWS)), dim3(MERGE_T), 0, s,
                           m, rows);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
