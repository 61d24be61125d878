// tq_moves.hip -- tokens of a packed layer chosen, copied and moved together (gfx950), all buffers of a layer
// in one launch: the rows of a batch forked or reordered, a history thinned out, an accepted path of drafted
// tokens closed up.
//
// Nothing is computed: bytes read plus bytes written bound it.  A buffer's rows have any number of bytes (124
// codes of 3 bits are 47), so reads take 16 bytes at any address and writes 16 at aligned ones where rows
// follow one another, 16 at any where they are picked one by one.
//
// 8 rows made of 4 of 32768 tokens (8 heads, 4-bit Q_prod: 421 MB) take 86 us = 4.9 TB/s, where a copy of 1 GiB reaches 5.1.
// Half of 16384 tokens chosen for each head of a layer in two channel groups (2 x 8 heads, twelve buffers with rows of 1 to
// 62 bytes, 37 MB) takes 15 us = 2.5 TB/s: small rows leave most of a 16-byte piece empty, and each piece reads its index.
// 6 of 16 tokens moved in place take 3.4 us, a launch.  Calls as small as the last two cost their host time: 5 us of the launch and
// the arguments, 1.5 us for each new buffer.

#include <algorithm>

#include "tq_common.h"

namespace {

constexpr int MAX_BUFFERS = 16;
constexpr int T = 256;
constexpr int UNITS = 4;              // 16-byte pieces a thread moves
constexpr int CHUNK = 16 * T * UNITS; // bytes of a workgroup

struct Moves {
    const uint8_t* src[MAX_BUFFERS];
    uint8_t* dst[MAX_BUFFERS];
    int row[MAX_BUFFERS];
    int64_t first_wg[MAX_BUFFERS + 1];  // workgroups of the buffers before
    int n_buffers, heads, src_batch;
    int64_t src_cap, dst_cap, tokens, n;  // n tokens arrive, the slots behind them are cleared
    int64_t wg_per_region[MAX_BUFFERS];
    const int32_t* rows;
    const int32_t* index;
    int64_t index_sb, index_sh;
};

__device__ __forceinline__ uint4 load16(const uint8_t* p) {
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
__device__ __forceinline__ void store16(uint8_t* p, uint4 v) { __builtin_memcpy(p, &v, 16); }

// `len` < 16 bytes, or zeros for a null source
__device__ __forceinline__ void copy_bytes(uint8_t* d, const uint8_t* s, int len) {
    for (int i = 0; i < len; ++i) d[i] = s ? s[i] : 0;
}

template <bool INDEXED>
__global__ __launch_bounds__(T) void gather_kernel(Moves m) {
    int b = 0;
    while (b + 1 < m.n_buffers && (int64_t)blockIdx.x >= m.first_wg[b + 1]) ++b;
    const int64_t wg = blockIdx.x - m.first_wg[b];
    const int64_t region = wg / m.wg_per_region[b], part = wg - region * m.wg_per_region[b];
    const int out_row = (int)(region / m.heads), head = (int)(region - (int64_t)out_row * m.heads);
    const int in_row = m.rows ? m.rows[out_row] : out_row;
    const int R = m.row[b];
    const uint8_t* src = in_row < 0 || in_row >= m.src_batch
                             ? nullptr
                             : m.src[b] + ((int64_t)in_row * m.heads + head) * m.src_cap * R;
    uint8_t* const dst = m.dst[b] + region * m.dst_cap * R;
    if constexpr (!INDEXED) {
        // bytes [0, n R) of the region from the source, zeros behind them; aligned pieces of the destination
        const int skew = (int)(reinterpret_cast<uintptr_t>(dst) & 15u);
        const int64_t size = m.dst_cap * R, full = src ? m.n * R : 0;
        uint4 v[UNITS];
        int64_t at[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            at[u] = part * CHUNK + 16 * (u * T + (int)threadIdx.x) - skew;
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            if (at[u] >= 0 && at[u] + 16 <= full) v[u] = load16(src + at[u]);
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int64_t lo = at[u] < 0 ? 0 : at[u], hi = std::min(at[u] + 16, size);
            if (lo >= hi) continue;
            if (hi - lo == 16 && (hi <= full || lo >= full)) {
                *reinterpret_cast<uint4*>(dst + lo) = v[u];
            } else {
                for (int64_t i = lo; i < hi; ++i) dst[i] = i < full ? src[i] : 0;
            }
        }
    } else {
        const int parts = (R + 15) / 16;  // pieces of a row, the last one set back to end with it
        const int32_t* const index = m.index + out_row * m.index_sb + head * m.index_sh;
        uint4 v[UNITS];
        int64_t tok[UNITS];
        const uint8_t* from[UNITS];
        int off[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int64_t unit = part * (T * UNITS) + u * T + threadIdx.x;
            tok[u] = unit / parts;
            off[u] = std::max(0, std::min(16 * (int)(unit - tok[u] * parts), R - 16));
            int64_t from_tok = -1;
            if (tok[u] < m.n) from_tok = index[tok[u]];
            from[u] = src && from_tok >= 0 && from_tok < m.tokens ? src + from_tok * R : nullptr;
            v[u] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if (!from[u]) continue;
            if (R >= 16) v[u] = load16(from[u] + off[u]);
            else if (R == 2) v[u].x = from[u][0] | from[u][1] << 8;
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if (tok[u] >= m.dst_cap) continue;
            uint8_t* const d = dst + tok[u] * R;
            if (R >= 16) store16(d + off[u], v[u]);
            else if (R == 2) d[0] = (uint8_t)v[u].x, d[1] = (uint8_t)(v[u].x >> 8);
            else copy_bytes(d, from[u], R);
        }
    }
}

// One region of one buffer per workgroup: the chosen rows are all read before any is written, so the index may
// name them in any order and more than once.
__global__ __launch_bounds__(T) void keep_kernel(Moves m) {
    extern __shared__ __align__(16) uint8_t s_rows[];
    const int b = blockIdx.y, R = m.row[b];
    const int out_row = blockIdx.x / m.heads, head = blockIdx.x - out_row * m.heads;
    uint8_t* const base = m.dst[b] + (int64_t)blockIdx.x * m.dst_cap * R;
    const int32_t* const index = m.index + out_row * m.index_sb + head * m.index_sh;
    const int parts = (R + 15) / 16, units = (int)m.n * parts;
    for (int u = threadIdx.x; u < units; u += T) {
        const int tok = u / parts, off = std::max(0, std::min(16 * (u - tok * parts), R - 16));
        const int64_t from_tok = index[tok];
        const uint8_t* from = from_tok >= 0 && from_tok < m.tokens ? base + from_tok * R : nullptr;
        if (R >= 16) store16(s_rows + tok * R + off, from ? load16(from + off) : make_uint4(0u, 0u, 0u, 0u));
        else copy_bytes(s_rows + tok * R, from, R);
    }
    __syncthreads();
    for (int u = threadIdx.x; u < units; u += T) {
        const int tok = u / parts, off = std::max(0, std::min(16 * (u - tok * parts), R - 16));
        if (R >= 16) store16(base + (int64_t)tok * R + off, load16(s_rows + tok * R + off));
        else copy_bytes(base + (int64_t)tok * R, s_rows + tok * R, R);
    }
}

bool bad_buffers(int n_buffers, const int* row_bytes, const void* const* a, const void* const* b) {
    if (n_buffers < 1 || n_buffers > MAX_BUFFERS || !row_bytes || !a || !b) return true;
    for (int i = 0; i < n_buffers; ++i)
        if (!a[i] || !b[i] || row_bytes[i] < 1 || row_bytes[i] > TQ_MAX_ROW_BYTES) return true;
    return false;
}

}  // namespace

extern "C" int tq_gather_tokens(int n_buffers, const void* const* src, void* const* dst, const int* row_bytes,
                                int src_batch, int heads, int64_t src_cap, int64_t tokens, int dst_batch,
                                int64_t dst_cap, const int32_t* rows, const int32_t* index, int64_t index_sb,
                                int64_t index_sh, int64_t n_index, void* stream) {
    if (bad_buffers(n_buffers, row_bytes, src, dst) || src_batch < 1 || heads < 1 || dst_batch < 1 || tokens < 0 ||
        tokens > src_cap || dst_cap < 1 || (!rows && dst_batch != src_batch) || (index && n_index < 0) ||
        (index ? n_index : tokens) > dst_cap)
        return TQ_ERR_INVALID_ARGUMENT;
    Moves m{};
    int64_t wgs = 0;
    for (int i = 0; i < n_buffers; ++i) {
        m.src[i] = static_cast<const uint8_t*>(src[i]);
        m.dst[i] = static_cast<uint8_t*>(dst[i]);
        m.row[i] = row_bytes[i];
        // a region that does not start at a 16-byte boundary reaches up to 15 bytes further in aligned pieces
        m.wg_per_region[i] = index ? (dst_cap * ((row_bytes[i] + 15) / 16) + T * UNITS - 1) / (T * UNITS)
                                   : (dst_cap * row_bytes[i] + 15 + CHUNK - 1) / CHUNK;
        m.first_wg[i] = wgs;
        wgs += m.wg_per_region[i] * dst_batch * heads;
    }
    m.first_wg[n_buffers] = wgs;
    if (wgs >= (int64_t)1 << 24) return TQ_ERR_UNSUPPORTED;
    m.n_buffers = n_buffers, m.heads = heads, m.src_batch = src_batch, m.src_cap = src_cap, m.dst_cap = dst_cap;
    m.tokens = tokens, m.n = index ? n_index : tokens, m.rows = rows, m.index = index;
    m.index_sb = index_sb, m.index_sh = index_sh;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (index) hipLaunchKernelGGL(gather_kernel<true>, dim3((unsigned)wgs), dim3(T), 0, s, m);
    else hipLaunchKernelGGL(gather_kernel<false>, dim3((unsigned)wgs), dim3(T), 0, s, m);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}

extern "C" int tq_keep_tokens(int n_buffers, void* const* buffers, const int* row_bytes, int batch, int heads,
                              int64_t cap, int64_t first, int64_t tokens, const int32_t* index, int64_t index_sb,
                              int64_t index_sh, int n_index, void* stream) {
    if (bad_buffers(n_buffers, row_bytes, buffers, buffers) || !index || batch < 1 || heads < 1 || first < 0 ||
        tokens < 0 || first > cap - tokens || n_index < 0 || n_index > tokens)
        return TQ_ERR_INVALID_ARGUMENT;
    int widest = 0;
    for (int i = 0; i < n_buffers; ++i) widest = std::max(widest, row_bytes[i]);
    if (n_index > TQ_MAX_KEEP || (int64_t)n_index * widest > TQ_MAX_KEEP_BYTES ||
        (int64_t)batch * heads >= (int64_t)1 << 24)
        return TQ_ERR_UNSUPPORTED;
    if (n_index == 0) return TQ_OK;
    Moves m{};
    for (int i = 0; i < n_buffers; ++i) {
        m.row[i] = row_bytes[i];
        m.dst[i] = static_cast<uint8_t*>(buffers[i]) + first * row_bytes[i];
    }
    m.n_buffers = n_buffers, m.heads = heads, m.dst_cap = cap, m.tokens = tokens, m.n = n_index;
    m.index = index, m.index_sb = index_sb, m.index_sh = index_sh;
    hipLaunchKernelGGL(keep_kernel, dim3((unsigned)(batch * heads), (unsigned)n_buffers), dim3(T),
                       (size_t)(n_index * widest), static_cast<hipStream_t>(stream), m);
    TQ_CHECK_LAUNCH();
    return TQ_OK;
}
