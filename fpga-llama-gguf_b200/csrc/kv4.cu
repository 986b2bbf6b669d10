// Block maps, and the rows of the paged 4-bit cache: quantized into it, read back, moved between beams.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv4.cuh"
#include "serve.h"

namespace b200q {
namespace {

__device__ __forceinline__ void tell(uint32_t *status, unsigned bit) {
    if (status) atomicOr(status, bit);
}

// ---- block_map ------------------------------------------------------------------------------------------------------
// Request r's new tokens take positions past .. past + new - 1. Blocks ceil(past / page) .. ceil(kv / page) - 1 of its
// table row come from the free list in request order: two exclusive sums over the requests (rows, fresh pages), then one
// slot a row. A single CTA: the work is two short sums, and rows are a few bytes each.
__global__ void __launch_bounds__(1024) block_map_kernel(const BlockMapArgs a) {
    __shared__ unsigned long long warp_rows[32], warp_need[32];
    __shared__ unsigned long long done_rows, done_need;
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned long long cap = (unsigned long long)a.stride * a.page;
    const unsigned cursor = *a.cursor_in;
    if (tid == 0) done_rows = done_need = 0;
    __syncthreads();
    for (unsigned r0 = 0; r0 < a.n_req; r0 += 1024) {
        const unsigned r = r0 + tid;
        unsigned long long past = 0, fresh = 0, first = 0, last = 0;
        if (r < a.n_req) {
            past = a.past[r];
            fresh = a.fresh[r];
            unsigned long long kv = past + fresh;
            if (kv > cap) {
                kv = cap;
                tell(a.status, kServeShort);
            }
            a.kv_len[r] = unsigned(kv);
            first = (past + a.page - 1) / a.page;
            last = (kv + a.page - 1) / a.page;
            if (last < first) last = first;
        }
        unsigned long long rows = fresh, need = last - first;
        for (unsigned o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(~0u, rows, o), y = __shfl_up_sync(~0u, need, o);
            if (lane >= o) rows += x, need += y;
        }
        if (lane == 31) warp_rows[warp] = rows, warp_need[warp] = need;
        __syncthreads();
        unsigned long long row0 = done_rows + rows - fresh, need0 = done_need + need - (last - first);
        for (unsigned w = 0; w < warp; ++w) row0 += warp_rows[w], need0 += warp_need[w];
        if (r < a.n_req) {
            a.q_start[r] = unsigned(row0);
            for (unsigned long long b = first; b < last; ++b) {
                const unsigned long long f = cursor + need0 + (b - first);
                a.table[size_t(r) * a.stride + b] = f < a.n_free ? a.free_pages[f] : kNoSlot;
            }
            if (last > first && cursor + need0 + (last - first) > a.n_free) tell(a.status, kServeShort);
        }
        __syncthreads();
        if (tid == 1023) {
            done_rows = row0 + fresh;
            done_need = need0 + (last - first);
        }
        __syncthreads();
    }
    if (tid == 0) {
        a.q_start[a.n_req] = unsigned(done_rows);
        const unsigned long long c = cursor + done_need;
        *a.cursor_out = unsigned(c < a.n_free ? c : (cursor < a.n_free ? a.n_free : cursor));
        if (done_rows > a.n_rows) tell(a.status, kServeRequest);
    }
    __syncthreads();
    for (unsigned j = tid; j < a.n_rows; j += 1024) {
        unsigned slot = kNoSlot, pos = 0;
        if (j < done_rows) {
            unsigned lo = 0, hi = a.n_req;  // the last request that starts at or before row j
            while (hi - lo > 1) {
                const unsigned mid = (lo + hi) / 2;
                if (a.q_start[mid] <= j) lo = mid;
                else hi = mid;
            }
            const unsigned long long p = (unsigned long long)a.past[lo] + (j - a.q_start[lo]);
            if (p < cap) {
                pos = unsigned(p);
                const unsigned page = a.table[size_t(lo) * a.stride + pos / a.page];
                if (page != kNoSlot) slot = page * a.page + pos % a.page;
            }
        }
        a.slots[j] = slot;
        a.positions[j] = pos;
    }
}

// ---- kv4_store / kv4_load -------------------------------------------------------------------------------------------
// Eight lanes take a 32-dim block (four values each); lane l < 4 writes word l, whose high nibbles lane l + 4 holds.
// The quantizer is Q4_0's: d = x[argmax |x|] / -8 (the first on ties), code = min(15, trunc(x (1 / d) + 8.5)), every step
// rounded to FP32 by itself; a block that holds a NaN or an infinity gets a NaN scale, so that it reads back as NaN.
__device__ __forceinline__ uint8_t *tile_of(const Kv4View &c, unsigned slot, unsigned head) {
    const unsigned page = slot / c.page, t = slot % c.page / kTileTokens;
    return c.base + ((size_t(page) * c.n_kv + head) * (c.page / kTileTokens) + t) * kv4_tile_bytes(c.dim);
}

__global__ void __launch_bounds__(256) kv4_store_kernel(const Kv4RowsArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned nb = a.c.dim / 32, per_row = a.c.n_kv * nb * 2;  // blocks of a token: K's, then V's
    const unsigned long long total = (unsigned long long)a.n * per_row * 8;
    for (unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x; i < (total + 31) / 32 * 32;
         i += (unsigned long long)gridDim.x * 256) {
        const bool real = i < total;
        const unsigned long long blk = real ? i / 8 : 0;
        const unsigned l = unsigned(i % 8), row = unsigned(blk / per_row), in_row = unsigned(blk % per_row);
        const bool is_v = in_row >= per_row / 2;
        const unsigned hb = is_v ? in_row - per_row / 2 : in_row, head = hb / nb, b = hb % nb;
        const float *src = (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) + hb * 32 + l * 4;
        float x[4];
        for (unsigned e = 0; e < 4; ++e) x[e] = real ? src[e] : 0.0f;
        float best = 0.0f, amax = 0.0f;
        bool bad = false;
        for (unsigned e = 0; e < 4; ++e) {
            bad = bad || !(fabsf(x[e]) <= 3.402823466e38f);
            if (fabsf(x[e]) > amax) amax = fabsf(x[e]), best = x[e];
        }
        for (unsigned o = 1; o < 8; o <<= 1) {
            const float m = __shfl_xor_sync(~0u, amax, o), v = __shfl_xor_sync(~0u, best, o);
            bad = __shfl_xor_sync(~0u, int(bad), o) || bad;
            if (m > amax || (m == amax && (l & o))) amax = m, best = v;  // the lower lanes' value on ties
        }
        const float d = best * -0.125f, inv = d != 0.0f ? fdiv(1.0f, d) : 0.0f;
        uint32_t half = 0;
        for (unsigned e = 0; e < 4; ++e) {
            const int q = bad ? 8 : int(fadd(fmul(x[e], inv), 8.5f));
            half |= uint32_t(q < 15 ? (q < 0 ? 0 : q) : 15) << (8 * e);
        }
        const uint32_t high = __shfl_down_sync(~0u, half, 4);
        if (!real) continue;
        const unsigned slot = a.slots[row];
        if (slot == kNoSlot) continue;
        if (slot / a.c.page >= a.c.n_pages) {
            tell(a.status, kServeSlot);
            continue;
        }
        uint8_t *tile = tile_of(a.c, slot, head);
        const unsigned t = slot % a.c.page % kTileTokens;
        if (l < 4)
            *reinterpret_cast<uint32_t *>(tile + (is_v ? kv4_v_word(nb, t, b, l) : kv4_k_word(nb, t, b, l))) = half | high << 4;
        else if (l == 4)
            *reinterpret_cast<uint16_t *>(tile + (is_v ? kv4_v_scale(nb, t, b) : kv4_k_scale(nb, t, b))) =
                bad ? uint16_t(0x7e00) : float_to_half_bits(d);
    }
}

__global__ void __launch_bounds__(256) kv4_load_kernel(const Kv4RowsArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned nb = a.c.dim / 32, per_row = a.c.n_kv * nb * 2;
    const unsigned long long total = (unsigned long long)a.n * per_row * 8;
    for (unsigned long long i = (unsigned long long)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (unsigned long long)gridDim.x * 256) {
        const unsigned long long blk = i / 8;
        const unsigned l = unsigned(i % 8), row = unsigned(blk / per_row), in_row = unsigned(blk % per_row);
        const bool is_v = in_row >= per_row / 2;
        const unsigned hb = is_v ? in_row - per_row / 2 : in_row, head = hb / nb, b = hb % nb;
        const unsigned slot = a.slots[row];
        if (slot == kNoSlot) continue;
        if (slot / a.c.page >= a.c.n_pages) {
            tell(a.status, kServeSlot);
            continue;
        }
        const uint8_t *tile = tile_of(a.c, slot, head);
        const unsigned t = slot % a.c.page % kTileTokens, w = l & 3;
        const uint32_t word = *reinterpret_cast<const uint32_t *>(tile + (is_v ? kv4_v_word(nb, t, b, w) : kv4_k_word(nb, t, b, w)));
        const float d = half_bits_to_float(*reinterpret_cast<const uint16_t *>(tile + (is_v ? kv4_v_scale(nb, t, b) : kv4_k_scale(nb, t, b))));
        float *dst = (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) + hb * 32 + l * 4;
        for (unsigned e = 0; e < 4; ++e) dst[e] = fmul(float(int(word >> (8 * e + (l & 4)) & 15) - 8), d);
    }
}

// ---- kv4_reorder ----------------------------------------------------------------------------------------------------
// In place, so every thread owns one column (16 bytes of the tail pages, or one table entry) across the request's beams:
// it reads the column of every beam's parent before it writes any.
template <int W>
__global__ void __launch_bounds__(128) kv4_reorder_kernel(const Kv4ReorderArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned req = blockIdx.y, layer = blockIdx.z, col = blockIdx.x * 128 + threadIdx.x, row0 = req * a.beams;
    const unsigned len = a.kv_len[row0], full = len / a.c.page, tail = len % a.c.page;
    if (full + (tail != 0) > a.stride) {
        if (col == 0) tell(a.status, kServeRequest);
        return;
    }
    if (layer == a.layers) {  // the table's entries of full pages
        for (unsigned e = col; e < full; e += gridDim.x * 128) {
            uint32_t v[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const unsigned p = unsigned(i) < a.beams ? a.parent[row0 + i] : kNoSlot;
                v[i] = p < a.beams ? a.table[size_t(row0 + p) * a.stride + e] : 0u;
            }
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (unsigned(i) < a.beams && a.parent[row0 + i] < a.beams) a.table[size_t(row0 + i) * a.stride + e] = v[i];
        }
        if (col == 0)
            for (unsigned i = 0; i < a.beams; ++i)
                if (a.parent[row0 + i] >= a.beams && a.parent[row0 + i] != kNoSlot) tell(a.status, kServeParent);
        return;
    }
    const unsigned tile_bytes = kv4_tile_bytes(a.c.dim), per_head = (tail + kTileTokens - 1) / kTileTokens * tile_bytes / 16;
    if (tail == 0 || col >= a.c.n_kv * per_head) return;
    const unsigned head = col / per_head;
    const size_t page_bytes = size_t(a.c.n_kv) * (a.c.page / kTileTokens) * tile_bytes;
    uint8_t *at = a.c.base + layer * a.layer_bytes + size_t(head) * (a.c.page / kTileTokens) * tile_bytes + size_t(col % per_head) * 16;
    uint4 v[W];
    unsigned from[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const unsigned p = unsigned(i) < a.beams ? a.parent[row0 + i] : kNoSlot;
        from[i] = p < a.beams && p != unsigned(i) ? a.table[size_t(row0 + p) * a.stride + full] : kNoSlot;
        if (from[i] < a.c.n_pages) v[i] = *reinterpret_cast<const uint4 *>(at + from[i] * page_bytes);
        else if (p < a.beams && p != unsigned(i)) tell(a.status, kServePage);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (from[i] >= a.c.n_pages) continue;
        const unsigned to = a.table[size_t(row0 + i) * a.stride + full];
        if (to < a.c.n_pages) *reinterpret_cast<uint4 *>(at + to * page_bytes) = v[i];
        else tell(a.status, kServePage);
    }
}

}  // namespace

cudaError_t launch_block_map(const BlockMapArgs &a, cudaStream_t st) {
    return launch_pdl(block_map_kernel, dim3(1), dim3(1024), 0, st, a);
}

static dim3 rows_grid(const Kv4RowsArgs &a) {
    const unsigned long long threads = (unsigned long long)a.n * a.c.n_kv * (a.c.dim / 32) * 16;
    const unsigned long long g = (threads + 255) / 256;
    return dim3(unsigned(g < 148 * 8 ? g : 148 * 8));
}
cudaError_t launch_kv4_store(const Kv4RowsArgs &a, cudaStream_t st) {
    return launch_pdl(kv4_store_kernel, rows_grid(a), dim3(256), 0, st, a);
}
cudaError_t launch_kv4_load(const Kv4RowsArgs &a, cudaStream_t st) {
    return launch_pdl(kv4_load_kernel, rows_grid(a), dim3(256), 0, st, a);
}

cudaError_t launch_kv4_reorder(const Kv4ReorderArgs &a, cudaStream_t st) {
    const unsigned cols = a.c.n_kv * (a.c.page / kTileTokens) * kv4_tile_bytes(a.c.dim) / 16;
    const dim3 grid((cols + 127) / 128, a.n_req, a.layers + 1);
    if (a.beams <= 4) return launch_pdl(kv4_reorder_kernel<4>, grid, dim3(128), 0, st, a);
    if (a.beams <= 8) return launch_pdl(kv4_reorder_kernel<8>, grid, dim3(128), 0, st, a);
    if (a.beams <= 16) return launch_pdl(kv4_reorder_kernel<16>, grid, dim3(128), 0, st, a);
    return launch_pdl(kv4_reorder_kernel<32>, grid, dim3(128), 0, st, a);
}

}  // namespace b200q
