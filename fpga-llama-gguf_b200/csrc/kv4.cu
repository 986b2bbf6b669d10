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
// table row come from the free list in request order: two exclusive sums over the requests (rows, fresh pages), which one
// CTA forms, then one slot a row. Latency is all that counts in the sums; the rows are 8 bytes each, so up to kMapRows of
// them the same CTA writes (one launch), more are shared out by a second kernel. 64 requests of a token 10.6 us, 512 with
// prompts 13.1 us, of which 8 are the host's (the stream's handle, 16 pointers checked, a launch).
constexpr unsigned kMapRows = 4096;

// rows j0 .. j0 + 3: each one's request is found once, by bisection, and then followed
__device__ __forceinline__ void map_rows(const BlockMapArgs &a, unsigned j0) {
    const unsigned rows = a.q_start[a.n_req], most = 0xFFFFFFFFu / a.page;  // pages whose slots 32 bits count
    unsigned slot[4], pos[4];
    unsigned r = 0;
    if (j0 < rows) {
        unsigned hi = a.n_req;  // the last request that starts at or before row j0
        while (hi - r > 1) {
            const unsigned mid = (r + hi) / 2;
            if (a.q_start[mid] <= j0) r = mid;
            else hi = mid;
        }
    }
    unsigned next = j0 < rows ? a.q_start[r + 1] : 0, start = j0 < rows ? a.q_start[r] : 0, past = j0 < rows ? a.past[r] : 0;
    unsigned block = ~0u, page = kNoSlot;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        const unsigned j = j0 + i;
        slot[i] = kNoSlot;
        pos[i] = 0;
        if (j >= rows) continue;
        while (next <= j) {
            start = next;
            ++r;
            next = a.q_start[r + 1];
            past = a.past[r];
            block = ~0u;
        }
        const unsigned long long p = (unsigned long long)past + (j - start);
        if (p >= (unsigned long long)a.stride * a.page) continue;
        pos[i] = unsigned(p);
        const unsigned b = pos[i] / a.page;
        if (b != block) page = a.table[size_t(r) * a.stride + b], block = b;
        if (page < most) slot[i] = page * a.page + (pos[i] - b * a.page);
        else if (page != kNoSlot) tell(a.status, kServePage);
    }
    if (j0 + 4 <= a.n_rows && ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0) {
        *reinterpret_cast<uint4 *>(a.slots + j0) = make_uint4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<uint4 *>(a.positions + j0) = make_uint4(pos[0], pos[1], pos[2], pos[3]);
    } else {
        for (unsigned i = 0; i < 4 && j0 + i < a.n_rows; ++i) a.slots[j0 + i] = slot[i], a.positions[j0 + i] = pos[i];
    }
}

__global__ void __launch_bounds__(1024) block_map_kernel(const BlockMapArgs a, bool rows_too) {
    __shared__ unsigned long long warp_rows[32], warp_need[32];
    __shared__ unsigned long long done_rows, done_need;
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned long long cap = (unsigned long long)a.stride * a.page;
    const unsigned cursor = *a.cursor_in;
    if (tid == 0) done_rows = done_need = 0;
    for (unsigned r0 = 0; r0 < a.n_req; r0 += blockDim.x) {
        const unsigned r = r0 + tid;
        unsigned fresh = 0, first = 0, last = 0;
        if (r < a.n_req) {
            const unsigned past = a.past[r];
            fresh = a.fresh[r];
            unsigned long long kv = (unsigned long long)past + fresh;
            if (kv > cap) {
                kv = cap;
                tell(a.status, kServeShort);
            }
            a.kv_len[r] = unsigned(kv);
            first = past / a.page + (past % a.page != 0);
            last = unsigned(kv) / a.page + (unsigned(kv) % a.page != 0);
            if (last < first) last = first;
        }
        unsigned long long rows = fresh, need = last - first;
        for (unsigned o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(~0u, rows, o), y = __shfl_up_sync(~0u, need, o);
            if (lane >= o) rows += x, need += y;
        }
        __syncthreads();  // the sums of the turn before are read, done_* written
        if (lane == 31) warp_rows[warp] = rows, warp_need[warp] = need;
        __syncthreads();
        unsigned long long row0 = done_rows + rows - fresh, need0 = done_need + need - (last - first);
        if (warp) {  // the warps before this one: a lane each, then added up
            unsigned long long x = lane < warp ? warp_rows[lane] : 0, y = lane < warp ? warp_need[lane] : 0;
            for (unsigned o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o), y += __shfl_xor_sync(~0u, y, o);
            row0 += x, need0 += y;
        }
        if (r < a.n_req) {
            a.q_start[r] = unsigned(row0);
            if (last > first && cursor + need0 + (last - first) > a.n_free) tell(a.status, kServeShort);
        }
        // a request's pages: a few by its thread, more by its warp
        auto take = [&](unsigned req, unsigned b, unsigned from, unsigned long long at) {
            const unsigned long long f = cursor + at + (b - from);
            a.table[size_t(req) * a.stride + b] = f < a.n_free ? a.free_pages[f] : kNoSlot;
        };
        const bool few = last - first <= 8;
        if (few)
            for (unsigned b = first; b < last; ++b) take(r, b, first, need0);
        for (unsigned many = __ballot_sync(~0u, !few); many; many &= many - 1) {
            const unsigned of = __ffs(many) - 1, from = __shfl_sync(~0u, first, of), to = __shfl_sync(~0u, last, of);
            const unsigned long long at = __shfl_sync(~0u, need0, of);
            for (unsigned b = from + lane; b < to; b += 32) take(r - lane + of, b, from, at);
        }
        __syncthreads();
        if (tid == blockDim.x - 1) {
            done_rows = row0 + fresh;
            done_need = need0 + (last - first);
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.q_start[a.n_req] = unsigned(done_rows);
        const unsigned long long c = cursor + done_need;
        *a.cursor_out = unsigned(c < a.n_free ? c : (cursor < a.n_free ? a.n_free : cursor));
        if (done_rows > a.n_rows) tell(a.status, kServeRequest);
    }
    if (!rows_too) return;
    __syncthreads();
    for (unsigned j = tid * 4; j < a.n_rows; j += blockDim.x * 4) map_rows(a, j);
}

__global__ void __launch_bounds__(256) map_rows_kernel(const BlockMapArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned j = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (j < a.n_rows) map_rows(a, j);
}

// ---- kv4_store / kv4_load -------------------------------------------------------------------------------------------
// Eight lanes take a 32-dim block (four values each); lane l < 4 writes word l, whose high nibbles lane l + 4 holds.
// The quantizer is Q4_0's: d = x[argmax |x|] / -8 (the first on ties), code = min(15, trunc(x (1 / d) + 8.5)), every step
// rounded to FP32 by itself; a block that holds a NaN or an infinity gets a NaN scale, so that it reads back as NaN.
// Both are bound by memory once there are rows enough: 8192 tokens of 8 heads of 128 stored and read back (145 MB) take 39 us,
// 22 at the measured copy rate. What kept them from it was arithmetic (50 us): each thread's own divisions of the slot by the
// page, the search for the largest value's sign, conversions at a quarter of the rate of additions. It still bounds them (72% and
// 77% of issue slots): eight lanes a block do every block's division eight times and half of them write no code word, in the
// load two lanes read each word. Two or eight rows a turn took 43 and 45 us, a quarter of the CTAs 48.
//
// A thread stays with its values of its block and goes down the rows, kRowsTurn at a time, so that what places them in a
// row is worked out once and several rows' loads are on their way together.
constexpr unsigned kRowsTurn = 4;

struct RowPlace {
    unsigned head, b, l;  // KV head, block of the head, lane of the block
    bool is_v, real;
    size_t in_row;        // of the thread's values, in floats
    uint8_t *head0;       // its KV head's first tile of page 0
    unsigned word, scale; // of token 0 in a tile: byte offsets of word l % 4 and of the scale
};
__device__ __forceinline__ RowPlace row_place(const Kv4RowsArgs &a) {
    const unsigned nb = a.c.dim / 32, half = a.c.n_kv * nb, i = blockIdx.x * 256 + threadIdx.x, blk = i / 8;
    RowPlace p;
    p.real = blk < 2 * half;
    p.is_v = blk >= half;
    const unsigned hb = p.is_v ? blk - half : blk;
    p.l = i % 8;
    p.head = hb / nb;
    p.b = hb % nb;
    p.in_row = size_t(hb) * 32 + p.l * 4;
    p.head0 = a.c.base + size_t(p.head) * (a.c.page / kTileTokens) * kv4_tile_bytes(a.c.dim);
    p.word = p.is_v ? kv4_v_word(nb, 0, p.b, p.l % 4) : kv4_k_word(nb, 0, p.b, p.l % 4);
    p.scale = p.is_v ? kv4_v_scale(nb, 0, p.b) : kv4_k_scale(nb, 0, p.b);
    return p;
}

// Where the turn's rows lie: lane i works it out for row i, with the divisions, and the warp asks it.
struct Spots {
    unsigned long long tile;  // of KV head 0, bytes from the pool's start
    unsigned t;               // its token there; kTileTokens: no slot
    __device__ __forceinline__ Spots(const Kv4RowsArgs &a, unsigned row0) : tile(0), t(kTileTokens) {
        const unsigned i = threadIdx.x & 31, slot = i < kRowsTurn && row0 + i < a.n ? a.slots[row0 + i] : kNoSlot;
        if (slot == kNoSlot) return;
        const unsigned page = slot / a.c.page, at = slot - page * a.c.page, tiles = a.c.page / kTileTokens;
        if (page >= a.c.n_pages) {
            tell(a.status, kServeSlot);
            return;
        }
        tile = ((unsigned long long)page * a.c.n_kv * tiles + at / kTileTokens) * kv4_tile_bytes(a.c.dim);
        t = at % kTileTokens;
    }
    __device__ __forceinline__ unsigned token(unsigned i) const { return __shfl_sync(~0u, t, i); }
    __device__ __forceinline__ unsigned long long at(unsigned i) const { return __shfl_sync(~0u, tile, i); }
};
// token t's word and scale behind token 0's
__device__ __forceinline__ unsigned word_of(const RowPlace &p, unsigned nb, unsigned t) {
    const unsigned row = kv4_plane_blocks(nb, p.b / 4) * 4;
    return p.word + row * (p.is_v ? (t / 8 * 2 + t % 2) * 16 + t / 2 % 4 : t * 4);
}

template <bool kWide>  // rows on 16 bytes
__global__ void __launch_bounds__(256) kv4_store_kernel(const Kv4RowsArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const RowPlace p = row_place(a);
    const unsigned nb = a.c.dim / 32;
    const float *from = (p.is_v ? a.v : a.k) + p.in_row;
    const size_t stride = p.is_v ? a.v_stride : a.k_stride;
    for (unsigned row0 = blockIdx.y * kRowsTurn; row0 < a.n; row0 += gridDim.y * kRowsTurn) {
        float x[kRowsTurn][4];
#pragma unroll
        for (unsigned i = 0; i < kRowsTurn; ++i) {
            const bool in = p.real && row0 + i < a.n;
            const float *src = from + (row0 + i) * stride;
            if (kWide && in) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(src));
                x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
            } else {
                for (unsigned e = 0; e < 4; ++e) x[i][e] = in ? src[e] : 0.0f;
            }
        }
        const Spots spots(a, row0);  // while the values come
#pragma unroll
        for (unsigned i = 0; i < kRowsTurn; ++i) {
            float amax = fmaxf(fmaxf(fabsf(x[i][0]), fabsf(x[i][1])), fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
#pragma unroll
            for (unsigned o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
            // The sign of the first value that is as large, and whether one is none (fmaxf passes a NaN over)
            float mine = x[i][3];
#pragma unroll
            for (int e = 2; e >= 0; --e) mine = fabsf(x[i][e]) == amax ? x[i][e] : mine;
            const unsigned has = __ballot_sync(~0u, fabsf(mine) == amax) >> (threadIdx.x & 24) & 0xff, minus = __ballot_sync(~0u, mine < 0.0f) >> (threadIdx.x & 24);
            const float zero = fmaf(x[i][0], 0.0f, fmaf(x[i][1], 0.0f, fmaf(x[i][2], 0.0f, x[i][3] * 0.0f)));
            const bool bad = __ballot_sync(~0u, zero != 0.0f) >> (threadIdx.x & 24) & 0xff;
            const float d = amax * (minus & has & (0u - has) ? 0.125f : -0.125f), inv = d != 0.0f ? fdiv(1.0f, d) : 0.0f;
            uint32_t code[4];
#pragma unroll
            for (unsigned e = 0; e < 4; ++e)  // (to an integer by an addition that drops what is behind the point; a NaN: 0)
                code[e] = __float_as_uint(__fadd_rz(fminf(fmaxf(fadd(fmul(x[i][e], inv), 8.5f), 0.0f), 15.0f), 0x1p23f));
            const uint32_t half = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
            const uint32_t high = __shfl_down_sync(~0u, half, 4);
            const unsigned tok = spots.token(i);
            uint8_t *tile = p.head0 + spots.at(i);
            if (tok == kTileTokens || !p.real) continue;
            if (p.l < 4)
                *reinterpret_cast<uint32_t *>(tile + word_of(p, nb, tok)) = half | high << 4;
            else if (p.l == 4)
                *reinterpret_cast<uint16_t *>(tile + p.scale + tok * nb * 2) =
                    bad ? uint16_t(0x7e00) : float_to_half_bits(d);
        }
    }
}

template <bool kWide>
__global__ void __launch_bounds__(256) kv4_load_kernel(const Kv4RowsArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const RowPlace p = row_place(a);
    const unsigned nb = a.c.dim / 32;
    float *to = (p.is_v ? a.v : a.k) + p.in_row;
    const size_t stride = p.is_v ? a.v_stride : a.k_stride;
    for (unsigned row0 = blockIdx.y * kRowsTurn; row0 < a.n; row0 += gridDim.y * kRowsTurn) {
        uint32_t word[kRowsTurn];
        uint16_t scale[kRowsTurn];
        bool some[kRowsTurn];
        const Spots spots(a, row0);
#pragma unroll
        for (unsigned i = 0; i < kRowsTurn; ++i) {
            const unsigned tok = spots.token(i);
            const uint8_t *tile = p.head0 + spots.at(i);
            some[i] = tok != kTileTokens && p.real;
            if (!some[i]) continue;
            word[i] = *reinterpret_cast<const uint32_t *>(tile + word_of(p, nb, tok));
            scale[i] = *reinterpret_cast<const uint16_t *>(tile + p.scale + tok * nb * 2);
        }
#pragma unroll
        for (unsigned i = 0; i < kRowsTurn; ++i) {
            if (!some[i]) continue;
            const float d = half_bits_to_float(scale[i]);
            float x[4];
#pragma unroll
            for (unsigned e = 0; e < 4; ++e)   // 2^23 + code, less 2^23 + 8
                x[e] = fmul(__uint_as_float((word[i] >> (8 * e + (p.l & 4)) & 15) | 0x4b000000u) - 8388616.0f, d);
            float *dst = to + (row0 + i) * stride;
            if (kWide) __stcs(reinterpret_cast<float4 *>(dst), make_float4(x[0], x[1], x[2], x[3]));
            else
                for (unsigned e = 0; e < 4; ++e) dst[e] = x[e];
        }
    }
}

// ---- kv4_reorder ----------------------------------------------------------------------------------------------------
// In place, so every thread owns one column (16 bytes of the tail pages, or one table entry) across the request's beams:
// it reads the column of every beam's parent before it writes any. One launch for table and tails; the host's part bounds
// small calls (9.9 us).
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

unsigned block_map_launches(const BlockMapArgs &a) { return a.n_rows <= kMapRows ? 1 : 2; }

cudaError_t launch_block_map(const BlockMapArgs &a, cudaStream_t st) {
    const bool one = a.n_rows <= kMapRows;
    const unsigned most = one && a.n_rows / 4 > a.n_req ? a.n_rows / 4 : a.n_req, threads = most <= 128 ? 128 : most <= 512 ? 512 : 1024;
    const cudaError_t e = launch_pdl(a.pdl, block_map_kernel, dim3(1), dim3(threads), 0, st, a, one);
    if (one || e != cudaSuccess) return e;
    return launch_pdl(a.pdl, map_rows_kernel, dim3((a.n_rows + 1023) / 1024), dim3(256), 0, st, a);
}

// x: the values of a row; y: the rows, as many at a time as fill the GPU a few times over
static dim3 rows_grid(const Kv4RowsArgs &a) {
    const unsigned x = (a.c.n_kv * (a.c.dim / 32) * 16 + 255) / 256, turns = (a.n + kRowsTurn - 1) / kRowsTurn, y = 148 * 16 / x + 1;
    return dim3(x, turns < y ? turns : y);
}
static bool wide_rows(const Kv4RowsArgs &a) {
    return ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | a.k_stride * 4 | a.v_stride * 4) & 15) == 0;
}
cudaError_t launch_kv4_store(const Kv4RowsArgs &a, cudaStream_t st) {
    return launch_pdl(a.pdl, wide_rows(a) ? kv4_store_kernel<true> : kv4_store_kernel<false>, rows_grid(a), dim3(256), 0, st, a);
}
cudaError_t launch_kv4_load(const Kv4RowsArgs &a, cudaStream_t st) {
    return launch_pdl(a.pdl, wide_rows(a) ? kv4_load_kernel<true> : kv4_load_kernel<false>, rows_grid(a), dim3(256), 0, st, a);
}

cudaError_t launch_kv4_reorder(const Kv4ReorderArgs &a, cudaStream_t st) {
    const unsigned cols = a.c.n_kv * (a.c.page / kTileTokens) * kv4_tile_bytes(a.c.dim) / 16;
    const dim3 grid((cols + 127) / 128, a.n_req, a.layers + 1);
    if (a.beams <= 4) return launch_pdl(a.pdl, kv4_reorder_kernel<4>, grid, dim3(128), 0, st, a);
    if (a.beams <= 8) return launch_pdl(a.pdl, kv4_reorder_kernel<8>, grid, dim3(128), 0, st, a);
    if (a.beams <= 16) return launch_pdl(a.pdl, kv4_reorder_kernel<16>, grid, dim3(128), 0, st, a);
    return launch_pdl(a.pdl, kv4_reorder_kernel<32>, grid, dim3(128), 0, st, a);
}

}  // namespace b200q
