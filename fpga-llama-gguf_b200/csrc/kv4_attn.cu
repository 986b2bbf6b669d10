// Attention over the paged 4-bit cache.
//
// Row i of request r (its new tokens are the last of its kv_len tokens) stands at position p = kv_len - new + i and sees
// the keys (p - window, p] (window 0: [0, p]). For a query head h of KV head g = h / (n_head / n_kv)
//   y = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = scale q . k_t,  m = max_t s_t
// in one pass over the keys with the running m and sum. A row that sees nothing is zero.
//
// A value is d_b (c - 8) with one d per 32-dim block b, so both products run on integers of four bits, exact in FP16,
// and the scales meet FP32 numbers only:
//   s_t  = sum_b d_tb (sum_i q_i (c_ti - 8))      per block a 16 x 8 x 32 matrix product, scaled and added in FP32
//   y_i  = sum_t (p_t d_tb) (c_ti - 8)            the weight of a token differs by block, not by dim
// The FP32 factors (q, and p_t d_tb) are split into two FP16 numbers, 22 bits in all, which sit in rows r and r + 8 of the
// matrix instruction's A operand: 8 query rows fill its 16 rows, and FP32 accuracy costs no second instruction. q's
// rows are first scaled by a power of two to below 2^11, and their lower parts by 2048.
#include <cuda_runtime.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kv4.cuh"
#include "pipeline.cuh"
#include "serve.h"

namespace b200q {

// More requests than this, and a launch's schedule would not fit its shared memory.
constexpr unsigned kAttnMaxReq = 4096;

namespace {

constexpr unsigned kWarps = 4, kThreads = kWarps * 32;
constexpr unsigned kMaxChunkTiles = 256;  // a warp adds at most 64 tiles into its accumulators before they are merged in FP32
constexpr unsigned kMergeChunk = 256;    // chunks whose factors the merge holds at a time
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void tell(uint32_t *status, unsigned bit) {
    if (status) atomicOr(status, bit);
}

struct Plan {
    unsigned max_items = 0;  // items the workspace holds partial results for
    unsigned target = 0;     // items wanted in all
    unsigned rows = 8;       // query rows (token, head) of an item
};

// ---- the schedule ---------------------------------------------------------------------------------------------------
// An item is a chunk of the keys for up to 8 (or 16) query rows of one KV head. The lengths are on the device, so every
// CTA counts the tiles itself, takes the chunk that gives about `target` items in all, and finds its items by
// their prefix sums. A request outside the stated bounds has no items.
struct Request {
    unsigned start = 0, fresh = 0, len = 0, groups = 0, span = 0;  // span: tiles that a group of rows sees at most
};

__device__ __forceinline__ Request request_of(const Kv4AttnArgs &a, unsigned r, unsigned rows, bool report) {
    Request q;
    const unsigned s = a.q_start[r], e = a.q_start[r + 1], len = a.kv_len[r];
    if (s > e || e > a.n_rows || e - s > a.max_q || len > a.max_kv) {
        if (report) tell(a.status, kServeRequest);
        return q;
    }
    const unsigned group = a.n_head / a.c.n_kv;
    q.start = s;
    q.fresh = e - s;
    q.len = len;
    q.groups = ((e - s) * group + rows - 1) / rows;
    q.span = (len + kTileTokens - 1) / kTileTokens;
    if (a.window) {
        const unsigned long long seen = (unsigned long long)a.window + (rows + group - 1) / group;
        if (seen + 2 * kTileTokens < len) q.span = unsigned(seen / kTileTokens) + 2;
    }
    return q;
}

struct Schedule {
    unsigned chunk = 0, total = 0;  // tiles of an item; items
};

__device__ __forceinline__ unsigned splits_of(const Request &q, unsigned chunk) {
    const unsigned n = (q.span + chunk - 1) / chunk;
    return n ? n : 1;
}

// prefix[r]: items before request r (n_req + 1 entries), units[r]: groups of rows x KV heads before it (or null)
__device__ Schedule make_schedule(const Kv4AttnArgs &a, const Plan &plan, unsigned *prefix, unsigned *units) {
    __shared__ unsigned long long tiles_in[kWarps];
    __shared__ unsigned items_in[kWarps], units_in[kWarps];
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (a.n_req + kThreads - 1) / kThreads;
    const unsigned r0 = tid * per < a.n_req ? tid * per : a.n_req, r1 = r0 + per < a.n_req ? r0 + per : a.n_req;
    unsigned long long tiles = 0;
    for (unsigned r = r0; r < r1; ++r) {
        const Request q = request_of(a, r, plan.rows, blockIdx.x == 0);
        tiles += (unsigned long long)q.groups * q.span;
    }
    for (unsigned o = 16; o; o >>= 1) tiles += __shfl_xor_sync(~0u, tiles, o);
    if (lane == 0) tiles_in[warp] = tiles;
    __syncthreads();
    tiles = 0;
    for (unsigned w = 0; w < kWarps; ++w) tiles += tiles_in[w];
    const unsigned long long even = (tiles * a.c.n_kv + plan.target - 1) / plan.target;
    Schedule s;
    s.chunk = even >= kMaxChunkTiles ? kMaxChunkTiles : (unsigned(even) + kWarps - 1) / kWarps * kWarps;
    if (s.chunk < kWarps) s.chunk = kWarps;
    unsigned items = 0, un = 0;
    for (unsigned r = r0; r < r1; ++r) {
        const Request q = request_of(a, r, plan.rows, false);
        items += q.groups * splits_of(q, s.chunk) * a.c.n_kv;
        un += q.groups * a.c.n_kv;
    }
    unsigned is = items, us = un;
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(~0u, is, o), y = __shfl_up_sync(~0u, us, o);
        if (lane >= o) is += x, us += y;
    }
    if (lane == 31) items_in[warp] = is, units_in[warp] = us;
    __syncthreads();
    is -= items, us -= un;
    for (unsigned w = 0; w < warp; ++w) is += items_in[w], us += units_in[w];
    for (unsigned r = r0; r < r1; ++r) {
        const Request q = request_of(a, r, plan.rows, false);
        prefix[r] = is;
        if (units) units[r] = us;
        is += q.groups * splits_of(q, s.chunk) * a.c.n_kv;
        us += q.groups * a.c.n_kv;
        if (r == a.n_req - 1) {
            prefix[a.n_req] = is;
            if (units) units[a.n_req] = us;
        }
    }
    __syncthreads();
    s.total = prefix[a.n_req];
    return s;
}

__device__ __forceinline__ unsigned find(const unsigned *prefix, unsigned n, unsigned i) {
    unsigned lo = 0, hi = n;
    while (hi - lo > 1) {
        const unsigned mid = (lo + hi) / 2;
        if (prefix[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The keys that a group of rows sees, and its tiles from the first one on.
struct GroupSpan {
    long long lo = 0, hi = -1;  // of its first row, of its last row
    unsigned tile0 = 0, tiles = 0;
};
__device__ __forceinline__ GroupSpan span_of(const Kv4AttnArgs &a, const Request &q, unsigned group, unsigned rows) {
    const unsigned per = a.n_head / a.c.n_kv, all = q.fresh * per, r0 = group * rows, r1 = r0 + rows < all ? r0 + rows : all;
    GroupSpan s;
    const long long base = (long long)q.len - q.fresh;
    s.hi = base + (r1 - 1) / per;
    s.lo = a.window && base + r0 / per + 1 > (long long)a.window ? base + r0 / per + 1 - a.window : 0;
    if (s.hi >= 0) {
        s.tile0 = unsigned(s.lo / kTileTokens);
        s.tiles = unsigned(s.hi / kTileTokens) - s.tile0 + 1;
    }
    return s;
}

// ---- the tile product -----------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// two FP32 multiply-adds in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2(half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ half2 as_h2(uint32_t x) { return *reinterpret_cast<half2 *>(&x); }

// Two nibbles of a word, bits 0..3 and 16..19 (low) or 4..7 and 20..23 (high), as FP16.
// K: left as they are they read c 2^-24 (16 c 2^-24), and the 8 that a code stands above its value comes off in the sum.
__device__ __forceinline__ uint32_t low_raw(uint32_t x) { return x & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_raw(uint32_t x) { return x & 0x00f000f0u; }
// V (whose sums run over many tokens, where that 8 would swamp them): put into the mantissa of 1024 they read 1024 + c
// (1024 + 16 c); less 1032 (1152) that is c - 8 (16 (c - 8)), exactly.
__device__ __forceinline__ uint32_t low_codes(uint32_t x) {
    uint32_t y;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(y) : "r"(x));
    return h2(__hsub2(as_h2(y), as_h2(0x64086408u)));
}
__device__ __forceinline__ uint32_t high_codes(uint32_t x) {
    uint32_t y;
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(y) : "r"(x));
    return h2(__hsub2(as_h2(y), as_h2(0x64806480u)));
}

// x = hi + lo / 2048, both FP16 pairs
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    const half2 h = __floats2half2_rn(x0, x1);
    const float2 b = __half22float2(h);
    hi = h2(h);
    lo = h2(__floats2half2_rn((x0 - b.x) * 2048.0f, (x1 - b.y) * 2048.0f));
}

// N words of shared memory, in the widest loads their alignment allows (N = 4, 8: 16 bytes, N = 2: 8 bytes)
template <int N>
__device__ __forceinline__ void load_words(uint32_t *w, const uint8_t *at) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(at + 4 * i);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(at + 4 * i);
            w[i] = x.x, w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t *>(at + 4 * i);
    }
}
// halves i and j of an array of words as a pair
__device__ __forceinline__ half2 pair_at(const uint32_t *w, int i, int j) {
    return as_h2(__byte_perm(w[i >> 1], w[j >> 1], (i & 1 ? 0x32u : 0x10u) | (j & 1 ? 0x7600u : 0x5400u)));
}
// half i of an array of words
__device__ __forceinline__ float half_at(const uint32_t *w, int i) {
    return __half2float(__ushort_as_half(uint16_t(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu)));
}

template <int NB, int MT>
struct Shape {
    static constexpr int kTile = NB * 576;                       // bytes of a tile
    static constexpr int kSlots = NB <= 2 ? 8 : NB <= 4 ? 6 : 4;  // tiles a warp has on their way
    static constexpr bool kQInRegs = NB * MT <= 4;
    static constexpr int kQBytes = kQInRegs ? 0 : MT * NB * 3 * 32 * 16;  // per block: two k-steps of q, and the sums' start
    static constexpr int kOutBytes = kWarps * MT * 8 * (NB * 32 + 2) * 4;  // the warps' results, in the ring's place
    static constexpr int kRing = kWarps * kSlots * kTile;
    static constexpr int kSmem = kQBytes + (kRing > kOutBytes ? kRing : kOutBytes);
};

// A warp takes every fourth tile of its CTA's chunk, with a running maximum, sum and output of its own; it fetches its
// tiles itself (one bulk copy each), so that nothing in the loop waits for another warp. Lane (g, t) = (lane / 4, lane % 4).
template <int NB, int MT>
__global__ void __launch_bounds__(kThreads) kv4_attn_kernel(const Kv4AttnArgs a, const Plan plan) {
    using S = Shape<NB, MT>;
    constexpr int kPlanes = (NB + 3) / 4, D = NB * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][S::kSlots];
    __shared__ float m_of[kWarps][MT * 8], l_of[kWarps][MT * 8];
    unsigned *prefix = reinterpret_cast<unsigned *>(smem + S::kSmem);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const unsigned per = a.n_head / a.c.n_kv, tiles_per_page = a.c.page / kTileTokens;
    uint8_t *ring = smem + S::kQBytes + warp * S::kSlots * S::kTile;
    if (tid == 0) {
        for (unsigned w = 0; w < kWarps; ++w)
            for (int i = 0; i < S::kSlots; ++i) mbar_init(&bars[w][i], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    const Schedule sched = make_schedule(a, plan, prefix, nullptr);  // its barriers also cover the mbarriers' start
    unsigned done = 0;  // tiles this warp has taken from its ring so far (slot and phase go by it)
    bool late = false;

    for (unsigned item = blockIdx.x; item < sched.total; item += gridDim.x) {
        const unsigned r = find(prefix, a.n_req, item);
        const Request rq = request_of(a, r, plan.rows, false);
        unsigned in = item - prefix[r];
        const unsigned head = in % a.c.n_kv;
        in /= a.c.n_kv;
        const unsigned group = in % rq.groups, split = in / rq.groups;
        const GroupSpan sp = span_of(a, rq, group, plan.rows);
        const unsigned n_split = (sp.tiles + sched.chunk - 1) / sched.chunk;
        if (split && split >= n_split) continue;
        const unsigned t0 = split * sched.chunk, t1 = t0 + sched.chunk < sp.tiles ? t0 + sched.chunk : sp.tiles;
        const unsigned mine = t0 + warp < t1 ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;  // tiles of this warp
        const uint32_t *table = a.table + size_t(r) * a.stride;
        const uint8_t *head_base = a.c.base + size_t(head) * tiles_per_page * S::kTile;
        const size_t page_bytes = size_t(a.c.n_kv) * tiles_per_page * S::kTile;

        // the k-th tile of this warp: lane k % 32 keeps where it lies
        const uint8_t *where = nullptr;
        auto look_up = [&](unsigned k) {
            where = nullptr;
            if (k < mine) {
                const unsigned tile = sp.tile0 + t0 + warp + k * kWarps, page = table[tile / tiles_per_page];
                if (page < a.c.n_pages) where = head_base + page * page_bytes + size_t(tile % tiles_per_page) * S::kTile;
                else tell(a.status, kServePage);
            }
        };
        auto fetch = [&](unsigned k) {  // where: of k's 32 tiles
            const uint8_t *src = reinterpret_cast<const uint8_t *>(__shfl_sync(~0u, (unsigned long long)where, k % 32));
            const unsigned slot = (done + k) % S::kSlots;
            if (lane == 0) {
                if (src) {
                    mbar_expect_tx(&bars[warp][slot], S::kTile);
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                     smem_addr(ring + slot * S::kTile)),
                                 "l"(src), "r"(S::kTile), "r"(smem_addr(&bars[warp][slot]))
                                 : "memory");
                } else {
                    mbar_expect_tx(&bars[warp][slot], 0);  // no page: the slot's phase ends at once
                }
            }
            return src != nullptr;
        };
        unsigned present = 0;  // bit s: slot s holds a tile
        look_up(lane);
        unsigned ahead = 0;
        for (; ahead < unsigned(S::kSlots) && ahead < mine; ++ahead) {
            const unsigned slot = (done + ahead) % S::kSlots;
            present = fetch(ahead) ? present | 1u << slot : present & ~(1u << slot);
        }

        // the rows' queries: split, in the order in which a block's words hold the dims
        uint32_t qa[S::kQInRegs ? MT : 1][S::kQInRegs ? NB * 2 : 1][4];
        float start[S::kQInRegs ? MT : 1][S::kQInRegs ? NB : 1][4];  // -8 sum q over a block, of the rows' upper and lower parts
        float scale[MT];
        int pos[MT], low[MT];  // the keys a row sees: [low, pos]
        const unsigned all = rq.fresh * per, row0 = group * plan.rows;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const unsigned row = row0 + m * 8 + g;
            const bool real = row < all;
            const float *src = a.q + (rq.start + (real ? row / per : 0)) * a.q_stride + (head * per + (real ? row % per : 0)) * a.q_head_stride;
            const long long p = (long long)rq.len - rq.fresh + row / per;
            pos[m] = real ? int(p) : -1;
            low[m] = a.window && p + 1 > (long long)a.window ? int(p + 1 - a.window) : 0;
            float x[NB * 2][4], top = 0.0f;
            const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | a.q_stride * 4 | a.q_head_stride * 4) & 15) == 0;
#pragma unroll
            for (int i = 0; i < NB * 2; ++i) {
                const float *at = src + i * 16 + t * 4;
                if (wide) {
                    const float4 v = *reinterpret_cast<const float4 *>(at);
                    x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
                } else {
                    for (int e = 0; e < 4; ++e) x[i][e] = at[e];
                }
            }
#pragma unroll
            for (int i = 0; i < NB * 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[i][e]));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
            top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
            int ex = int(__float_as_uint(top) >> 23) - 127 - 10;  // x / 2^ex is below 2^11
            ex = ex < -110 ? -110 : ex > 100 ? 100 : ex;
            const float down = __uint_as_float(unsigned(127 - ex) << 23);
            scale[m] = a.scale * kLog2e * __uint_as_float(unsigned(127 + 24 + ex) << 23);  // (K's codes come times 2^-24)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float hi = 0.0f, lo = 0.0f;
#pragma unroll
                for (int i = 2 * b; i < 2 * b + 2; ++i) {
                    const float f = i & 1 ? down * 0.0625f : down;  // the high nibbles' codes come times 16
                    uint32_t v[4];
                    split2(x[i][0] * f, x[i][2] * f, v[0], v[1]);
                    split2(x[i][1] * f, x[i][3] * f, v[2], v[3]);
                    const float2 s0 = __half22float2(as_h2(v[0])), s1 = __half22float2(as_h2(v[1])), s2 = __half22float2(as_h2(v[2])),
                                 s3 = __half22float2(as_h2(v[3]));
                    const float up = i & 1 ? 16.0f : 1.0f;
                    hi += up * ((s0.x + s0.y) + (s2.x + s2.y));
                    lo += up * ((s1.x + s1.y) + (s3.x + s3.y));
                    if constexpr (S::kQInRegs) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) qa[m][i][e] = v[e];
                    } else {
                        if (warp == 0) *reinterpret_cast<uint4 *>(smem + ((m * NB * 3 + i) * 32 + lane) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                hi += __shfl_xor_sync(~0u, hi, 1);
                lo += __shfl_xor_sync(~0u, lo, 1);
                hi = -0x1p-21f * (hi + __shfl_xor_sync(~0u, hi, 2));
                lo = -0x1p-21f * (lo + __shfl_xor_sync(~0u, lo, 2));
                if constexpr (S::kQInRegs) {
                    start[m][b][0] = start[m][b][1] = hi;
                    start[m][b][2] = start[m][b][3] = lo;
                } else {
                    if (warp == 0) *reinterpret_cast<float4 *>(smem + ((m * NB * 3 + NB * 2 + b) * 32 + lane) * 16) = make_float4(hi, hi, lo, lo);
                }
            }
        }
        if constexpr (!S::kQInRegs) __syncthreads();

        float o[MT][NB * 4][4], top[MT], sum[MT], limit = 0.0f, lift = 1.0f, lift_d = 1.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            top[m] = -INFINITY;
            sum[m] = 0.0f;
#pragma unroll
            for (int i = 0; i < NB * 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][i][e] = 0.0f;
        }

        // Keys that every row of the group sees need no masks.
        const long long all_low = a.window ? (long long)rq.len - rq.fresh + (row0 + plan.rows < all ? row0 + plan.rows - 1 : all - 1) / per + 1 - a.window : 0;
        const long long all_high = (long long)rq.len - rq.fresh + row0 / per;

        auto take = [&](const uint8_t *tile, int key0, auto masked) {
            constexpr bool kMasked = decltype(masked)::value;
            // scores of the tile's keys 8 j + 2 t + i
            float2 s[MT][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t ds[NB];
                load_words<NB>(ds, tile + NB * 512 + (4 * j + t) * NB * 4);
#pragma unroll
                for (int m = 0; m < MT; ++m) s[m][j] = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int p = 0; p < kPlanes; ++p) {
                    const int nbp = NB - 4 * p < 4 ? NB - 4 * p : 4;
                    uint32_t w[4];
                    const uint8_t *at = tile + p * 1024 + ((8 * j + g) * 4 + t) * nbp * 4;
                    if (nbp == 4) load_words<4>(w, at);
                    if (nbp == 3) load_words<3>(w, at);
                    if (nbp == 2) load_words<2>(w, at);
                    if (nbp == 1) load_words<1>(w, at);
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if (b >= nbp) break;
                        const int bb = 4 * p + b;
                        const uint32_t x8 = w[b] >> 8;
                        const float2 d = make_float2(half_at(ds, bb), half_at(ds, NB + bb));
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            float c[4], e[4];
                            uint32_t q0[4], q1[4];
                            if constexpr (S::kQInRegs) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) q0[i] = qa[m][bb * 2][i], q1[i] = qa[m][bb * 2 + 1][i], c[i] = start[m][bb][i];
                            } else {
                                load_words<4>(q0, smem + ((m * NB * 3 + bb * 2) * 32 + lane) * 16);
                                load_words<4>(q1, smem + ((m * NB * 3 + bb * 2 + 1) * 32 + lane) * 16);
                                load_words<4>(reinterpret_cast<uint32_t *>(c), smem + ((m * NB * 3 + NB * 2 + bb) * 32 + lane) * 16);
                            }
                            mma16816(e, q0, low_raw(w[b]), low_raw(x8), c);
                            mma16816(c, q1, high_raw(w[b]), high_raw(x8), e);
                            const float2 both = fma2(make_float2(c[2], c[3]), make_float2(1.0f / 2048, 1.0f / 2048), make_float2(c[0], c[1]));
                            s[m][j] = fma2(d, both, s[m][j]);
                        }
                    }
                }
            }
            // The running maximum. It moves only when a score passes it, and then to 4 (in powers of two) above the largest, so
            // that it moves seldom; the weights stay below 1.
            float2 pr[MT][2];
            uint32_t seen[MT][2];  // of a pair of keys, as a mask of halves
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int key = key0 + 8 * j + 2 * int(t);
                    s[m][j].x *= scale[m];
                    s[m][j].y *= scale[m];
                    if (kMasked) {
                        const bool x = key >= low[m] && key <= pos[m], y = key + 1 >= low[m] && key + 1 <= pos[m];
                        seen[m][j] = (x ? 0x0000ffffu : 0u) | (y ? 0xffff0000u : 0u);
                        if (!x) s[m][j].x = -INFINITY;
                        if (!y) s[m][j].y = -INFINITY;
                    }
                    mx = fmaxf(mx, fmaxf(s[m][j].x, s[m][j].y));
                }
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
                if (__any_sync(~0u, mx > top[m])) {
                    const float nt = mx > top[m] ? mx + 4.0f : top[m];
                    const float f = top[m] == nt ? 1.0f : exp2_fast(top[m] - nt);  // top -inf: 0
                    sum[m] *= f;
#pragma unroll
                    for (int i = 0; i < NB * 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[m][i][e] *= f;
                    top[m] = nt;
                }
                const float ref = top[m] == -INFINITY ? 0.0f : top[m];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pr[m][j] = make_float2(exp2_fast(s[m][j].x - ref), exp2_fast(s[m][j].y - ref));
                    sum[m] += pr[m][j].x + pr[m][j].y;
                }
            }
            // the weighted sum of the values: keys along k, dims along n
            uint32_t dv[2][NB];
#pragma unroll
            for (int j = 0; j < 2; ++j) load_words<NB>(dv[j], tile + NB * 544 + (4 * j + t) * NB * 4);
            // A weight p d is a product of FP16 pairs: with p = ph + pl, wh = fp16(ph d) and wl = fp16(pl d + (ph d - wh)),
            // where ph d - wh is exact in one FP16 multiply-add. p is lifted by a power of two that keeps the largest weight
            // below 2^14 (`limit`: a power of two that no scale seen so far passes), so that small values keep 22 bits too; scales
            // below 1/16 are lifted as well.
            half2 big2 = __float2half2_rn(0.0f);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (kMasked) {
                        uint32_t any = 0;
#pragma unroll
                        for (int m = 0; m < MT; ++m) any |= seen[m][j];
                        const half2 d = pair_at(dv[j], b, NB + b);
                        big2 = __hmax2(big2, __habs2(as_h2(h2(d) & any)));
                    } else {
                        big2 = __hmax2(big2, __habs2(as_h2(dv[j][b])));
                    }
                }
            float big = fmaxf(__low2float(big2), __high2float(big2));
            if (__any_sync(~0u, big > limit)) {
#pragma unroll
                for (int x = 1; x < 32; x <<= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, x));
                const float was = lift * lift_d;
                limit = __uint_as_float((__float_as_uint(fminf(big, 65504.0f)) & 0x7f800000u) + 0x00800000u);  // the next power of two
                lift_d = limit < 0x1p-4f ? 0x1p15f : 1.0f;
                lift = fminf(0x1p14f / (limit * lift_d), 0x1p15f);
                const float f = lift * lift_d / was;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < NB * 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[m][i][e] *= f;
            }
            if (lift_d != 1.0f) {
                const half2 f = __float2half2_rn(lift_d);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int b = 0; b < NB; ++b) dv[j][b] = h2(__hmul2(as_h2(dv[j][b]), f));
            }
            half2 ph[MT][2], pl[MT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float x = pr[m][j].x * lift, y = pr[m][j].y * lift;
                    ph[m][j] = __floats2half2_rn(x, y);
                    const float2 back = __half22float2(ph[m][j]);
                    pl[m][j] = __floats2half2_rn(x - back.x, y - back.y);
                }
            const uint32_t sel = (g >> 2) * 0x2222u + 0x4400u;  // byte 2 (g / 4) of two words, each twice
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                const int nbp = NB - 4 * p < 4 ? NB - 4 * p : 4;
                uint32_t v[2][2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint8_t *at = tile + NB * 256 + p * 1024 + (((j * 2 + i) * 4 + (g & 3)) * 4 + t) * nbp * 4;
                        if (nbp == 4) load_words<4>(v[j][i], at);
                        if (nbp == 3) load_words<3>(v[j][i], at);
                        if (nbp == 2) load_words<2>(v[j][i], at);
                        if (nbp == 1) load_words<1>(v[j][i], at);
                    }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (b >= nbp) break;
                    const int bb = 4 * p + b;
                    uint32_t wa[MT][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t dd = h2(pair_at(dv[j], bb, NB + bb));
                            if (kMasked) dd &= seen[m][j];  // a key that is not seen weighs nothing, whatever its scale holds
                            const half2 wh = __hmul2(ph[m][j], as_h2(dd));
                            wa[m][2 * j] = h2(wh);
                            wa[m][2 * j + 1] = h2(__hfma2(pl[m][j], as_h2(dd), __hfma2(ph[m][j], as_h2(dd), __hneg2(wh))));
                        }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t b0 = __byte_perm(v[0][0][b], v[0][1][b], sel + x * 0x1111u), b1 = __byte_perm(v[1][0][b], v[1][1][b], sel + x * 0x1111u);
                        const uint32_t l0 = low_codes(b0), l1 = low_codes(b1), h0 = high_codes(b0), h1 = high_codes(b1);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            mma16816(o[m][bb * 4 + x * 2], wa[m], l0, l1, o[m][bb * 4 + x * 2]);
                            mma16816(o[m][bb * 4 + x * 2 + 1], wa[m], h0, h1, o[m][bb * 4 + x * 2 + 1]);
                        }
                    }
                }
            }
        };

        for (unsigned k = 0; k < mine; ++k) {
            const unsigned slot = (done + k) % S::kSlots, phase = (done + k) / S::kSlots & 1;
            if (__any_sync(~0u, !mbar_wait(&bars[warp][slot], phase))) {
                // A copy did not arrive. Let those on their way land (each wait is bounded again); the CTA stops below.
                for (unsigned i = k; i < ahead; ++i) mbar_wait(&bars[warp][(done + i) % S::kSlots], (done + i) / S::kSlots & 1);
                late = true;
                break;
            }
            if (present >> slot & 1) {
                const uint8_t *tile = ring + slot * S::kTile;
                const int key0 = int(sp.tile0 + t0 + warp + k * kWarps) * int(kTileTokens);
                if (key0 >= all_low && key0 + int(kTileTokens) - 1 <= all_high) take(tile, key0, std::false_type{});
                else take(tile, key0, std::true_type{});
            }
            __syncwarp();
            if (ahead < mine) {  // the slot is free again
                if (ahead % 32 == 0) look_up(ahead + lane);
                present = fetch(ahead) ? present | 1u << slot : present & ~(1u << slot);
                ++ahead;
            }
        }
        done += mine;
        if (__syncthreads_or(late)) {
            if (tid == 0) tell(a.status, kServeWait);
            return;
        }

        // the warps' results, joined in the ring's place: [warp][row][dim]
        float *out = reinterpret_cast<float *>(smem + S::kQBytes);
        const float drop = 1.0f / (lift * lift_d);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            sum[m] += __shfl_xor_sync(~0u, sum[m], 1);
            sum[m] += __shfl_xor_sync(~0u, sum[m], 2);
            if (t == 0) m_of[warp][m * 8 + g] = top[m], l_of[warp][m * 8 + g] = sum[m];
            float *to = out + ((warp * MT + m) * 8 + g) * (D + 2);
#pragma unroll
            for (int i = 0; i < NB * 4; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int n = 2 * int(t) + e, b = i / 4, x = i / 2 % 2, h = i & 1;
                    to[32 * b + 16 * h + 4 * (n & 3) + 2 * (n >> 2) + x] = (o[m][i][e] + o[m][i][2 + e]) * (h ? 0.0625f : 1.0f) * drop;
                }
        }
        __syncthreads();
        const bool direct = n_split <= 1;
        if (!direct && item >= plan.max_items) {  // rows counted twice (row starts that overlap): no room
            if (tid == 0) tell(a.status, kServeRequest);
        } else {
            float *part = reinterpret_cast<float *>(a.room) + size_t(item) * plan.rows * D;
            float2 *stat = reinterpret_cast<float2 *>(reinterpret_cast<float *>(a.room) + size_t(plan.max_items) * plan.rows * D) + size_t(item) * plan.rows;
            for (unsigned i = tid; i < MT * 8 * D; i += kThreads) {
                const unsigned row = i / D, dim = i % D;
                if (row0 + row >= all) break;
                float mm = -INFINITY;
                for (unsigned w = 0; w < kWarps; ++w) mm = fmaxf(mm, m_of[w][row]);
                const float ref = mm == -INFINITY ? 0.0f : mm;
                float ov = 0.0f, lv = 0.0f;
                for (unsigned w = 0; w < kWarps; ++w) {
                    const float f = exp2_fast(m_of[w][row] - ref);
                    ov += out[((w * MT + row / 8) * 8 + row % 8) * (D + 2) + dim] * f;
                    lv += l_of[w][row] * f;
                }
                if (direct) {
                    const unsigned at = row0 + row;
                    a.y[(rq.start + at / per) * a.y_stride + size_t(head * per + at % per) * D + dim] = lv == 0.0f ? 0.0f : ov / lv;
                } else {
                    part[row * D + dim] = ov;
                    if (dim == 0) stat[row] = make_float2(mm, lv);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();  // the ring is free for the next item's copies
    }
}

// Rows whose keys were split: the chunks' maxima, sums and outputs joined. One CTA a row of a unit.
__global__ void __launch_bounds__(kThreads) kv4_attn_merge_kernel(const Kv4AttnArgs a, const Plan plan) {
    extern __shared__ unsigned prefix_units[];
    __shared__ float red[kWarps], factor[kMergeChunk], weight[kMergeChunk], sums[kThreads];
    __shared__ float4 joined[kThreads];
    unsigned *prefix = prefix_units, *units = prefix_units + a.n_req + 1;
    pdl_wait();
    pdl_launch_dependents();
    const Schedule sched = make_schedule(a, plan, prefix, units);
    const unsigned dim = a.c.dim, per = a.n_head / a.c.n_kv, total = units[a.n_req];
    for (unsigned long long ur = blockIdx.x; ur < (unsigned long long)total * plan.rows; ur += gridDim.x) {
        const unsigned unit = unsigned(ur / plan.rows), row = unsigned(ur % plan.rows);
        const unsigned r = find(units, a.n_req, unit);
        const Request rq = request_of(a, r, plan.rows, false);
        const unsigned head = (unit - units[r]) % a.c.n_kv, group = (unit - units[r]) / a.c.n_kv;
        const GroupSpan sp = span_of(a, rq, group, plan.rows);
        const unsigned n_split = (sp.tiles + sched.chunk - 1) / sched.chunk, at = group * plan.rows + row;
        if (n_split <= 1 || at >= rq.fresh * per) continue;
        const unsigned first = prefix[r] + group * a.c.n_kv + head, step = rq.groups * a.c.n_kv;
        if (first + (n_split - 1) * step >= plan.max_items) continue;
        const size_t gap = size_t(plan.rows) * dim;
        const float *part = reinterpret_cast<const float *>(a.room) + first * gap + size_t(row) * dim;
        const float2 *stat = reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(a.room) + plan.max_items * gap) + size_t(first) * plan.rows + row;
        const size_t part_step = step * gap, stat_step = size_t(step) * plan.rows;
        float m = -INFINITY;
        for (unsigned s = threadIdx.x; s < n_split; s += kThreads) m = fmaxf(m, stat[s * stat_step].x);
        for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        __syncthreads();
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = m;
        __syncthreads();
        for (unsigned w = 0; w < kWarps; ++w) m = fmaxf(m, red[w]);
        const float ref = m == -INFINITY ? 0.0f : m;
        // four dims a lane; the groups of lanes that cover the dims share out the chunks, whose factors lie in shared memory
        const unsigned lanes = dim / 4, groups = kThreads / lanes, mine = threadIdx.x / lanes, d = threadIdx.x % lanes * 4;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (unsigned s0 = 0; s0 < n_split; s0 += kMergeChunk) {
            const unsigned n = n_split - s0 < kMergeChunk ? n_split - s0 : kMergeChunk;
            __syncthreads();
            for (unsigned s = threadIdx.x; s < n; s += kThreads) {
                const float2 x = stat[(s0 + s) * stat_step];
                const float f = exp2_fast(x.x - ref);
                factor[s] = f;
                weight[s] = f * x.y;
            }
            __syncthreads();
            if (mine < groups) {
#pragma unroll 4
                for (unsigned s = mine; s < n; s += groups) {
                    const float4 x = *reinterpret_cast<const float4 *>(part + (s0 + s) * part_step + d);
                    const float f = factor[s];
                    o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
                    l += weight[s];
                }
            }
        }
        __syncthreads();
        if (mine < groups) joined[mine * lanes + threadIdx.x % lanes] = o, sums[mine] = l;
        __syncthreads();
        if (mine == 0) {
            for (unsigned i = 1; i < groups; ++i) {
                const float4 x = joined[i * lanes + threadIdx.x];
                o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
                l += sums[i];
            }
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            float *y = a.y + (rq.start + at / per) * a.y_stride + size_t(head * per + at % per) * dim + d;
            y[0] = l == 0.0f ? 0.0f : o.x * f, y[1] = l == 0.0f ? 0.0f : o.y * f, y[2] = l == 0.0f ? 0.0f : o.z * f, y[3] = l == 0.0f ? 0.0f : o.w * f;
        }
    }
}

template <int NB, int MT>
cudaError_t launch_tiles(const Kv4AttnArgs &a, const Plan &plan, unsigned sms, cudaStream_t st) {
    using S = Shape<NB, MT>;
    const size_t smem = S::kSmem + (size_t(a.n_req) + 1) * 4;
    static std::mutex mu;
    static int resident[64] = {};  // CTAs an SM takes, by device
    int dev = 0, ctas = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 64) ctas = resident[dev];
        if (!ctas) {
            e = cudaFuncSetAttribute(kv4_attn_kernel<NB, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem + int(kAttnMaxReq + 1) * 4);
            if (e != cudaSuccess) return e;
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kv4_attn_kernel<NB, MT>, kThreads, S::kSmem + 1024);
            if (e != cudaSuccess) return e;
            if (ctas < 1) ctas = 1;
            if (dev < 64) resident[dev] = ctas;
        }
    }
    const unsigned grid = sms * unsigned(ctas);
    return launch_pdl(kv4_attn_kernel<NB, MT>, dim3(grid < plan.max_items ? grid : plan.max_items), dim3(kThreads), smem, st, a, plan);
}

Plan plan_of(const Kv4AttnArgs &a, unsigned sms) {
    Plan p;
    const unsigned per = a.n_head / a.c.n_kv;
    p.rows = a.c.dim <= 128 && (unsigned long long)a.max_q * per > 8 ? 16 : 8;
    p.target = sms * 4;
    // the most units there can be, and the items: `target`, or a chunk's worth each, and a rest for each unit
    const unsigned long long q = a.max_q < a.n_rows ? a.max_q : a.n_rows, rows = (unsigned long long)a.n_rows * per;
    unsigned long long groups = rows / p.rows + (a.n_req < a.n_rows ? a.n_req : a.n_rows);
    const unsigned long long each = (q * per + p.rows - 1) / p.rows * a.n_req;
    if (each < groups) groups = each;
    const unsigned long long tiles = groups * a.c.n_kv * ((a.max_kv + kTileTokens - 1) / kTileTokens);
    const unsigned long long by_chunk = tiles / kMaxChunkTiles;
    unsigned long long items = groups * a.c.n_kv + (by_chunk > p.target ? by_chunk : p.target);
    if (tiles / kWarps + groups * a.c.n_kv < items) items = tiles / kWarps + groups * a.c.n_kv;
    p.max_items = items < 0x7fffffffull ? unsigned(items) : 0x7fffffffu;
    return p;
}

}  // namespace

size_t kv4_attn_room(const Kv4AttnArgs &a, unsigned sms) {
    const Plan p = plan_of(a, sms);
    return size_t(p.max_items) * p.rows * (a.c.dim * 4 + 8);
}
unsigned kv4_attn_launches(const Kv4AttnArgs &a, unsigned) { return a.max_kv > kWarps * kTileTokens ? 2 : 1; }

cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, unsigned sms, cudaStream_t st) {
    const Plan p = plan_of(a, sms);
    const unsigned nb = a.c.dim / 32;
    cudaError_t e = cudaErrorInvalidValue;
    if (p.rows == 16) {
        if (nb == 1) e = launch_tiles<1, 2>(a, p, sms, st);
        if (nb == 2) e = launch_tiles<2, 2>(a, p, sms, st);
        if (nb == 3) e = launch_tiles<3, 2>(a, p, sms, st);
        if (nb == 4) e = launch_tiles<4, 2>(a, p, sms, st);
    } else {
        if (nb == 1) e = launch_tiles<1, 1>(a, p, sms, st);
        if (nb == 2) e = launch_tiles<2, 1>(a, p, sms, st);
        if (nb == 3) e = launch_tiles<3, 1>(a, p, sms, st);
        if (nb == 4) e = launch_tiles<4, 1>(a, p, sms, st);
        if (nb == 5) e = launch_tiles<5, 1>(a, p, sms, st);
        if (nb == 6) e = launch_tiles<6, 1>(a, p, sms, st);
        if (nb == 7) e = launch_tiles<7, 1>(a, p, sms, st);
        if (nb == 8) e = launch_tiles<8, 1>(a, p, sms, st);
    }
    // up to 64 keys are never split
    if (e != cudaSuccess || kv4_attn_launches(a, sms) == 1) return e;
    const unsigned long long rows = (unsigned long long)p.max_items * p.rows;
    return launch_pdl(kv4_attn_merge_kernel, dim3(unsigned(rows < sms * 16ull ? rows : sms * 16ull)), dim3(kThreads), (size_t(a.n_req) + 1) * 8, st, a, p);
}

}  // namespace b200q
