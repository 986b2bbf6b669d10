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
// The FP32 factors (q, and p_t d_tb) are split into two FP16 numbers, 22 bits in all, which sit side by side in two columns of
// the matrix instruction's B operand: four query rows fill its eight columns, and FP32 accuracy costs no second
// instruction. q's rows are first scaled by a power of two to below 2^15, and their lower parts by 2048, so that a number of
// a row 2^20 below its largest has its 22 bits too.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv4.cuh"
#include "pipeline.cuh"
#include "launch.h"
#include "serve.h"

namespace b200q {

namespace {

constexpr unsigned kWarps = 4, kThreads = kWarps * 32;
constexpr unsigned kMaxRange = 1024;     // a warp adds at most 256 tiles into its accumulators before they are joined in FP32
// What a unit costs besides its tiles, in tiles: its queries' way into matrix operands, the joining of its warps' outputs,
// the start of its copies. 64 requests of 5 to 8192 keys, three rows of 32 heads of 128 each: 87 us with 9, 74 with 12, 70
// with 16, 74 with 24 (short requests pile up on a CTA with less, its long ones wait with more).
constexpr unsigned kUnitCost = 16;
// Requests with this many rows (token, head of a KV head's group) are the prompt kernel's when a call's rows and heads make
// work enough for it. New tokens on 512 keys before them, 16 heads of 128 (of 256), us here / there: 128 tokens 32 / 47 (41 / 65),
// 256 45 / 54 (69 / 74), 384 64 / 60 (103 / 82), 1024 202 / 92 (376 / 128); 32 requests of 17 tokens on 1000 keys, 32 heads
// 185 / 128 (306 / 178), of 1 to 8 tokens (4 to 32 rows a request) 70 / 124 (100 / 167).
constexpr unsigned kPromptRows = 64, kPromptWork = 6144;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void tell(uint32_t *status, unsigned bit) {
    if (status) atomicOr(status, bit);
}

struct AttnPlan {
    unsigned grid = 0;        // CTAs
    unsigned max_ranges = 0;  // ranges the workspace holds partial results for
    unsigned rows = 4;        // query rows (token, head) of a unit
    unsigned most_rows = ~0u; // requests with more rows are the prompt kernel's
    bool fits = true;         // the line's places fit 32 bits
};

// ---- the schedule ---------------------------------------------------------------------------------------------------
// A unit is a group of up to 4, 8, 12 or 16 query rows of one KV head; its work is the tiles of keys that they see. All units' tiles
// lie in one line, a unit's kUnitCost and its tiles behind the unit before it, and the line is cut into ranges of equal
// length, one a CTA (several, when a range would pass kMaxRange): every CTA has the same to do whatever the requests'
// lengths, and at most two of a range's pieces are parts of a unit: one that an earlier range began (its
// partial result goes to slot 0 of the range) and one that a later range goes on with (slot 1). The lengths are on the
// device, so every CTA counts the line itself. A request outside the stated bounds has no units.
struct Request {
    unsigned start = 0, fresh = 0, len = 0, groups = 0, span = 0;  // span: tiles that a group of rows sees at most
};

__device__ __forceinline__ Request request_of(const Kv4AttnArgs &a, unsigned r, const AttnPlan &plan, bool report) {
    Request q;
    const unsigned s = a.q_start[r], e = a.q_start[r + 1], len = a.kv_len[r];
    if (s > e || e > a.n_rows || e - s > a.max_q || len > a.max_kv) {
        if (report) tell(a.status, kServeRequest);
        return q;
    }
    const unsigned group = a.n_head / a.c.n_kv, rows = plan.rows;
    if ((unsigned long long)(e - s) * group > plan.most_rows) return q;
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
    unsigned line = 0;  // its length
    unsigned range = 0, ranges = 0;
};

__device__ __forceinline__ unsigned line_of(const Kv4AttnArgs &a, const Request &q) { return q.groups * a.c.n_kv * (q.span + kUnitCost); }

// before[r]: the line's length before request r (n_req + 1 entries)
__device__ Schedule make_schedule(const Kv4AttnArgs &a, const AttnPlan &plan, unsigned *before) {
    __shared__ unsigned line_in[kWarps], broken_in[kWarps];
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (a.n_req + kThreads - 1) / kThreads;
    const unsigned r0 = tid * per < a.n_req ? tid * per : a.n_req, r1 = r0 + per < a.n_req ? r0 + per : a.n_req;
    unsigned broken = a.n_req;  // the first request whose rows run backwards: no rows are counted twice before it
    for (unsigned r = r1; r > r0; --r)
        if (a.q_start[r - 1] > a.q_start[r]) broken = r - 1;
    broken = __reduce_min_sync(~0u, broken);
    if (lane == 0) broken_in[warp] = broken;
    __syncthreads();
    for (unsigned w = 0; w < kWarps; ++w) broken = broken_in[w] < broken ? broken_in[w] : broken;
    unsigned line = 0;
    for (unsigned r = r0; r < r1; ++r) {
        before[r] = line;
        if (r < broken) line += line_of(a, request_of(a, r, plan, blockIdx.x == 0));
        else if (blockIdx.x == 0) tell(a.status, kServeRequest);
    }
    unsigned ls = line;
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(~0u, ls, o);
        if (lane >= o) ls += x;
    }
    if (lane == 31) line_in[warp] = ls;
    __syncthreads();
    Schedule s;
    ls -= line;
    for (unsigned w = 0; w < kWarps; ++w) {
        if (w < warp) ls += line_in[w];
        s.line += line_in[w];
    }
    for (unsigned r = r0; r < r1; ++r) before[r] += ls;
    if (tid == 0) before[a.n_req] = s.line;
    const unsigned each = (s.line + plan.grid - 1) / plan.grid, turns = (each + kMaxRange - 1) / kMaxRange;
    s.range = turns ? ((each + turns - 1) / turns + kWarps - 1) / kWarps * kWarps : kWarps;
    s.ranges = (s.line + s.range - 1) / s.range;
    __syncthreads();
    return s;
}

__device__ __forceinline__ unsigned find(const unsigned *prefix, unsigned n, unsigned i) {  // the last of n with prefix[.] <= i
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

// The workspace: the pieces' outputs, their maxima and sums (two slots a range), and for every range what its edge to the
// range before it cuts.
struct Edge {
    unsigned n = 0;            // pieces of the unit that the edge cuts (0: it cuts none), in the ranges first, first + 1, ...
    unsigned first = 0, slot0 = 0;  // piece 0 lies in slot slot0 of range `first`, the others in slot 0 of theirs
    unsigned rows = 0;         // rows of the unit
    unsigned row0 = 0, head = 0;  // the unit's first (token, head of the group) row of the request, its KV head
    unsigned start = 0;        // the request's first row
    unsigned ranges = 0;       // entry 0 alone: how many there are
};
struct Room {
    float *part;
    float2 *stat;
    Edge *edge;
};
__host__ __device__ inline Room room_of(uint8_t *room, const AttnPlan &plan, unsigned dim) {
    Room r;
    const size_t slots = size_t(plan.max_ranges) * 2 * plan.rows;
    r.part = reinterpret_cast<float *>(room);
    r.stat = reinterpret_cast<float2 *>(r.part + slots * dim);
    r.edge = reinterpret_cast<Edge *>(r.stat + slots);
    return r;
}

// ---- the tile product -----------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2(half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ half2 as_h2(uint32_t x) { return *reinterpret_cast<half2 *>(&x); }

// Two nibbles of a word, bits 0..3 and 16..19 (low) or 4..7 and 20..23 (high), as FP16: put into the mantissa of 1024 they
// read 1024 + c (1024 + 16 c); less 1032 (1152) that is c - 8 (16 (c - 8)), exactly. The subtractions run at half the
// issue rate, 16 a block of a tile. Raw codes (c 2^-24, as they are) with the 8 taken off a block's sum of K, or by a
// product of its own for V, saved 3% at one set of rows and nothing at several, but the sums they swamp cost accuracy: 513
// keys of heads of 256 came out off by 1.3 10^-6 and not 4 10^-7, as FP32 arithmetic is.
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
template <int N>  // N halves, 2 N bytes aligned (N odd: 2)
__device__ __forceinline__ void load_halves(uint32_t *w, const uint8_t *at) {
    if constexpr (N % 2 == 0) {
        load_words<N / 2>(w, at);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            w[i / 2] = *reinterpret_cast<const uint16_t *>(at + 2 * i);
            if (i + 1 < N) w[i / 2] |= uint32_t(*reinterpret_cast<const uint16_t *>(at + 2 * i + 2)) << 16;
        }
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

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8 x 8 matrix of halves, two columns of row lane / 4 a lane
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// CTAs on an SM, by the accumulators a thread holds (8 for each of `blocks` = NB NT) and the registers they leave: 128, 168 or
// 255 a thread. One query token of 16 heads (4 KV heads) on 131,000 keys, us a call with 2 / 3 / 4 CTAs: heads of 64 30.9 / 25.3 /
// 25.1, of 128 36.4 / 31.5 / -, of 256 50.1 / 56.0 / -.
constexpr unsigned ctas_of(unsigned blocks) { return blocks <= 2 ? 4 : blocks <= 4 ? 3 : 2; }
// Sets of four rows that a unit may have, as far as their accumulators fit the registers. Twelve rows of heads of 128 in one
// unit took 1410 cycles a tile, in two (of eight and four rows) 2200.
constexpr unsigned most_sets(unsigned nb) { return nb <= 4 ? 4 : 16 / nb; }

// NB: 32-dim blocks of a head; NT: sets of four query rows.
template <int NB, int NT>
struct Shape {
    static constexpr int kTile = NB * 576;                       // bytes of a tile
    static constexpr int kSlots = NB <= 2 ? 8 : NB <= 4 ? 6 : 3;  // tiles a warp has on their way: all CTAs' rings fill shared memory
    static constexpr int kRows = NT * 4;
    static constexpr int kCtas = ctas_of(NB * NT);           // on an SM, by the accumulators' registers (8 NB NT a thread)
    static constexpr bool kQInRegs = NB * NT <= 8;                // 4 registers a block and set; with more they stay in shared memory
    static constexpr int kQBytes = NT * NB * 2 * 32 * 8;
    static constexpr int kOutBytes = kWarps * kRows * NB * 32 * 4;  // the warps' results
    static constexpr int kRing = kWarps * kSlots * kTile;
    static constexpr int kSmem = kQBytes + kOutBytes + kRing;
};

// The matrix instructions are 16 x 8 x 16 with the codes as A (16 keys by dims, then 16 dims by keys) and the FP32 factor as
// B: four query rows, an upper and a lower column each. Lane (g, t) = (lane / 4, lane % 4) then holds the scores of the keys
// g and g + 8 for row t, and of the output the dims g and g + 8 of a set for row t.
//
// A warp takes every fourth tile of its CTA's chunk, with a running maximum, sum and output of its own; it fetches its
// tiles itself (one bulk copy each), so that nothing in the loop waits for another warp.
//
// Instructions and their latencies bound it: the registers leave two to four warps a quarter SM. A tile of 16 keys takes a
// quarter 380 cycles at 4 rows of heads of 32, 710 at 128, 1290 at 256 (4.6 KB: 820 at the copy rate), 1410 at 12 rows of 128.
// One row of 16 heads of 256 on 131,000 keys: 49 us, 3.1 TB/s; 12 us of it lie before and behind the loop (the wait for
// the kernel before, 2 us of schedule, 2 until the first tile is there, 5 for the merge). A unit's rows follow the bound on new
// tokens and not the request: 64 single tokens of 32 heads of 128 take 39 us where max_q is 1, 90 where it is 4 or more (of 256:
// 65 and 92), since their units then have 16 (8) rows, 4 of them real. Tried without gain: two tiles'
// products at a time, one tile's values beside the next one's scores, the next piece looked up before this one's tiles.
template <int NB, int NT>
__global__ void __launch_bounds__(kThreads, Shape<NB, NT>::kCtas) kv4_attn_kernel(const Kv4AttnArgs a, const AttnPlan plan) {
    using S = Shape<NB, NT>;
    constexpr int kPlanes = (NB + 3) / 4, D = NB * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][S::kSlots];
    __shared__ float m_of[kWarps][S::kRows], l_of[kWarps][S::kRows];
    __shared__ float scale_of[S::kRows];
    // of a warp's piece, by block: the scales seen are below 2^top_of, and are lifted by 4^lift_of
    constexpr int kNoScale = -128;
    __shared__ int8_t top_of[kWarps][NB], lift_of[kWarps][NB];
    auto *before = reinterpret_cast<unsigned *>(smem + S::kSmem);
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const unsigned per = a.n_head / a.c.n_kv, tiles_per_page = a.c.page / kTileTokens;
    float *out = reinterpret_cast<float *>(smem + S::kQBytes);
    uint8_t *ring = smem + S::kQBytes + S::kOutBytes + warp * S::kSlots * S::kTile;
    if (tid == 0) {
        for (unsigned w = 0; w < kWarps; ++w)
            for (int i = 0; i < S::kSlots; ++i) mbar_init(&bars[w][i], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    const Schedule sched = make_schedule(a, plan, before);  // its barriers also cover the mbarriers' start
    const Room room = room_of(a.room, plan, D);
    const size_t page_bytes = size_t(a.c.n_kv) * tiles_per_page * S::kTile;
    if (sched.ranges == 0 && blockIdx.x == 0 && tid == 0) room.edge[0] = Edge{};

    // The pieces of this CTA's ranges, one after another.
    struct Piece {
        unsigned start, all, row0, head;  // the request's first row; its rows; the unit's first row, its KV head
        int base;                         // the position of the request's first new token
        unsigned tile0, mine;             // this warp's first tile, and how many (each kWarps behind the one before)
        unsigned table;                   // the request's row of the table
        unsigned slot;                    // of its result in the workspace; kNoSlot: the piece is a whole unit
    };
    unsigned range = blockIdx.x, at_line = range * sched.range, req = 0;
    bool fresh_range = true;
    auto next_piece = [&](Piece &p) {
        while (range < sched.ranges) {
            const unsigned from = range * sched.range, to = sched.line - from < sched.range ? sched.line : from + sched.range;
            if (at_line >= to) {
                range += gridDim.x;
                at_line = range * sched.range;
                fresh_range = true;
                continue;
            }
            if (fresh_range) req = find(before, a.n_req, from);
            while (before[req + 1] <= at_line) ++req;
            const Request rq = request_of(a, req, plan, false);
            const unsigned length = rq.span + kUnitCost, unit = (at_line - before[req]) / length, begin = before[req] + unit * length;
            const unsigned u0 = at_line - begin, u1 = (to - begin < length ? to - begin : length);
            const GroupSpan sp = span_of(a, rq, unit / a.c.n_kv, plan.rows);
            p.head = unit % a.c.n_kv;
            p.row0 = unit / a.c.n_kv * plan.rows;
            p.all = rq.fresh * per;
            p.start = rq.start;
            p.base = int(rq.len) - int(rq.fresh);
            p.table = req;
            const unsigned t0 = u0 > kUnitCost ? u0 - kUnitCost : 0, end = u1 > kUnitCost ? u1 - kUnitCost : 0, t1 = end < sp.tiles ? end : sp.tiles;
            const bool whole = t0 == 0 && t1 == sp.tiles;
            if (fresh_range && tid == 0) {  // what this range's edge cuts: for the merge
                Edge e;
                const unsigned first = (begin + kUnitCost) / sched.range;
                unsigned last = sp.tiles ? (begin + kUnitCost + sp.tiles - 1) / sched.range : first;
                if (last >= sched.ranges) last = sched.ranges - 1;
                if (begin < from && first < range && range <= last) {
                    e.n = last - first + 1;
                    e.first = first;
                    e.slot0 = begin >= first * sched.range;
                    e.rows = p.all - p.row0 < plan.rows ? p.all - p.row0 : plan.rows;
                    e.row0 = p.row0;
                    e.head = p.head;
                    e.start = p.start;
                }
                if (range == 0) e.ranges = sched.ranges;
                room.edge[range] = e;
            }
            fresh_range = false;
            at_line = begin + length;
            if (sp.tiles == 0 ? u0 != 0 : t0 >= t1) continue;  // (a unit that sees nothing belongs to the range with its first place)
            p.tile0 = sp.tile0 + t0 + warp;
            p.mine = t0 + warp < t1 ? (t1 - t0 - warp + kWarps - 1) / kWarps : 0;
            p.slot = whole ? kNoSlot : range * 2 + (begin >= from);
            return true;
        }
        return false;
    };

    // A warp's tiles: the k-th lies where lane k % 32 keeps.
    Piece pc;
    unsigned slot = 0, phase = 0;  // of the warp's next tile
    unsigned ahead = 0;            // of the piece's tiles, fetched
    unsigned present = 0;          // bit s: slot s holds a tile
    const uint8_t *where = nullptr;
    bool late = false;
    auto look_up = [&](unsigned k) {
        where = nullptr;
        if (k < pc.mine) {
            const unsigned tile = pc.tile0 + k * kWarps, page = a.table[size_t(pc.table) * a.stride + tile / tiles_per_page];
            if (page < a.c.n_pages) where = a.c.base + page * page_bytes + size_t(pc.head * tiles_per_page + tile % tiles_per_page) * S::kTile;
            else tell(a.status, kServePage);
        }
    };
    auto fetch = [&](unsigned k, unsigned slot) {
        const uint8_t *src = reinterpret_cast<const uint8_t *>(__shfl_sync(~0u, (unsigned long long)where, k % 32));
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
        present = src ? present | 1u << slot : present & ~(1u << slot);
    };
    auto begin_piece = [&] {
        look_up(lane);
        unsigned s = slot;
        for (ahead = 0; ahead < unsigned(S::kSlots) && ahead < pc.mine; ++ahead) {
            fetch(ahead, s);
            s = s + 1 == unsigned(S::kSlots) ? 0 : s + 1;
        }
    };
    // waits (each bounded) for n tiles on their way, from the next one on
    auto land = [&](unsigned n) {
        for (unsigned i = 0, s = slot, p = phase; i < n; ++i) {
            mbar_wait(&bars[warp][s], p);
            if (++s == unsigned(S::kSlots)) s = 0, p ^= 1;
        }
    };

    // A warp takes the rows warp, warp + 4, ...; lane: four dims (of 128), then the four 128 behind them.
    constexpr int kQuads = (NB * 8 + 31) / 32;
    float4 x[NT][kQuads];
    const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | a.q_stride * 4 | a.q_head_stride * 4) & 15) == 0;
    auto load_q = [&] {
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            const unsigned at = pc.row0 + m * 4 + warp, row = at < pc.all ? at : pc.row0;
            const float *src = a.q + (pc.start + row / per) * a.q_stride + (pc.head * per + row % per) * a.q_head_stride + lane * 4;
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
                x[m][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (lane + 32 * i >= NB * 8) break;
                const float *at_i = src + i * 128;
                if (wide) x[m][i] = *reinterpret_cast<const float4 *>(at_i);
                else x[m][i] = make_float4(at_i[0], at_i[1], at_i[2], at_i[3]);
            }
        }
    };

    bool more = next_piece(pc);
    if (more) {
        load_q();
        begin_piece();
    }
    while (more) {
        // The queries as B operands, in the order in which a block's words hold the dims: column g is the upper (g even) or
        // lower part of row g / 2.
        const unsigned all = pc.all, row0 = pc.row0, mine = pc.mine;
        const int base = pc.base;
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < kQuads; ++i) big = fmaxf(big, fmaxf(fmaxf(fabsf(x[m][i].x), fabsf(x[m][i].y)), fmaxf(fabsf(x[m][i].z), fabsf(x[m][i].w))));
            big = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(big)));
            int ex = int(__float_as_uint(big) >> 23) - 127 - 14;  // x / 2^ex is below 2^15
            ex = ex < -110 ? -110 : ex > 113 ? 113 : ex;  // (NaN, infinity: what they are)
            const float down = __uint_as_float(unsigned(127 - ex) << 23);
            if (lane == 0) scale_of[m * 4 + warp] = a.scale * kLog2e * __uint_as_float(unsigned(127 + ex) << 23);
#pragma unroll
            for (int i = 0; i < kQuads; ++i) {
                const unsigned quad = lane + 32 * i, set = quad / 4;
                const bool high = set & 1;  // the high nibbles' codes come times 16
                const float f = high ? down * 0.0625f : down;
                uint32_t h0, l0, h1, l1;
                split2(x[m][i].x * f, x[m][i].z * f, h0, l0);
                split2(x[m][i].y * f, x[m][i].w * f, h1, l1);
                if (quad < NB * 8) {
                    uint8_t *to = smem + ((m * NB * 2 + set) * 32 + warp * 8 + quad % 4) * 8;
                    *reinterpret_cast<uint2 *>(to) = make_uint2(h0, h1);
                    *reinterpret_cast<uint2 *>(to + 32) = make_uint2(l0, l1);
                }
            }
        }
        if (lane < NB) top_of[warp][lane] = int8_t(kNoScale), lift_of[warp][lane] = 0;
        __syncthreads();
        uint32_t qb[S::kQInRegs ? NT : 1][S::kQInRegs ? NB * 2 : 1][2];
        float scale[NT];        // of row t
        int pos[NT], low[NT];   // the keys row t sees: [low, pos]
        int wpos[NT], wlow[NT]; // and row g / 2
        auto sees = [&](unsigned row, int &lo, int &hi) {
            const int p = base + int(row / per);
            hi = row < all ? p : -1;
            lo = a.window && p >= 0 && unsigned(p) + 1 > a.window ? p + 1 - int(a.window) : 0;
        };
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            sees(row0 + m * 4 + t, low[m], pos[m]);
            sees(row0 + m * 4 + g / 2, wlow[m], wpos[m]);
            scale[m] = scale_of[m * 4 + t];
            if constexpr (S::kQInRegs) {
#pragma unroll
                for (int i = 0; i < NB * 2; ++i) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(smem + ((m * NB * 2 + i) * 32 + lane) * 8);
                    qb[m][i][0] = v.x, qb[m][i][1] = v.y;
                }
            }
        }

        float o[NT][NB * 2][4], top[NT], sum[NT], limit = 0.0f, lift = 1.0f;
        bool mixed = false;  // a block has a lift of its own
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            top[m] = -INFINITY;
            sum[m] = 0.0f;
#pragma unroll
            for (int i = 0; i < NB * 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][i][e] = 0.0f;
        }

        // Keys that every row of the group sees need no masks.
        const int last_row = base + int((row0 + plan.rows < all ? row0 + plan.rows - 1 : all - 1) / per);
        const int all_low = a.window && last_row >= 0 && unsigned(last_row) + 1 > a.window ? last_row + 1 - int(a.window) : 0;
        const int all_high = base + int(row0 / per);
        // and keys that some row sees lie in [any_low, last_row]
        const int any_low = a.window && all_high >= 0 && unsigned(all_high) + 1 > a.window ? all_high + 1 - int(a.window) : 0;
        auto edge = [&](int key0) { return key0 < all_low || key0 + int(kTileTokens) - 1 > all_high; };

        // the scores of row t and the tile's keys g, g + 8
        auto score = [&](const uint8_t *tile, float (&s)[NT][2]) {
            constexpr float kZero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int m = 0; m < NT; ++m) s[m][0] = s[m][1] = 0.0f;
            {
                uint32_t ds[2][(NB + 1) / 2];
#pragma unroll
                for (int j = 0; j < 2; ++j) load_halves<NB>(ds[j], tile + NB * 512 + (g + 8 * j) * NB * 2);
#pragma unroll
                for (int p = 0; p < kPlanes; ++p) {
                    const int nbp = NB - 4 * p < 4 ? NB - 4 * p : 4;
                    uint32_t w[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint8_t *at = tile + p * 1024 + ((8 * j + g) * 4 + t) * nbp * 4;
                        if (nbp == 4) load_words<4>(w[j], at);
                        if (nbp == 3) load_words<3>(w[j], at);
                        if (nbp == 2) load_words<2>(w[j], at);
                        if (nbp == 1) load_words<1>(w[j], at);
                    }
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        if (b >= nbp) break;
                        const int bb = 4 * p + b;
                        const uint32_t w8[2] = {w[0][b] >> 8, w[1][b] >> 8};
                        const uint32_t lo[4] = {low_codes(w[0][b]), low_codes(w[1][b]), low_codes(w8[0]), low_codes(w8[1])};
                        const uint32_t hi[4] = {high_codes(w[0][b]), high_codes(w[1][b]), high_codes(w8[0]), high_codes(w8[1])};
                        const float d0 = half_at(ds[0], bb), d1 = half_at(ds[1], bb);
#pragma unroll
                        for (int m = 0; m < NT; ++m) {
                            float c[4], e[4];
                            uint2 q0, q1;
                            if constexpr (S::kQInRegs) {
                                q0 = make_uint2(qb[m][bb * 2][0], qb[m][bb * 2][1]);
                                q1 = make_uint2(qb[m][bb * 2 + 1][0], qb[m][bb * 2 + 1][1]);
                            } else {
                                q0 = *reinterpret_cast<const uint2 *>(smem + ((m * NB * 2 + bb * 2) * 32 + lane) * 8);
                                q1 = *reinterpret_cast<const uint2 *>(smem + ((m * NB * 2 + bb * 2 + 1) * 32 + lane) * 8);
                            }
                            mma16816(e, lo, q0.x, q0.y, kZero);
                            mma16816(c, hi, q1.x, q1.y, e);
                            s[m][0] += d0 * (c[0] + c[1] * (1.0f / 2048));
                            s[m][1] += d1 * (c[2] + c[3] * (1.0f / 2048));
                        }
                    }
                }
            }
        };
        // Scores to weights. The running maximum moves only when a score passes it, and then to 4 (in powers of two) above the
        // largest, so that it moves seldom; the weights stay below 1.
        auto weigh = [&](int key0, float (&s)[NT][2]) {
            const bool some = edge(key0);
#pragma unroll
            for (int m = 0; m < NT; ++m) {
                s[m][0] *= scale[m];
                s[m][1] *= scale[m];
                if (some) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int key = key0 + 8 * j + int(g);
                        if (key < low[m] || key > pos[m]) s[m][j] = -INFINITY;
                    }
                }
                float mx = fmaxf(s[m][0], s[m][1]);
                if (__any_sync(~0u, mx > top[m])) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, x));
                    const float nt = mx > top[m] ? mx + 4.0f : top[m];
                    const float f = top[m] == nt ? 1.0f : exp2_fast(top[m] - nt);  // top -inf: 0
                    sum[m] *= f;
#pragma unroll
                    for (int i = 0; i < NB * 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[m][i][e] *= f;
                    top[m] = nt;
                }
                const float ref = top[m] == -INFINITY ? 0.0f : top[m];
                s[m][0] = exp2_fast(s[m][0] - ref);
                s[m][1] = exp2_fast(s[m][1] - ref);
                sum[m] += s[m][0] + s[m][1];
            }
        };
        // A tile holds scales that pass what they are lifted for: every block's largest so far (four lanes a block), and from these
        // the common lift of the weights and each block's own, 4^lift_of: none where its largest scale is within 2^4 of `limit`, so
        // that most caches need none. What the outputs hold already follows. (With one lift for all blocks, values 2^20 below
        // another block's were off by 3 10^-5, and lost from 2^30 on. The lifts of their own cost 0.7% on average, 3% at most, over 30
        // shapes of one request and of 64 whose scales are alike: the first tile of a piece raises, and a second one where the largest
        // scale passes a power of two. With 1/2 as the least limit in the place of 1, where more pieces raise twice, 1.7%.)
        auto raise = [&](const uint8_t *tile, int key0) {
            const unsigned b = lane % 8;
            unsigned big = 0;  // the largest number among the block's scales that some row sees, in a half's bits
            if (b < NB) {
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) {
                    const unsigned tok = lane / 8 * 4 + i, d = *reinterpret_cast<const uint16_t *>(tile + NB * 544 + (tok * NB + b) * 2) & 0x7fffu;
                    const int key = key0 + int(tok);
                    if (key >= any_low && key <= last_row && d <= 0x7bffu) big = max(big, d);
                }
            }
            big = max(big, __shfl_xor_sync(~0u, big, 8));
            big = max(big, __shfl_xor_sync(~0u, big, 16));
            const int exponent = int(__float_as_uint(__half2float(__ushort_as_half(uint16_t(big)))) >> 23) - 126;
            const int own = b < NB ? max(int(top_of[warp][b]), big ? exponent : kNoScale) : kNoScale;  // below 2^own so far
            const int most = __reduce_max_sync(~0u, own), at = most < 0 ? 0 : most > 8 ? 8 : most;
            // limit = 2^at: at 2^8 p's lower part loses as much as a scale that is lowered does
            const int r = at - own, own_lift = r >= 30 ? 15 : r >= 4 ? r / 2 : r >= 0 ? 0 : (r - 1) / 2;
            const float now = __uint_as_float(unsigned(127 + 14 - at) << 23);
            if (limit != 0.0f) {  // (else the outputs hold nothing yet)
                const float follow = now / lift * __uint_as_float(unsigned(127 + 2 * (b < NB ? own_lift - lift_of[warp][b] : 0)) << 23);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const float f = __shfl_sync(~0u, follow, i);
#pragma unroll
                    for (int m = 0; m < NT; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[m][2 * i][e] *= f, o[m][2 * i + 1][e] *= f;
                }
            }
            mixed = __any_sync(~0u, b < NB && own_lift != 0);
            if (lane < NB) top_of[warp][lane] = int8_t(own), lift_of[warp][lane] = int8_t(own_lift);
            __syncwarp();
            lift = now;
            limit = __uint_as_float(unsigned(127 + at) << 23);
        };
        auto value = [&](const uint8_t *tile, int key0, const float (&s)[NT][2]) {
            // The weighted sum of the values: dims by keys, keys by rows.
            // A weight p d is a product of FP16 pairs: with p = ph + pl, wh = fp16(ph d) and wl = fp16(pl d + (ph d - wh)),
            // where ph d - wh is exact in one FP16 multiply-add. What is below 2^-24 is lost, so p is lifted by the power of two that
            // keeps the weights below 2^14 while no d passes `limit`, and a block's d by one of its own (raise, above). Together the
            // parts lost are 2^-34 of the block's largest d, or less (2^-30 where that passes 2^4), whatever the other blocks hold.
            uint32_t dv[2][NB];    // the scales of the keys 2 t + 8 j and the one behind it
            uint32_t seen[NT][2];  // these pairs of keys, by row g / 2, as masks of halves: a key that is not seen weighs nothing, whatever its scale holds
            auto load = [&] {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t raw[NB];
                    load_words<NB>(raw, tile + NB * 544 + (4 * j + t) * NB * 4);
#pragma unroll
                    for (int b = 0; b < NB; ++b) dv[j][b] = h2(pair_at(raw, b, NB + b));
                }
            };
            auto hide = [&] {  // keys that no row sees
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t any = 0;
#pragma unroll
                    for (int m = 0; m < NT; ++m) any |= seen[m][j];
#pragma unroll
                    for (int b = 0; b < NB; ++b) dv[j][b] &= any;
                }
            };
            auto lift_blocks = [&] {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const half2 f = as_h2(unsigned(15 + lift_of[warp][b]) * 0x04000400u);  // twice: a half reaches 2^15
#pragma unroll
                    for (int j = 0; j < 2; ++j) dv[j][b] = h2(__hmul2(__hmul2(as_h2(dv[j][b]), f), f));
                }
            };
            load();
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int m = 0; m < NT; ++m) seen[m][j] = ~0u;
            if (edge(key0)) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int key = key0 + 8 * j + 2 * int(t);
#pragma unroll
                    for (int m = 0; m < NT; ++m)
                        seen[m][j] = (key >= wlow[m] && key <= wpos[m] ? 0x0000ffffu : 0u) | (key + 1 >= wlow[m] && key + 1 <= wpos[m] ? 0xffff0000u : 0u);
                }
                hide();
            }
            if (mixed) lift_blocks();
            half2 big2 = __float2half2_rn(0.0f);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int b = 0; b < NB; ++b) big2 = __hmax2(big2, __habs2(as_h2(dv[j][b])));
            if (__any_sync(~0u, fmaxf(__low2float(big2), __high2float(big2)) > limit)) {
                const bool was_mixed = mixed;
                raise(tile, key0);
                if (was_mixed) load(), hide();
                if (mixed) lift_blocks();
            }
            // Of row g / 2 and the keys 2 t + 8 j, + 1. A lane of an upper column wants ph d, one of a lower column the rest: with
            // (x, y) = (0, ph) in the one and (ph, pl) in the other both are y d + (x d - fp16(x d)).
            half2 wx[NT][2], wy[NT][2];
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float x = s[m][j] * lift;
                    const half h = __float2half_rn(x);
                    const uint32_t ph = transpose8(h2(__half2half2(h))), pl = transpose8(h2(__half2half2(__float2half_rn(x - __half2float(h)))));
                    wx[m][j] = as_h2(g & 1 ? ph : 0u);
                    wy[m][j] = as_h2(g & 1 ? pl : ph);
                }
            const uint32_t sel = (g & 1) * 0x2222u + 0x4400u;  // byte 2 (g % 2) of two words, each twice
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                const int nbp = NB - 4 * p < 4 ? NB - 4 * p : 4;
                uint32_t v[2][2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint8_t *at = tile + NB * 256 + p * 1024 + (((j * 2 + i) * 4 + (g >> 1)) * 4 + t) * nbp * 4;
                        if (nbp == 4) load_words<4>(v[j][i], at);
                        if (nbp == 3) load_words<3>(v[j][i], at);
                        if (nbp == 2) load_words<2>(v[j][i], at);
                        if (nbp == 1) load_words<1>(v[j][i], at);
                    }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (b >= nbp) break;
                    const int bb = 4 * p + b;
                    uint32_t w[NT][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int m = 0; m < NT; ++m) {
                            const half2 d = as_h2(NT == 1 ? dv[j][bb] : dv[j][bb] & seen[m][j]);
                            w[m][j] = h2(__hfma2(wy[m][j], d, __hfma2(wx[m][j], d, __hneg2(__hmul2(wx[m][j], d)))));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t b0 = __byte_perm(v[0][0][b], v[0][1][b], sel + x * 0x1111u), b1 = __byte_perm(v[1][0][b], v[1][1][b], sel + x * 0x1111u);
                        const uint32_t av[4] = {low_codes(b0), high_codes(b0), low_codes(b1), high_codes(b1)};
#pragma unroll
                        for (int m = 0; m < NT; ++m) mma16816(o[m][bb * 2 + x], av, w[m][0], w[m][1], o[m][bb * 2 + x]);
                    }
                }
            }
        };

        float s[NT][2];
        int key0 = int(pc.tile0 * kTileTokens);
        for (unsigned k = 0; k < mine; ++k) {
            if (__any_sync(~0u, !mbar_wait(&bars[warp][slot], phase))) {
                land(ahead - k);  // a copy did not arrive: those on their way land, and the CTA stops below
                late = true;
                break;
            }
            const uint8_t *tile = ring + slot * S::kTile;
            if (present >> slot & 1) {
                score(tile, s);
                weigh(key0, s);
                value(tile, key0, s);
            }
            __syncwarp();
            if (ahead < mine) {  // the tile's slot is free again, for the one kSlots behind it
                if (ahead % 32 == 0) look_up(ahead + lane);
                fetch(ahead, slot);
                ++ahead;
            }
            if (++slot == unsigned(S::kSlots)) slot = 0, phase ^= 1;
            key0 += int(kWarps * kTileTokens);
        }
        const Piece was = pc;
        if (!late) {
            ahead = 0;
            more = next_piece(pc);
            if (more) begin_piece();  // the next piece's tiles come while this one's results are joined
        }

        // the warps' results: [warp][row][dim] (the barrier: all have read the piece before's)
        __syncthreads();
        const float drop = 1.0f / lift;
#pragma unroll
        for (int m = 0; m < NT; ++m) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum[m] += __shfl_xor_sync(~0u, sum[m], x);
            if (g == 0) m_of[warp][m * 4 + t] = top[m], l_of[warp][m * 4 + t] = sum[m];
            float *to = out + (warp * S::kRows + m * 4 + t) * D + 4 * (g >> 1) + 2 * (g & 1);
#pragma unroll
            for (int b = 0; b < NB; ++b) {  // two bytes of a word: the low nibbles, then the high ones
                const float f = drop * __uint_as_float(unsigned(127 - 2 * lift_of[warp][b]) << 23), f16 = 0.0625f * f;
                *reinterpret_cast<float2 *>(to + 32 * b) = make_float2((o[m][2 * b][0] + o[m][2 * b][1]) * f, (o[m][2 * b + 1][0] + o[m][2 * b + 1][1]) * f);
                *reinterpret_cast<float2 *>(to + 32 * b + 16) = make_float2((o[m][2 * b][2] + o[m][2 * b][3]) * f16, (o[m][2 * b + 1][2] + o[m][2 * b + 1][3]) * f16);
            }
        }
        if (__syncthreads_or(late)) {
            // some copy did not arrive: let the others land (each wait is bounded again), and stop
            if (!late) land(ahead);
            if (tid == 0) tell(a.status, kServeWait);
            return;
        }
        if (more) load_q();
        for (unsigned i = tid; i < S::kRows * D / 4; i += kThreads) {
            const unsigned row = i / (D / 4), dim = i % (D / 4) * 4, at = was.row0 + row;
            if (at >= was.all) break;
            float mm = -INFINITY, lv = 0.0f;
            for (unsigned w = 0; w < kWarps; ++w) mm = fmaxf(mm, m_of[w][row]);
            const float ref = mm == -INFINITY ? 0.0f : mm;
            float4 ov = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (unsigned w = 0; w < kWarps; ++w) {
                const float f = exp2_fast(m_of[w][row] - ref);
                const float4 x = *reinterpret_cast<const float4 *>(out + (w * S::kRows + row) * D + dim);
                ov.x += x.x * f, ov.y += x.y * f, ov.z += x.z * f, ov.w += x.w * f;
                lv += l_of[w][row] * f;
            }
            if (was.slot == kNoSlot) {
                const float f = 1.0f / lv;
                float *y = a.y + (was.start + at / per) * a.y_stride + size_t(was.head * per + at % per) * D + dim;
                y[0] = lv == 0.0f ? 0.0f : ov.x * f, y[1] = lv == 0.0f ? 0.0f : ov.y * f, y[2] = lv == 0.0f ? 0.0f : ov.z * f,
                y[3] = lv == 0.0f ? 0.0f : ov.w * f;
            } else {
                const size_t slot_row = size_t(was.slot) * S::kRows + row;
                *reinterpret_cast<float4 *>(room.part + slot_row * D + dim) = ov;
                if (dim == 0) room.stat[slot_row] = make_float2(mm, lv);
            }
        }
    }
}

// Units that lie in more than one range: the pieces' maxima, sums and outputs joined. Every edge between two ranges has a
// CTA, which reads what it cuts, and the CTAs of a unit's edges share out its rows and dims. Few pieces: a warp takes 128
// dims of a row, piece after piece. Many: a CTA takes 32 dims of a row, eight lanes to a piece, so that all loads are on
// their way at once.
__global__ void __launch_bounds__(kThreads) kv4_attn_merge_kernel(const Kv4AttnArgs a, const AttnPlan plan) {
    __shared__ float4 o_of[kWarps][8];
    __shared__ float2 s_of[kWarps];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned dim = a.c.dim, per = a.n_head / a.c.n_kv, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const Room room = room_of(a.room, plan, dim);
    const unsigned ranges = room.edge[0].ranges < plan.max_ranges ? room.edge[0].ranges : plan.max_ranges;
    for (unsigned edge = blockIdx.x + 1; edge < ranges; edge += gridDim.x) {
        const Edge e = room.edge[edge];
        // (a range that was given up after a wait ran out has left no edge here: whatever lies there is not followed)
        if (e.n < 2 || e.first >= edge || edge - e.first >= e.n || e.first + e.n > ranges || e.rows > plan.rows || e.head >= a.c.n_kv ||
            e.start >= a.n_rows || (e.row0 + e.rows - 1) / per >= a.n_rows - e.start)
            continue;
        const bool many = e.n >= 16;
        const unsigned lanes = many ? 8 : 32, chunks = (dim / 4 + lanes - 1) / lanes, share = e.n - 1;
        unsigned w = edge - e.first - 1;
        if (!many) w = w * kWarps + warp;
        for (; w < e.rows * chunks; w += many ? share : share * kWarps) {
            const unsigned row = w / chunks, d = (w % chunks * lanes + lane % lanes) * 4;
            const bool in = d < dim;
            float m = -INFINITY, l = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (unsigned s0 = many ? warp * 4 + lane / 8 : 0; s0 < e.n; s0 += many ? 128 : 8) {
                float2 x[8];
                float4 v[8];
                const unsigned step = many ? 16 : 1;
#pragma unroll
                for (unsigned i = 0; i < 8; ++i) {
                    const unsigned s = s0 + i * step;
                    const size_t at = ((size_t(e.first + s) * 2 + (s ? 0 : e.slot0)) * plan.rows + row);
                    x[i] = s < e.n ? room.stat[at] : make_float2(-INFINITY, 0.0f);
                    v[i] = s < e.n && in ? *reinterpret_cast<const float4 *>(room.part + at * dim + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
                float top = m;
#pragma unroll
                for (unsigned i = 0; i < 8; ++i) top = fmaxf(top, x[i].x);
                const float ref = top == -INFINITY ? 0.0f : top, f0 = exp2_fast(m - ref);
                m = top;
                l *= f0;
                o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
                for (unsigned i = 0; i < 8; ++i) {
                    const float f = exp2_fast(x[i].x - ref);
                    l += f * x[i].y;
                    o.x += v[i].x * f, o.y += v[i].y * f, o.z += v[i].z * f, o.w += v[i].w * f;
                }
            }
            if (many) {  // the pieces' lanes, then the warps
                float top = m;
                for (unsigned x = 8; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
                const float f = exp2_fast(m - (top == -INFINITY ? 0.0f : top));
                m = top;
                l *= f;
                o.x *= f, o.y *= f, o.z *= f, o.w *= f;
                for (unsigned x = 8; x < 32; x <<= 1)
                    o.x += __shfl_xor_sync(~0u, o.x, x), o.y += __shfl_xor_sync(~0u, o.y, x), o.z += __shfl_xor_sync(~0u, o.z, x),
                        o.w += __shfl_xor_sync(~0u, o.w, x), l += __shfl_xor_sync(~0u, l, x);
                __syncthreads();
                if (lane < 8) o_of[warp][lane] = o;
                if (lane == 0) s_of[warp] = make_float2(m, l);
                __syncthreads();
                if (warp || lane >= 8) continue;
                top = -INFINITY;
                for (unsigned i = 0; i < kWarps; ++i) top = fmaxf(top, s_of[i].x);
                const float ref = top == -INFINITY ? 0.0f : top;
                l = 0.0f;
                o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (unsigned i = 0; i < kWarps; ++i) {
                    const float fi = exp2_fast(s_of[i].x - ref);
                    const float4 v = o_of[i][lane];
                    l += s_of[i].y * fi;
                    o.x += v.x * fi, o.y += v.y * fi, o.z += v.z * fi, o.w += v.w * fi;
                }
            }
            if (!in) continue;
            const unsigned at = e.row0 + row;
            const float f = 1.0f / l;
            float *y = a.y + (e.start + at / per) * a.y_stride + size_t(e.head * per + at % per) * dim + d;
            y[0] = l == 0.0f ? 0.0f : o.x * f, y[1] = l == 0.0f ? 0.0f : o.y * f, y[2] = l == 0.0f ? 0.0f : o.z * f, y[3] = l == 0.0f ? 0.0f : o.w * f;
        }
    }
}

template <int NB, int NT>
cudaError_t launch_tiles(const Kv4AttnArgs &a, const AttnPlan &plan, unsigned grid, cudaStream_t st) {
    using S = Shape<NB, NT>;
    const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kv4_attn_kernel<NB, NT>), S::kSmem + int(kMaxAttnReq + 1) * 4);
    if (e != cudaSuccess) return e;
    return launch_pdl(a.pdl, kv4_attn_kernel<NB, NT>, dim3(grid), dim3(kThreads), S::kSmem + (size_t(a.n_req) + 1) * 4, st, a, plan);
}

template <int NB>
cudaError_t launch_sets(const Kv4AttnArgs &a, const AttnPlan &plan, cudaStream_t st) {
    switch (plan.rows / 4) {
        case 1: return launch_tiles<NB, 1>(a, plan, plan.grid, st);
        case 2: return launch_tiles<NB, 2>(a, plan, plan.grid, st);
        case 3:
            if constexpr (most_sets(NB) >= 3) return launch_tiles<NB, 3>(a, plan, plan.grid, st);
            break;
        case 4:
            if constexpr (most_sets(NB) >= 4) return launch_tiles<NB, 4>(a, plan, plan.grid, st);
            break;
    }
    return cudaErrorInvalidValue;
}

AttnPlan plan_of(const Kv4AttnArgs &a, unsigned sms) {
    AttnPlan p;
    const unsigned per = a.n_head / a.c.n_kv;
    const unsigned nb = a.c.dim / 32, most = most_sets(nb) * 4;
    const unsigned long long rows_of = (unsigned long long)a.max_q * per, groups_of = (rows_of + most - 1) / most;
    const unsigned sets = unsigned((rows_of + groups_of * 4 - 1) / (groups_of * 4));
    p.rows = 4 * sets;
    if ((unsigned long long)a.max_q * per >= kPromptRows && (unsigned long long)a.n_rows * a.n_head >= kPromptWork) p.most_rows = kPromptRows - 1;
    p.grid = sms * ctas_of(nb * sets);  // as many as run at once
    // the most units there can be, and the line's length
    const unsigned long long q = a.max_q < a.n_rows ? a.max_q : a.n_rows, rows = (unsigned long long)a.n_rows * per;
    unsigned long long groups = rows / p.rows + (a.n_req < a.n_rows ? a.n_req : a.n_rows);
    const unsigned long long most_of = q * per < p.most_rows ? q * per : p.most_rows;  // of a request's rows
    const unsigned long long each = (most_of + p.rows - 1) / p.rows * a.n_req;
    if (each < groups) groups = each;
    const unsigned long long units = groups * a.c.n_kv;
    unsigned long long line = units * ((a.max_kv + kTileTokens - 1) / kTileTokens + kUnitCost);
    if (line == 0) line = 1;  // (no rows: a workspace all the same, so that a room of 0 means a shape that is refused)
    if ((line + kWarps - 1) / kWarps < p.grid) p.grid = unsigned((line + kWarps - 1) / kWarps);
    const unsigned long long turns = (line + (unsigned long long)p.grid * kMaxRange - 1) / ((unsigned long long)p.grid * kMaxRange);
    p.max_ranges = unsigned(turns * p.grid);
    p.fits = line < 0x80000000ull && rows < 0x80000000ull && (rows / 128 + a.n_req + 1) * a.c.n_kv < 0x80000000ull;
    return p;
}

}  // namespace

size_t kv4_attn_room(const Kv4AttnArgs &a, unsigned sms) {
    const AttnPlan p = plan_of(a, sms);
    if (!p.fits) return 0;
    return size_t(p.max_ranges) * (2 * p.rows * (a.c.dim * 4 + 8) + sizeof(Edge));
}
unsigned kv4_attn_launches(const Kv4AttnArgs &a, unsigned sms) {
    const AttnPlan p = plan_of(a, sms);
    return (p.max_ranges > 1 ? 2 : 1) + (p.most_rows != ~0u);
}

cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, unsigned sms, cudaStream_t st) {
    const AttnPlan p = plan_of(a, sms);
    cudaError_t e = cudaErrorInvalidValue;
    switch (a.c.dim / 32) {
        case 1: e = launch_sets<1>(a, p, st); break;
        case 2: e = launch_sets<2>(a, p, st); break;
        case 3: e = launch_sets<3>(a, p, st); break;
        case 4: e = launch_sets<4>(a, p, st); break;
        case 5: e = launch_sets<5>(a, p, st); break;
        case 6: e = launch_sets<6>(a, p, st); break;
        case 7: e = launch_sets<7>(a, p, st); break;
        case 8: e = launch_sets<8>(a, p, st); break;
    }
    if (e != cudaSuccess) return e;
    if (p.max_ranges > 1) {  // (else nothing lies in two ranges)
        const unsigned edges = p.max_ranges - 1;
        e = launch_pdl(a.pdl, kv4_attn_merge_kernel, dim3(edges < sms * 8 ? edges : sms * 8), dim3(kThreads), 0, st, a, p);
    }
    if (e != cudaSuccess || p.most_rows == ~0u) return e;
    return launch_kv4_prompt(a, p.most_rows + 1, st);
}

}  // namespace b200q
