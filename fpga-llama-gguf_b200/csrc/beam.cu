// Beam search: the best continuations over a request's beams and the vocabulary, and dense state rows moved to their
// beams' parents.
#include <cuda_runtime.h>

#include "common.cuh"
#include "launch.h"
#include "pipeline.cuh"
#include "serve.h"

namespace b200q {
namespace {

constexpr unsigned kSelThreads = 256, kSelPer = 32, kSelChunk = kSelThreads * kSelPer;  // logits a CTA ranks
constexpr unsigned kMergeThreads = 512;

unsigned chunks_of(unsigned vocab) { return (vocab + kSelChunk - 1) / kSelChunk; }

// A logit as an integer of the same order (0: a NaN or -inf, no candidate; -0 and +0 are one)
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// A candidate as one word: larger is better (the higher logit, then the lower token); 0: none.
__device__ __forceinline__ unsigned long long cand(float x, unsigned token) {
    const unsigned key = order_of(x);
    return key ? (unsigned long long)key << 32 | (0xFFFFFFFFu - token) : 0;
}
__device__ __forceinline__ float cand_logit(unsigned long long c) {
    const unsigned key = unsigned(c >> 32);
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ unsigned cand_token(unsigned long long c) { return 0xFFFFFFFFu - unsigned(c); }

// A value that at least n of the CTA's values (one a thread) reach, and not many more: each warp sorts its own (bitonic, across
// the lanes); of a set of s warps at least n values reach the least of their n / s-th ones; the best of all sets of 8, 4, 2
// and 1 warps is taken. (0: there are not n values.) sorted: the CTA's values.
template <unsigned kWarpsOf>
__device__ __forceinline__ unsigned reached_by(unsigned mine, unsigned n, unsigned (*sorted)[32]) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
    for (unsigned k = 2; k <= 32; k *= 2)
#pragma unroll
        for (unsigned j = k / 2; j; j /= 2) {  // the larger one goes to the lower lane where bit k of the lane is clear
            const unsigned x = __shfl_xor_sync(~0u, mine, j);
            const bool larger = ((lane & j) == 0) == ((lane & k) == 0 || k == 32);
            mine = (x > mine) == larger ? x : mine;
        }
    sorted[warp][lane] = mine;
    __syncthreads();
    // lane l: set size kWarpsOf >> l / 8, the set that holds warp l % 8
    const unsigned s = kWarpsOf >> (lane / kWarpsOf), set = lane % kWarpsOf / (s ? s : 1) * s, each = s ? (n + s - 1) / s : 33;
    unsigned low = each <= 32 ? ~0u : 0;
    for (unsigned i = 0; i < s && each <= 32; ++i) low = min(low, sorted[set + i][each - 1]);
    return __reduce_max_sync(~0u, low);
}

// A segment of a row: some chunks of 8192 logits after one another. Of them the maximum m, sum e^(x - m), and the n_out best in
// order. The logits are read once, by asynchronous copies into shared memory (a thread's own, so no barrier; the next
// chunk's are on their way while one is looked through). A thread keeps a maximum and a sum of its own. In the first chunk
// the threads' own best give a bound that n_out of them reach; what is above it in the segment's chunks, some dozens each, is
// collected and ranked by counting at the end. Should more come together, the n_out best so far are taken out first and the
// worst of them is the bound from then on; should ties put more there than can be held, they are taken out one by one.
// 16 requests of 8 beams over 151,936 logits, 16 each: 34 us with the lists' merge (the bytes alone: 12); by themselves and
// with cold caches the kernels take 30 and 10 us. 128 rows in 3 segments are 384 of the 444 CTAs that run at once, of 7, 6 and 6
// chunks. A chunk takes a CTA 1.9 us (0.6 to issue the next one's copies, 0.2 maxima, 0.5 exponentials, 0.4 candidates and the barrier),
// at which three CTAs an SM ask for all of the memory's rate; the first one (2.5 with its bound) and the end (1.5) do not. With
// a list a chunk instead, each ranked by itself and five CTAs an SM, the whole call took 40 us, with chunks of 4096 57.
constexpr unsigned kFound = 512, kSelCtas = 3;  // CTAs on an SM, by shared memory
static_assert(kSelPer == 32 && kFound / 2 > kMaxBeamOut);
template <bool kWide>  // rows on 16 bytes
__global__ void __launch_bounds__(kSelThreads, kSelCtas)
    beam_chunk_kernel(const BeamSelectArgs a, unsigned long long *list, float2 *stat, unsigned chunks) {
    extern __shared__ __align__(16) float rooms[];  // two chunks, or the segment's only one
    __shared__ __align__(16) unsigned long long found[kFound];
    __shared__ unsigned long long kept[kMaxBeamOut], best_of[kSelThreads / 32];
    __shared__ unsigned sorted[kSelThreads / 32][32];
    __shared__ unsigned more_found[3];
    __shared__ float2 sums[kSelThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y, n_out = a.n_out;
    const unsigned c0 = unsigned((unsigned long long)chunks * blockIdx.x / gridDim.x), c1 = unsigned((unsigned long long)chunks * (blockIdx.x + 1) / gridDim.x);
    const float *x = a.logits + row * a.stride;
    auto place = [&](unsigned i) { return (i / 4 * kSelThreads + tid) * 4 + i % 4; };  // of the thread's value i in a chunk
    auto fetch = [&](unsigned chunk, float *values) {
        const unsigned first = chunk * kSelChunk;
#pragma unroll
        for (unsigned i = 0; i < kSelPer; i += 4) {
            float *to = values + place(i);
            const unsigned at = first + place(i);
            if (kWide && at + 4 <= a.vocab) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(x + at) : "memory");
            } else {
                for (unsigned e = 0; e < 4; ++e) {
                    if (at + e < a.vocab) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(to + e)), "l"(x + at + e) : "memory");
                    else to[e] = -INFINITY;
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(c0, rooms);
    if (tid < 3) more_found[tid] = 0;
    __syncthreads();
    float m = -INFINITY, sum = 0.0f;  // of the thread's values so far
    float floor = -INFINITY;          // candidates are above it
    unsigned have = 0;                // of them
    // The best n_out of n candidates (kept, or written out), and 0 where there are fewer.
    auto rank = [&](unsigned n, unsigned long long *to) {
        if (n % 2 && tid == 0) found[n] = 0;  // (n < kFound)
        __syncthreads();
        for (unsigned i = tid; i < n; i += kSelThreads) {
            const unsigned long long c = found[i];
            unsigned r = 0;
#pragma unroll 8
            for (unsigned j = 0; j < n; j += 2) {
                const ulonglong2 y = *reinterpret_cast<const ulonglong2 *>(found + j);
                r += (y.x > c) + (y.y > c);
            }
            if (r < n_out) to[r] = c;
        }
        for (unsigned i = n + tid; i < n_out; i += kSelThreads) to[i] = 0;
    };
    for (unsigned c = c0; c < c1; ++c) {
        const unsigned turn = c - c0, first = c * kSelChunk;
        const float *values = rooms + turn % 2 * kSelChunk;
        if (c + 1 < c1) {
            fetch(c + 1, rooms + (turn + 1) % 2 * kSelChunk);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        auto four = [&](unsigned i) { return *reinterpret_cast<const float4 *>(values + place(i)); };
        float top = -INFINITY;  // (fmaxf passes a NaN over)
#pragma unroll
        for (unsigned i = 0; i < kSelPer; i += 4) {
            const float4 y = four(i);
            top = fmaxf(fmaxf(top, y.x), fmaxf(fmaxf(y.y, y.z), y.w));
        }
        if (floor == -INFINITY) {
            const unsigned limit = reached_by<kSelThreads / 32>(order_of(top), n_out, sorted);
            // the number below it (none lies between +0 and the largest negative one: -0 counts as +0)
            if (limit > order_of(-3.402823466e38f)) floor = cand_logit((unsigned long long)(limit - (limit == 0x80000000u ? 2 : 1)) << 32);
        }
        // e^(x - m) as a power of two (values that are all -inf or NaN add nothing)
        const float was = m;
        m = fmaxf(m, top);
        const float shift = m == -INFINITY ? 0.0f : m;
        auto power = [&](float v) {  // (a NaN counts as -inf)
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((fmaxf(v, -INFINITY) - shift) * 1.4426950408889634f));
            return e;
        };
        if (was != m) sum *= power(was);
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        unsigned hits = 0;  // of the thread's values, those above the bound
#pragma unroll
        for (unsigned i = 0; i < kSelPer; i += 4) {
            const float4 y = four(i);
            s[0] += power(y.x), s[1] += power(y.y), s[2] += power(y.z), s[3] += power(y.w);
            hits |= (y.x > floor ? 1u << i : 0u) | (y.y > floor ? 2u << i : 0u) | (y.z > floor ? 4u << i : 0u) | (y.w > floor ? 8u << i : 0u);
        }
        sum += (s[0] + s[1]) + (s[2] + s[3]);
        if (hits) {
            unsigned at = have + atomicAdd(&more_found[turn % 3], unsigned(__popc(hits)));
            for (; hits; hits &= hits - 1, ++at) {
                const unsigned i = place(__ffs(hits) - 1);
                if (at < kFound) found[at] = cand(values[i], first + i);
            }
        }
        if (tid == 0) more_found[(turn + 1) % 3] = 0;  // (last looked at two chunks ago)
        __syncthreads();
        const unsigned held = have;
        have += more_found[turn % 3];
        if (have < kFound / 2) continue;
        if (have < kFound) {
            rank(have, kept);
        } else {
            unsigned long long last = ~0ull;
            for (unsigned r = 0; r < n_out; ++r) {
                unsigned long long best = 0;
                for (unsigned i = tid; i < held; i += kSelThreads)
                    if (found[i] < last && found[i] > best) best = found[i];
                for (unsigned i = 0; i < kSelPer; ++i) {
                    const unsigned long long y = cand(values[place(i)], first + place(i));
                    if (y < last && y > best) best = y;
                }
                for (unsigned o = 16; o; o >>= 1) {
                    const unsigned long long y = __shfl_xor_sync(~0u, best, o);
                    best = y > best ? y : best;
                }
                __syncthreads();
                if (lane == 0) best_of[warp] = best;
                __syncthreads();
                for (unsigned w = 0; w < kSelThreads / 32; ++w) best = best_of[w] > best ? best_of[w] : best;
                last = best;
                if (tid == 0) kept[r] = best;
            }
        }
        __syncthreads();
        if (tid < n_out) found[tid] = kept[tid];
        floor = cand_logit(kept[n_out - 1]);  // (a later token loses a tie)
        have = n_out;
        __syncthreads();
    }
    const size_t at = size_t(row) * gridDim.x + blockIdx.x;
    rank(have, list + at * n_out);
    // the threads' maxima and sums
    float all = m;
    for (unsigned o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(~0u, all, o));
    if (m != all) sum *= exp2f((m - all) * 1.4426950408889634f);
    for (unsigned o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) sums[warp] = make_float2(all, sum);
    __syncthreads();
    if (warp == 0) {
        const float2 part = lane < kSelThreads / 32 ? sums[lane] : make_float2(-INFINITY, 0.0f);
        m = part.x;
        for (unsigned o = 4; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        sum = part.x == m ? part.y : part.y * exp2f((part.x - m) * 1.4426950408889634f);
        for (unsigned o = 4; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) stat[at] = make_float2(m, sum);
    }
}

// One CTA a request. A warp a beam: log sum e^x from the chunks' statistics (in 64 bits), and the n_out best of the
// chunks' ordered lists, the largest head each time (lane c holds the heads of the lists c, c + 32, ...; the lists lie in
// shared memory when they fit). Then every candidate's rank among all beams', by a search in each beam's list: the
// score in 64 bits, so that the order does not hang on how FP32 rounds; ties to the lower beam, then token.
struct Scored {
    double score;
    unsigned token;
};
constexpr unsigned kHeads = kMaxVocab / kSelChunk / 32;  // lists a lane holds
constexpr unsigned kListBytes = 64 * 1024;               // of lists in shared memory, at most
constexpr unsigned kCounted = 128;                       // a beam's candidates that are ranked by counting

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamSelectArgs a, const unsigned long long *list, const float2 *stat,
                                                                   unsigned chunks, unsigned in_smem) {
    extern __shared__ __align__(16) uint8_t merge_smem[];
    Scored *best = reinterpret_cast<Scored *>(merge_smem);  // [beams][n_out], descending
    __shared__ unsigned count[kMaxBeams];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned req = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = a.n_out;
    const size_t per_beam = size_t(chunks) * n;
    const unsigned long long *lists = list + size_t(req) * a.beams * per_beam;
    auto *rank = reinterpret_cast<unsigned *>(best + size_t(a.beams) * n);
    auto *held = reinterpret_cast<unsigned long long *>(rank + (size_t(a.beams) * n + 1) / 2 * 2);
    for (unsigned i = threadIdx.x; i < a.beams * n; i += kMergeThreads) rank[i] = 0;
    for (unsigned b = warp; b < a.beams; b += kMergeThreads / 32) {
        const unsigned row = req * a.beams + b;
        const float score = a.scores[row];
        const float2 *st = stat + size_t(row) * chunks;
        const float2 st0 = lane < chunks ? st[lane] : make_float2(-INFINITY, 0.0f);
        const unsigned long long *mine = lists + b * per_beam;
        if (in_smem) {
            for (unsigned i = lane; i < per_beam; i += 32) held[b * per_beam + i] = mine[i];
            mine = held + b * per_beam;
        }
        float m = st0.x;
        for (unsigned c = lane + 32; c < chunks; c += 32) m = fmaxf(m, st[c].x);
        for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        double s = st0.x > -INFINITY ? double(st0.y) * exp2((double(st0.x) - double(m)) * 1.4426950408889634074) : 0.0;
        for (unsigned c = lane + 32; c < chunks; c += 32)
            if (st[c].x > -INFINITY) s += double(st[c].y) * exp2((double(st[c].x) - double(m)) * 1.4426950408889634074);
        for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        unsigned got = 0;
        if (fabsf(m) < INFINITY && fabsf(score) < INFINITY) {
            const double log_s = log(s);
            __syncwarp();
            auto put = [&](unsigned place, unsigned long long c) {
                best[b * n + place] = Scored{double(score) + ((double(cand_logit(c)) - double(m)) - log_s), cand_token(c)};
            };
            if (in_smem && per_beam <= kCounted) {  // few: each one's place is the number of larger ones
                unsigned long long c[kCounted / 32];
                unsigned place[kCounted / 32];
#pragma unroll
                for (unsigned i = 0; i < kCounted / 32; ++i) c[i] = i * 32 + lane < per_beam ? mine[i * 32 + lane] : 0, place[i] = 0;
#pragma unroll 4
                for (unsigned j = 0; j < per_beam; ++j) {
                    const unsigned long long y = mine[j];
#pragma unroll
                    for (unsigned i = 0; i < kCounted / 32; ++i) place[i] += y > c[i];
                }
#pragma unroll
                for (unsigned i = 0; i < kCounted / 32; ++i) {
                    got += __popc(__ballot_sync(~0u, c[i] != 0));
                    if (c[i] && place[i] < n) put(place[i], c[i]);
                }
                got = got < n ? got : n;
            } else {
                unsigned long long head[kHeads];
                unsigned at[kHeads];
#pragma unroll
                for (unsigned i = 0; i < kHeads; ++i) {
                    at[i] = 0;
                    head[i] = i * 32 + lane < chunks ? mine[(i * 32 + lane) * n] : 0;
                }
                for (; got < n; ++got) {
                    unsigned long long top = head[0];
                    unsigned which = 0;
#pragma unroll
                    for (unsigned i = 1; i < kHeads; ++i)
                        if (head[i] > top) top = head[i], which = i;
                    const unsigned key = __reduce_max_sync(~0u, unsigned(top >> 32));
                    if (key == 0) break;
                    const unsigned low = __reduce_max_sync(~0u, unsigned(top >> 32) == key ? unsigned(top) : 0u);
                    if (unsigned(top >> 32) == key && unsigned(top) == low) {
                        put(got, top);
#pragma unroll
                        for (unsigned i = 0; i < kHeads; ++i)
                            if (i == which) head[i] = ++at[i] < n ? mine[(i * 32 + lane) * n + at[i]] : 0;
                    }
                }
            }
        }
        if (lane == 0) count[b] = got;
    }
    __syncthreads();
    unsigned total = 0;
    for (unsigned b = 0; b < a.beams; ++b) total += count[b];
    // A candidate's rank: its place in its own beam's list, and the places before it in every other one's, a thread a list.
    for (unsigned p = threadIdx.x; p < a.beams * n * a.beams; p += kMergeThreads) {
        const unsigned i = p / a.beams, x = p % a.beams, b = i / n, k = i % n;
        if (k >= count[b]) continue;
        unsigned before = k;
        if (x != b) {
            const double score = best[i].score;
            unsigned lo = 0, hi = count[x];
            while (lo < hi) {
                const unsigned mid = (lo + hi) / 2;
                const double o = best[x * n + mid].score;
                if (o > score || (o == score && x < b)) lo = mid + 1;
                else hi = mid;
            }
            before = lo;
        }
        if (before) atomicAdd(&rank[i], before);
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < a.beams * n; i += kMergeThreads) {
        const unsigned b = i / n;
        if (i % n >= count[b] || rank[i] >= n) continue;
        const Scored c = best[i];
        a.out[req * n + rank[i]] = float(c.score);
        a.parent[req * n + rank[i]] = b;
        a.token[req * n + rank[i]] = c.token;
    }
    for (unsigned i = total + threadIdx.x; i < n; i += kMergeThreads) {
        a.out[req * n + i] = -INFINITY;
        a.parent[req * n + i] = kNoSlot;
        a.token[req * n + i] = kNoSlot;
    }
}

// ---- beam_reorder ---------------------------------------------------------------------------------------------------
// A thread owns one column (16, 4 or 1 bytes, by the rows' alignment) of a request's beams in one layer and reads every
// beam's parent before it writes any, so that src and dst may be the same. Bound by memory: 277 MB in 44.4 us, 6.2 TB/s, 95%
// of the measured copy rate.
template <typename T, int W>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const BeamReorderArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned row0 = blockIdx.y * a.beams;
    const size_t cols = a.row_bytes / sizeof(T);
    const uint8_t *src = a.src + blockIdx.z * a.src_layer + row0 * a.row_bytes;
    uint8_t *dst = a.dst + blockIdx.z * a.dst_layer + row0 * a.row_bytes;
    const bool same = a.src == a.dst;
    unsigned p[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        p[i] = unsigned(i) < a.beams ? a.parent[row0 + i] : kNoSlot;
        if (p[i] >= a.beams && p[i] != kNoSlot && threadIdx.x == 0 && a.status) atomicOr(a.status, kServeParent);
    }
    for (size_t c = size_t(blockIdx.x) * 256 + threadIdx.x; c < cols; c += size_t(gridDim.x) * 256) {
        T v[W];
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (p[i] < a.beams && !(same && p[i] == unsigned(i))) v[i] = *reinterpret_cast<const T *>(src + p[i] * a.row_bytes + c * sizeof(T));
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (p[i] < a.beams && !(same && p[i] == unsigned(i))) *reinterpret_cast<T *>(dst + size_t(i) * a.row_bytes + c * sizeof(T)) = v[i];
    }
}

template <typename T>
cudaError_t launch_reorder(const BeamReorderArgs &a, cudaStream_t st) {
    const size_t cols = a.row_bytes / sizeof(T), want = (cols + 255) / 256;
    const dim3 grid(unsigned(want < 4096 ? want : 4096), a.n_req, a.layers);
    if (a.beams <= 4) return launch_pdl(a.pdl, beam_reorder_kernel<T, 4>, grid, dim3(256), 0, st, a);
    if (a.beams <= 8) return launch_pdl(a.pdl, beam_reorder_kernel<T, 8>, grid, dim3(256), 0, st, a);
    if (a.beams <= 16) return launch_pdl(a.pdl, beam_reorder_kernel<T, 16>, grid, dim3(256), 0, st, a);
    return launch_pdl(a.pdl, beam_reorder_kernel<T, 32>, grid, dim3(256), 0, st, a);
}

}  // namespace

size_t beam_select_room(const BeamSelectArgs &a) {
    const size_t lists = size_t(a.n_req) * a.beams * chunks_of(a.vocab);
    return lists * (a.n_out * sizeof(unsigned long long) + sizeof(float2));
}

cudaError_t launch_beam_select(const BeamSelectArgs &a, unsigned sms, cudaStream_t st) {
    const unsigned chunks = chunks_of(a.vocab), rows = a.n_req * a.beams;
    auto *list = reinterpret_cast<unsigned long long *>(a.room);
    auto *stat = reinterpret_cast<float2 *>(list + size_t(rows) * chunks * a.n_out);
    const bool wide = ((reinterpret_cast<uintptr_t>(a.logits) | a.stride * 4) & 15) == 0;
    const auto kernel = wide ? beam_chunk_kernel<true> : beam_chunk_kernel<false>;
    constexpr int kRooms = 2 * kSelChunk * sizeof(float);
    cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kernel), kRooms);
    if (e != cudaSuccess) return e;
    // Segments: as many as run at once, as far as rows and chunks go round. (For two / three / four CTAs an SM 128 rows of 151,936
    // took 35.9 / 35.7 / 37.1 us, 192 rows 50.6 / 44.3 / 48.3, 256 rows 51.3 / 51.3 / 60.9.)
    const unsigned fit = sms * kSelCtas / rows, segments = fit < 1 ? 1 : fit < chunks ? fit : chunks;
    e = launch_pdl(a.pdl, kernel, dim3(segments, rows), dim3(kSelThreads), segments == chunks ? kRooms / 2 : kRooms, st, a, list, stat, chunks);
    if (e != cudaSuccess) return e;
    const size_t scored = size_t(a.beams) * a.n_out * sizeof(Scored) + (size_t(a.beams) * a.n_out + 1) / 2 * 8, lists = size_t(a.beams) * segments * a.n_out * 8;
    const unsigned in_smem = lists <= kListBytes;
    e = ensure_smem_attr(reinterpret_cast<const void *>(beam_merge_kernel), int(kMaxBeams * kMaxBeamOut * (sizeof(Scored) + 4) + kListBytes));
    if (e != cudaSuccess) return e;
    return launch_pdl(a.pdl, beam_merge_kernel, dim3(a.n_req), dim3(kMergeThreads), scored + (in_smem ? lists : 0), st, a,
                      static_cast<const unsigned long long *>(list), static_cast<const float2 *>(stat), segments, in_smem);
}

cudaError_t launch_beam_reorder(const BeamReorderArgs &a, cudaStream_t st) {
    const size_t all = a.row_bytes | a.src_layer | a.dst_layer | reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst);
    if (all % 16 == 0) return launch_reorder<uint4>(a, st);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, st);
    return launch_reorder<uint8_t>(a, st);
}

}  // namespace b200q
