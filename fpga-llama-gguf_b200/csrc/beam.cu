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

// Of 8192 logits of one row: the maximum m, sum e^(x - m), and the n_out best in order. The logits are read once, by
// asynchronous copies into shared memory (a thread's own: no registers held and no barrier, so that five CTAs an SM
// keep loads on their way while others compute): the threads' own best give a bound that n_out reach, and the few
// candidates at or above it are ranked by counting. Should ties put more than kFound there, the best are taken out one
// by one.
constexpr unsigned kFound = 512;
template <bool kWide>  // rows on 16 bytes
__global__ void __launch_bounds__(kSelThreads, 5) beam_chunk_kernel(const BeamSelectArgs a, unsigned long long *list, float2 *stat) {
    __shared__ __align__(16) float values[kSelChunk];
    __shared__ unsigned long long found[kFound], kept[kMaxBeamOut], best_of[kSelThreads / 32];
    __shared__ unsigned sorted[kSelThreads / 32][32];
    __shared__ unsigned n_found;
    __shared__ float red[kSelThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chunk = blockIdx.x, row = blockIdx.y, first = chunk * kSelChunk;
    const float *x = a.logits + row * a.stride;
#pragma unroll
    for (unsigned i = 0; i < kSelPer; i += 4) {  // four values of this thread
        float *to = values + (i / 4 * kSelThreads + tid) * 4;
        const unsigned at = first + (i / 4 * kSelThreads + tid) * 4;
        if (kWide && at + 4 <= a.vocab) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(x + at) : "memory");
        } else {
            for (unsigned e = 0; e < 4; ++e) {
                if (at + e < a.vocab) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(to + e)), "l"(x + at + e) : "memory");
                else to[e] = -INFINITY;
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    auto token = [&](unsigned i) { return first + (i / 4 * kSelThreads + tid) * 4 + i % 4; };
    auto four = [&](unsigned i) { return *reinterpret_cast<const float4 *>(values + (i / 4 * kSelThreads + tid) * 4); };
    float m = -INFINITY;  // (fmaxf passes a NaN over)
#pragma unroll
    for (unsigned i = 0; i < kSelPer; i += 4) {
        const float4 y = four(i);
        m = fmaxf(fmaxf(m, y.x), fmaxf(fmaxf(y.y, y.z), y.w));
    }
    if (tid == 0) n_found = 0;
    float top = m;
    for (unsigned o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if (lane == 0) red[warp] = top;
    const unsigned limit = reached_by<kSelThreads / 32>(order_of(m), a.n_out, sorted);  // (with a barrier)
    const float floor = limit ? __uint_as_float(limit & 0x80000000u ? limit & 0x7FFFFFFFu : ~limit) : -3.402823466e38f;
    if (m >= floor) {
        for (unsigned i = 0; i < kSelPer; i += 4) {
            const float4 y = four(i);
            if (!(fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= floor)) continue;
            for (unsigned e = 0; e < 4; ++e) {
                const float v = e == 0 ? y.x : e == 1 ? y.y : e == 2 ? y.z : y.w;
                if (!(v >= floor)) continue;
                const unsigned at = atomicAdd(&n_found, 1u);
                if (at < kFound) found[at] = cand(v, token(i + e));
            }
        }
    }
    top = red[0];
#pragma unroll
    for (unsigned w = 1; w < kSelThreads / 32; ++w) top = fmaxf(top, red[w]);
    // e^(x - m) as a power of two (a chunk without a finite logit adds nothing)
    const float shift = top == -INFINITY ? 0.0f : top;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto power = [&](float v) {  // (a NaN counts as -inf)
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((fmaxf(v, -INFINITY) - shift) * 1.4426950408889634f));
        return e;
    };
#pragma unroll
    for (unsigned i = 0; i < kSelPer; i += 4) {
        const float4 y = four(i);
        s[0] += power(y.x), s[1] += power(y.y), s[2] += power(y.z), s[3] += power(y.w);
    }
    float sum = (s[0] + s[1]) + (s[2] + s[3]);
    for (unsigned o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    __syncthreads();  // found is whole, red is read
    if (lane == 0) red[warp] = sum;
    const unsigned n = n_found;
    if (n <= kFound) {
        for (unsigned i = tid; i < n; i += kSelThreads) {
            const unsigned long long c = found[i];
            unsigned r = 0;
            for (unsigned j = 0; j < n; ++j) r += found[j] > c;
            if (r < a.n_out) kept[r] = c;
        }
        for (unsigned i = n + tid; i < a.n_out; i += kSelThreads) kept[i] = 0;
    } else {
        unsigned long long last = ~0ull;
        for (unsigned r = 0; r < a.n_out; ++r) {
            unsigned long long best = 0;
            for (unsigned i = 0; i < kSelPer; ++i) {
                const unsigned long long c = cand(values[(i / 4 * kSelThreads + tid) * 4 + i % 4], token(i));
                if (c < last && c > best) best = c;
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
    const size_t at = size_t(row) * gridDim.x + chunk;
    if (tid == 0) {
        sum = red[0];
        for (unsigned w = 1; w < kSelThreads / 32; ++w) sum += red[w];
        stat[at] = make_float2(top, sum);
    }
    for (unsigned i = tid; i < a.n_out; i += kSelThreads) list[at * a.n_out + i] = kept[i];
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
    auto *held = reinterpret_cast<unsigned long long *>(best + size_t(a.beams) * n);
    for (unsigned b = warp; b < a.beams; b += kMergeThreads / 32) {
        const unsigned row = req * a.beams + b;
        const float score = a.scores[row];
        const float2 *st = stat + size_t(row) * chunks;
        const unsigned long long *mine = lists + b * per_beam;
        if (in_smem) {
            for (unsigned i = lane; i < per_beam; i += 32) held[b * per_beam + i] = mine[i];
            mine = held + b * per_beam;
        }
        float m = -INFINITY;
        for (unsigned c = lane; c < chunks; c += 32) m = fmaxf(m, st[c].x);
        for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        double s = 0.0;
        for (unsigned c = lane; c < chunks; c += 32)
            if (st[c].x > -INFINITY) s += double(st[c].y) * exp2((double(st[c].x) - double(m)) * 1.4426950408889634074);
        for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        unsigned got = 0;
        if (fabsf(m) < INFINITY && fabsf(score) < INFINITY) {
            const double offset = double(score) - (double(m) + log(s));
            __syncwarp();
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
                    best[b * n + got] = Scored{offset + double(cand_logit(top)), cand_token(top)};
#pragma unroll
                    for (unsigned i = 0; i < kHeads; ++i)
                        if (i == which) head[i] = ++at[i] < n ? mine[(i * 32 + lane) * n + at[i]] : 0;
                }
            }
        }
        if (lane == 0) count[b] = got;
    }
    __syncthreads();
    unsigned total = 0;
    for (unsigned b = 0; b < a.beams; ++b) total += count[b];
    for (unsigned i = threadIdx.x; i < a.beams * n; i += kMergeThreads) {
        const unsigned b = i / n, k = i % n;
        if (k >= count[b]) continue;
        const Scored c = best[i];
        unsigned rank = k;
        for (unsigned x = 0; x < a.beams && rank < n; ++x) {
            if (x == b) continue;
            unsigned lo = 0, hi = count[x];  // candidates of beam x that come before c
            while (lo < hi) {
                const unsigned mid = (lo + hi) / 2;
                const double o = best[x * n + mid].score;
                if (o > c.score || (o == c.score && x < b)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < n) {
            a.out[req * n + rank] = float(c.score);
            a.parent[req * n + rank] = b;
            a.token[req * n + rank] = c.token;
        }
    }
    for (unsigned i = total + threadIdx.x; i < n; i += kMergeThreads) {
        a.out[req * n + i] = -INFINITY;
        a.parent[req * n + i] = kNoSlot;
        a.token[req * n + i] = kNoSlot;
    }
}

// ---- beam_reorder ---------------------------------------------------------------------------------------------------
// A thread owns one column (16, 4 or 1 bytes, by the rows' alignment) of a request's beams in one layer and reads every
// beam's parent before it writes any, so that src and dst may be the same.
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

cudaError_t launch_beam_select(const BeamSelectArgs &a, cudaStream_t st) {
    const unsigned chunks = chunks_of(a.vocab), rows = a.n_req * a.beams;
    auto *list = reinterpret_cast<unsigned long long *>(a.room);
    auto *stat = reinterpret_cast<float2 *>(list + size_t(rows) * chunks * a.n_out);
    const bool wide = ((reinterpret_cast<uintptr_t>(a.logits) | a.stride * 4) & 15) == 0;
    const cudaError_t e = launch_pdl(a.pdl, wide ? beam_chunk_kernel<true> : beam_chunk_kernel<false>, dim3(chunks, rows), dim3(kSelThreads), 0, st, a, list, stat);
    if (e != cudaSuccess) return e;
    const size_t scored = size_t(a.beams) * a.n_out * sizeof(Scored), lists = size_t(a.beams) * chunks * a.n_out * 8;
    const unsigned in_smem = lists <= kListBytes;
    const cudaError_t f = ensure_smem_attr(reinterpret_cast<const void *>(beam_merge_kernel), int(kMaxBeams * kMaxBeamOut * sizeof(Scored) + kListBytes));
    if (f != cudaSuccess) return f;
    return launch_pdl(a.pdl, beam_merge_kernel, dim3(a.n_req), dim3(kMergeThreads), scored + (in_smem ? lists : 0), st, a,
                      static_cast<const unsigned long long *>(list), static_cast<const float2 *>(stat), chunks, in_smem);
}

cudaError_t launch_beam_reorder(const BeamReorderArgs &a, cudaStream_t st) {
    const size_t all = a.row_bytes | a.src_layer | a.dst_layer | reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst);
    if (all % 16 == 0) return launch_reorder<uint4>(a, st);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, st);
    return launch_reorder<uint8_t>(a, st);
}

}  // namespace b200q
