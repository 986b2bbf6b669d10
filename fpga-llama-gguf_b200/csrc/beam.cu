// Beam search: the best continuations over a request's beams and the vocabulary, and dense state rows moved to their
// beams' parents.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve.h"

namespace b200q {
namespace {

constexpr unsigned kSelThreads = 256, kSelPer = 32, kSelChunk = kSelThreads * kSelPer;  // logits a CTA ranks
constexpr unsigned kMergeThreads = 1024;

unsigned chunks_of(unsigned vocab) { return (vocab + kSelChunk - 1) / kSelChunk; }

// A candidate as one word: larger is better (the higher logit, then the lower token); 0: none. The upper half orders FP32
// values; a NaN or -inf logit is no candidate.
__device__ __forceinline__ unsigned long long cand(float x, unsigned token) {
    if (!(x > -INFINITY)) return 0;
    if (x == 0.0f) x = 0.0f;  // -0 and +0 tie
    const unsigned b = __float_as_uint(x), key = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)key << 32 | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float cand_logit(unsigned long long c) {
    const unsigned key = unsigned(c >> 32);
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ unsigned cand_token(unsigned long long c) { return 0xFFFFFFFFu - unsigned(c); }

// Of 8192 logits of one row: the maximum m, sum e^(x - m), and the n_out best in order. The n-th best of the threads' own
// maxima is a lower bound of the n-th best of all, and only the n threads at or above it can hold a better value, so at
// most 32 n candidates are ranked, by counting.
__global__ void __launch_bounds__(kSelThreads) beam_chunk_kernel(const BeamSelectArgs a, unsigned long long *list, float2 *stat) {
    __shared__ unsigned long long top[kSelThreads], found[kMaxBeamOut * kSelPer];
    __shared__ unsigned long long bound;
    __shared__ unsigned n_found;
    __shared__ float red[kSelThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const float *x = a.logits + row * a.stride;
    float v[kSelPer];
    float m = -INFINITY;
    unsigned long long best = 0;
#pragma unroll
    for (unsigned i = 0; i < kSelPer; ++i) {
        const unsigned t = chunk * kSelChunk + i * kSelThreads + tid;
        v[i] = t < a.vocab ? x[t] : -INFINITY;
        if (v[i] > m) m = v[i], best = cand(v[i], t);  // the first of equal values: the lowest token
    }
    if (tid == 0) bound = 0, n_found = 0;
    top[tid] = best;
    for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (tid % 32 == 0) red[tid / 32] = m;
    __syncthreads();
    for (unsigned w = 0; w < kSelThreads / 32; ++w) m = fmaxf(m, red[w]);
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (unsigned i = 0; i < kSelPer; ++i)
        if (v[i] > -INFINITY) s += m == INFINITY ? INFINITY : expf(v[i] - m);
    for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (tid % 32 == 0) red[tid / 32] = s;
    unsigned rank = 0;
    for (unsigned i = 0; i < kSelThreads; ++i) rank += top[i] > best;
    if (best && rank == a.n_out - 1) bound = best;
    __syncthreads();
    const unsigned long long limit = bound ? bound : 1;
    if (best >= limit) {
#pragma unroll
        for (unsigned i = 0; i < kSelPer; ++i) {
            const unsigned long long c = cand(v[i], chunk * kSelChunk + i * kSelThreads + tid);
            if (c >= limit) found[atomicAdd(&n_found, 1u)] = c;
        }
    }
    __syncthreads();
    const size_t at = size_t(row) * gridDim.x + chunk;
    if (tid == 0) {
        s = 0.0f;
        for (unsigned w = 0; w < kSelThreads / 32; ++w) s += red[w];
        stat[at] = make_float2(m, s);
    }
    const unsigned n = n_found;
    for (unsigned i = tid; i < n; i += kSelThreads) {
        const unsigned long long c = found[i];
        unsigned r = 0;
        for (unsigned j = 0; j < n; ++j) r += found[j] > c;
        if (r < a.n_out) list[at * a.n_out + r] = c;
    }
    for (unsigned i = n + tid; i < a.n_out; i += kSelThreads) list[at * a.n_out + i] = 0;
}

// One CTA a request. A warp a beam: log sum e^x from the chunks' statistics (in 64 bits), and the n_out best of the
// chunks' ordered lists, the largest head each time. Then every candidate's rank among all beams' (the score in 64 bits,
// so that the order does not hang on how FP32 rounds; ties to the lower beam, then token), by a search in each list.
struct Scored {
    double score;
    unsigned token;
};
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamSelectArgs a, const unsigned long long *list, const float2 *stat,
                                                                   unsigned chunks) {
    extern __shared__ Scored best[];  // [beams][n_out], descending
    __shared__ unsigned count[kMaxBeams];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned req = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = a.n_out;
    for (unsigned b = warp; b < a.beams; b += kMergeThreads / 32) {
        const unsigned row = req * a.beams + b;
        const float score = a.scores[row];
        const float2 *st = stat + size_t(row) * chunks;
        float m = -INFINITY;
        for (unsigned c = lane; c < chunks; c += 32) m = fmaxf(m, st[c].x);
        for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        double s = 0.0;
        for (unsigned c = lane; c < chunks; c += 32)
            if (st[c].x > -INFINITY) s += double(st[c].y) * exp(double(st[c].x) - double(m));
        for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        const bool live = fabsf(m) < INFINITY && fabsf(score) < INFINITY;
        const double lse = double(m) + log(s);
        unsigned got = 0;
        if (live) {
            // lane c holds the heads of the lists c, c + 32, ...
            unsigned at[kMaxVocab / kSelChunk / 32];
#pragma unroll
            for (unsigned i = 0; i < kMaxVocab / kSelChunk / 32; ++i) at[i] = 0;
            for (; got < n; ++got) {
                unsigned long long top = 0;
                unsigned mine = 0;
#pragma unroll
                for (unsigned i = 0; i < kMaxVocab / kSelChunk / 32; ++i) {
                    const unsigned c = i * 32 + lane;
                    const unsigned long long h = c < chunks && at[i] < n ? list[(size_t(row) * chunks + c) * n + at[i]] : 0;
                    if (h > top) top = h, mine = i;
                }
                unsigned long long all = top;
                for (unsigned o = 16; o; o >>= 1) {
                    const unsigned long long x = __shfl_xor_sync(~0u, all, o);
                    all = x > all ? x : all;
                }
                if (all == 0) break;
                if (top == all) {
#pragma unroll
                    for (unsigned i = 0; i < kMaxVocab / kSelChunk / 32; ++i) at[i] += i == mine;
                }
                if (lane == 0) best[b * n + got] = Scored{double(score) + (double(cand_logit(all)) - lse), cand_token(all)};
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
        unsigned rank = 0;
        for (unsigned x = 0; x < a.beams; ++x) {
            unsigned lo = 0, hi = count[x];  // candidates of beam x that come before c
            while (lo < hi) {
                const unsigned mid = (lo + hi) / 2;
                const Scored o = best[x * n + mid];
                const bool before = o.score > c.score || (o.score == c.score && (x < b || (x == b && mid < k)));
                if (before) lo = mid + 1;
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
    if (a.beams <= 4) return launch_pdl(beam_reorder_kernel<T, 4>, grid, dim3(256), 0, st, a);
    if (a.beams <= 8) return launch_pdl(beam_reorder_kernel<T, 8>, grid, dim3(256), 0, st, a);
    if (a.beams <= 16) return launch_pdl(beam_reorder_kernel<T, 16>, grid, dim3(256), 0, st, a);
    return launch_pdl(beam_reorder_kernel<T, 32>, grid, dim3(256), 0, st, a);
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
    cudaError_t e = launch_pdl(beam_chunk_kernel, dim3(chunks, rows), dim3(kSelThreads), 0, st, a, list, stat);
    if (e != cudaSuccess) return e;
    return launch_pdl(beam_merge_kernel, dim3(a.n_req), dim3(kMergeThreads), size_t(a.beams) * a.n_out * sizeof(Scored), st, a,
                      static_cast<const unsigned long long *>(list), static_cast<const float2 *>(stat), chunks);
}

cudaError_t launch_beam_reorder(const BeamReorderArgs &a, cudaStream_t st) {
    const size_t all = a.row_bytes | a.src_layer | a.dst_layer | reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst);
    if (all % 16 == 0) return launch_reorder<uint4>(a, st);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, st);
    return launch_reorder<uint8_t>(a, st);
}

}  // namespace b200q
