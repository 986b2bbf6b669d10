// Beam search: the best continuations over a request's beams and the vocabulary, and dense state rows moved to their
// beams' parents.
#include <cuda_runtime.h>

#include "common.cuh"
#include "serve.h"

namespace b200q {
namespace {

constexpr unsigned kSelThreads = 256, kSelPer = 32, kSelChunk = kSelThreads * kSelPer;  // logits a CTA ranks
constexpr unsigned kMergeThreads = 512;

unsigned chunks_of(unsigned vocab) { return (vocab + kSelChunk - 1) / kSelChunk; }

// FP32 and FP64 values as integers of the same order (0: a NaN or -inf, no candidate; -0 and +0 are one)
__device__ __forceinline__ unsigned order_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const unsigned b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_of(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
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

// A value that at least n of a CTA's values reach, as high as one finds cheaply: `mine` is the best of each thread's. Among
// the 32 of a warp the n-th best does; of `sets` warps with n / sets each the worst does; of all such sets the
// best. (0: there are not n values.)
template <typename T, unsigned kWarpsOf>
__device__ __forceinline__ T reached_by(T mine, unsigned n, T *of_warp) {
    const unsigned lane = threadIdx.x & 31, sets = (n + 31) / 32, each = (n + sets - 1) / sets;
    unsigned rank = 0;
#pragma unroll 8
    for (unsigned i = 1; i < 32; ++i) {
        const T x = __shfl_sync(~0u, mine, (lane + i) & 31);
        rank += x > mine || (x == mine && ((lane + i) & 31) < lane);
    }
    if (rank == each - 1) of_warp[threadIdx.x / 32] = mine;
    __syncthreads();
    T best = 0;
#pragma unroll
    for (unsigned w = 0; w < kWarpsOf; w += sets) {
        T low = of_warp[w];
        for (unsigned i = 1; i < sets; ++i) low = w + i < kWarpsOf ? (of_warp[w + i] < low ? of_warp[w + i] : low) : 0;
        best = low > best ? low : best;
    }
    return best;
}

// Of 8192 logits of one row: the maximum m, sum e^(x - m), and the n_out best in order. One pass over the logits, which stay
// in registers: each thread's best gives a bound (reached_by), the few candidates at or above it are ranked by counting.
// They are at most kFound: a thread whose best lies below the bound has none, and should ties or an even slope
// put more threads above it, the list is cut down to the n_out best whenever it is full.
constexpr unsigned kFound = 1024;
template <bool kWide>  // rows on 16 bytes
__global__ void __launch_bounds__(kSelThreads) beam_chunk_kernel(const BeamSelectArgs a, unsigned long long *list, float2 *stat) {
    __shared__ unsigned long long found[kFound], kept[kMaxBeamOut];
    __shared__ unsigned bound_of[kSelThreads / 32];
    __shared__ unsigned n_found;
    __shared__ float red[kSelThreads / 32];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned tid = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y, first = chunk * kSelChunk;
    const float *x = a.logits + row * a.stride;
    float v[kSelPer];
    auto token = [&](unsigned i) { return first + (kWide ? (i / 4 * kSelThreads + tid) * 4 + i % 4 : i * kSelThreads + tid); };
    if (kWide && first + kSelChunk <= a.vocab) {
#pragma unroll
        for (unsigned i = 0; i < kSelPer; i += 4) {
            const float4 y = __ldcs(reinterpret_cast<const float4 *>(x + token(i)));
            v[i] = y.x, v[i + 1] = y.y, v[i + 2] = y.z, v[i + 3] = y.w;
        }
    } else {
#pragma unroll
        for (unsigned i = 0; i < kSelPer; ++i) v[i] = token(i) < a.vocab ? __ldcs(x + token(i)) : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (unsigned i = 0; i < kSelPer; ++i) m = fmaxf(m, v[i]);  // (a NaN is passed over)
    if (tid == 0) n_found = 0;
    const unsigned limit = reached_by<unsigned, kSelThreads / 32>(order_of(m), a.n_out, bound_of);
    const float floor = limit ? __uint_as_float(limit & 0x80000000u ? limit & 0x7FFFFFFFu : ~limit) : -INFINITY;
    float top = m;
    for (unsigned o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    if (tid % 32 == 0) red[tid / 32] = top;
    // one round as a rule; a full list is cut down, and what found no room comes again
    bool left = m >= floor && m > -INFINITY;
    unsigned from = 0;
    for (;;) {
        __syncthreads();
        if (left) {
            left = false;
#pragma unroll
            for (unsigned i = 0; i < kSelPer; ++i) {
                if (i >= from && !left && v[i] >= floor && v[i] > -INFINITY) {
                    const unsigned at = atomicAdd(&n_found, 1u);
                    if (at < kFound) found[at] = cand(v[i], token(i));
                    else left = true, from = i;
                }
            }
        }
        const bool again = __syncthreads_or(left);
        const unsigned n = n_found < kFound ? n_found : kFound;
        for (unsigned i = tid; i < n; i += kSelThreads) {
            const unsigned long long c = found[i];
            unsigned r = 0;
            for (unsigned j = 0; j < n; ++j) r += found[j] > c;
            if (r < a.n_out) kept[r] = c;
        }
        for (unsigned i = n + tid; i < a.n_out; i += kSelThreads) kept[i] = 0;
        __syncthreads();
        if (!again) break;
        for (unsigned i = tid; i < a.n_out; i += kSelThreads) found[i] = kept[i];
        if (tid == 0) n_found = a.n_out;
    }
    top = red[0];
#pragma unroll
    for (unsigned w = 1; w < kSelThreads / 32; ++w) top = fmaxf(top, red[w]);
    // e^(x - m) as a power of two; a row of the chunk without a finite logit adds nothing
    constexpr float kLog2e = 1.4426950408889634f;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (unsigned i = 0; i < kSelPer; ++i) {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((v[i] - shift) * kLog2e));
        s[i % 4] += v[i] > -INFINITY ? e : 0.0f;
    }
    float sum = (s[0] + s[1]) + (s[2] + s[3]);
    for (unsigned o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    __syncthreads();
    if (tid % 32 == 0) red[tid / 32] = sum;
    __syncthreads();
    const size_t at = size_t(row) * gridDim.x + chunk;
    if (tid == 0) {
        sum = red[0];
        for (unsigned w = 1; w < kSelThreads / 32; ++w) sum += red[w];
        stat[at] = make_float2(top, sum);
    }
    for (unsigned i = tid; i < a.n_out; i += kSelThreads) list[at * a.n_out + i] = kept[i];
}

// One CTA a request. log sum e^x of every beam from its chunks' statistics, in 64 bits; then the chunks' ordered lists,
// whose heads give a bound that n_out candidates reach, and the candidates at or above it are ranked by counting: the
// score in 64 bits, so that the order does not hang on how FP32 rounds, ties to the lower beam, then token.
struct Scored {
    unsigned long long score, place;  // place: beam and token, the lower the better
};
__device__ __forceinline__ bool before(const Scored &x, const Scored &y) { return x.score > y.score || (x.score == y.score && x.place < y.place); }

__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamSelectArgs a, const unsigned long long *list, const float2 *stat,
                                                                   unsigned chunks) {
    __shared__ Scored found[kFound], kept[kMaxBeamOut];
    __shared__ double offset[kMaxBeams];  // score - log sum e^x
    __shared__ bool live[kMaxBeams];
    __shared__ unsigned long long bound_of[kMergeThreads / 32];
    __shared__ unsigned n_found;
    pdl_wait();
    pdl_launch_dependents();
    const unsigned req = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_out, lists = a.beams * chunks;
    for (unsigned b = warp; b < a.beams; b += kMergeThreads / 32) {
        const float score = a.scores[req * a.beams + b];
        const float2 *st = stat + size_t(req * a.beams + b) * chunks;
        float m = -INFINITY;
        for (unsigned c = lane; c < chunks; c += 32) m = fmaxf(m, st[c].x);
        for (unsigned o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        double s = 0.0;
        for (unsigned c = lane; c < chunks; c += 32)
            if (st[c].x > -INFINITY) s += double(st[c].y) * exp2((double(st[c].x) - double(m)) * 1.4426950408889634074);
        for (unsigned o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        if (lane == 0) {
            live[b] = fabsf(m) < INFINITY && fabsf(score) < INFINITY;
            offset[b] = double(score) - (double(m) + log(s));
        }
    }
    if (tid == 0) n_found = 0;
    __syncthreads();
    const unsigned long long *lists_of = list + size_t(req) * lists * n;
    auto scored = [&](unsigned l, unsigned k, Scored &c) {  // candidate k of list l
        const unsigned long long w = lists_of[size_t(l) * n + k];
        const unsigned b = l / chunks;
        if (!w || !live[b]) return false;
        c.score = order_of(offset[b] + double(cand_logit(w)));
        c.place = (unsigned long long)b << 32 | cand_token(w);
        return true;
    };
    unsigned long long mine = 0;
    for (unsigned l = tid; l < lists; l += kMergeThreads) {
        Scored c;
        if (scored(l, 0, c) && c.score > mine) mine = c.score;
    }
    const unsigned long long limit = reached_by<unsigned long long, kMergeThreads / 32>(mine, n, bound_of);
    // the candidates at or above the bound (a list's come first in it); a full list is cut down, as above
    unsigned l = tid, k = 0;
    bool left = true;
    for (;;) {
        __syncthreads();
        if (left) {
            left = false;
            while (l < lists && !left) {
                Scored c;
                if (k < n && scored(l, k, c) && c.score >= limit) {
                    const unsigned at = atomicAdd(&n_found, 1u);
                    if (at < kFound) found[at] = c, ++k;
                    else left = true;
                } else {
                    l += kMergeThreads, k = 0;
                }
            }
        }
        const bool again = __syncthreads_or(left);
        const unsigned total = n_found < kFound ? n_found : kFound;
        for (unsigned i = tid; i < total; i += kMergeThreads) {
            const Scored c = found[i];
            unsigned r = 0;
            for (unsigned j = 0; j < total; ++j) r += before(found[j], c);
            if (r < n) kept[r] = c;
        }
        __syncthreads();
        if (!again) {
            for (unsigned i = tid; i < n; i += kMergeThreads) {
                const bool some = i < total;
                const unsigned b = some ? unsigned(kept[i].place >> 32) : kNoSlot;
                const unsigned long long s = some ? kept[i].score : 0;
                a.out[req * n + i] = some ? float(__longlong_as_double((long long)(s >> 63 ? s & ~(1ull << 63) : ~s))) : -INFINITY;
                a.parent[req * n + i] = b;
                a.token[req * n + i] = some ? unsigned(kept[i].place) : kNoSlot;
            }
            return;
        }
        for (unsigned i = tid; i < n; i += kMergeThreads) found[i] = kept[i];
        if (tid == 0) n_found = n;
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
    const bool wide = ((reinterpret_cast<uintptr_t>(a.logits) | a.stride * 4) & 15) == 0;
    const cudaError_t e = launch_pdl(wide ? beam_chunk_kernel<true> : beam_chunk_kernel<false>, dim3(chunks, rows), dim3(kSelThreads), 0, st, a, list, stat);
    if (e != cudaSuccess) return e;
    return launch_pdl(beam_merge_kernel, dim3(a.n_req), dim3(kMergeThreads), 0, st, a, static_cast<const unsigned long long *>(list),
                      static_cast<const float2 *>(stat), chunks);
}

cudaError_t launch_beam_reorder(const BeamReorderArgs &a, cudaStream_t st) {
    const size_t all = a.row_bytes | a.src_layer | a.dst_layer | reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.dst);
    if (all % 16 == 0) return launch_reorder<uint4>(a, st);
    if (all % 4 == 0) return launch_reorder<uint32_t>(a, st);
    return launch_reorder<uint8_t>(a, st);
}

}  // namespace b200q
