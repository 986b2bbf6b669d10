// Attention over the paged 4-bit cache.
//
// Row i of request r (its new tokens are the last of its kv_len tokens) stands at position p = kv_len - new + i and sees
// the keys (p - window, p] (window 0: [0, p]). For a query head h of KV head g = h / (n_head / n_kv)
//   y = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = scale q . k_t,  m = max_t s_t
// in one pass over the keys with the running m and sum. A row that sees nothing is zero.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv4.cuh"
#include "serve.h"

namespace b200q {
namespace {

__device__ __forceinline__ void tell(uint32_t *status, unsigned bit) {
    if (status) atomicOr(status, bit);
}

// One warp a (row, head): a lane scores a key, then the lanes share out the dims of the weighted sum.
__global__ void __launch_bounds__(32) kv4_attn_simple(const Kv4AttnArgs a) {
    __shared__ float q[kMaxKv4Dim];
    pdl_wait();
    pdl_launch_dependents();
    const unsigned row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, nb = a.c.dim / 32;
    if (row >= a.q_start[a.n_req]) return;
    unsigned lo = 0, hi = a.n_req;
    while (hi - lo > 1) {
        const unsigned mid = (lo + hi) / 2;
        if (a.q_start[mid] <= row) lo = mid;
        else hi = mid;
    }
    const unsigned start = a.q_start[lo], end = a.q_start[lo + 1], len = a.kv_len[lo];
    if (start > end || end > a.n_rows || end - start > a.max_q || len > a.max_kv || len > a.stride * (unsigned long long)a.c.page) {
        tell(a.status, kServeRequest);
        return;
    }
    const long long pos = (long long)len - (end - start) + (row - start);
    const long long first = a.window && pos + 1 > (long long)a.window ? pos + 1 - a.window : 0;
    const unsigned group = a.n_head / a.c.n_kv, g = h / group;
    for (unsigned d = lane; d < a.c.dim; d += 32) q[d] = a.q[row * a.q_stride + h * a.q_head_stride + d];
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o[kMaxKv4Dim / 32] = {};
    for (long long k0 = first / 32 * 32; k0 <= pos; k0 += 32) {
        const long long key = k0 + lane;
        float s = -INFINITY;
        unsigned page = 0;
        bool seen = key >= first && key <= pos;
        if (seen) {
            page = a.table[size_t(lo) * a.stride + unsigned(key) / a.c.page];
            if (page >= a.c.n_pages) {
                tell(a.status, kServePage);
                seen = false;
            }
        }
        const unsigned in = unsigned(key) % a.c.page, t = in % kTileTokens;
        const uint8_t *tile = a.c.base + ((size_t(page) * a.c.n_kv + g) * (a.c.page / kTileTokens) + in / kTileTokens) * kv4_tile_bytes(a.c.dim);
        if (seen) {
            s = 0.0f;
            for (unsigned b = 0; b < nb; ++b) {
                float x = 0.0f;
                for (unsigned w = 0; w < 4; ++w) {
                    const uint32_t c = *reinterpret_cast<const uint32_t *>(tile + kv4_k_word(nb, t, b, w));
                    for (unsigned e = 0; e < 8; ++e)
                        x += q[b * 32 + e / 4 * 16 + w * 4 + e % 4] * float(int(c >> (8 * (e % 4) + e / 4 * 4) & 15) - 8);
                }
                s += x * half_bits_to_float(*reinterpret_cast<const uint16_t *>(tile + kv4_k_scale(nb, t, b)));
            }
            s *= a.scale;
        }
        float top = s;
        for (unsigned x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
        const float mn = fmaxf(m, top);
        if (mn == -INFINITY && !__any_sync(~0u, seen)) continue;
        const float p = seen ? expf(s - mn) : 0.0f, alpha = m == mn ? 1.0f : expf(m - mn);
        float sum = p;
        for (unsigned x = 16; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
        l = l * alpha + sum;
        m = mn;
        for (unsigned b = 0; b < nb; ++b) o[b] *= alpha;
        for (unsigned i = 0; i < 32; ++i) {
            const float pi = __shfl_sync(~0u, p, i);
            const unsigned long long ti = __shfl_sync(~0u, (unsigned long long)tile, i);
            const unsigned tt = __shfl_sync(~0u, t, i);
            if (!__shfl_sync(~0u, int(seen), i)) continue;
            const uint8_t *src = reinterpret_cast<const uint8_t *>(ti);
            for (unsigned b = 0; b < nb; ++b) {
                const uint32_t c = *reinterpret_cast<const uint32_t *>(src + kv4_v_word(nb, tt, b, lane % 16 / 4));
                const float d = half_bits_to_float(*reinterpret_cast<const uint16_t *>(src + kv4_v_scale(nb, tt, b)));
                o[b] += pi * (d * float(int(c >> (8 * (lane % 4) + lane / 16 * 4) & 15) - 8));
            }
        }
    }
    for (unsigned b = 0; b < nb; ++b) a.y[row * a.y_stride + size_t(h) * a.c.dim + b * 32 + lane] = l == 0.0f ? 0.0f : o[b] / l;
}

}  // namespace

size_t kv4_attn_room(const Kv4AttnArgs &, unsigned) { return 16; }
unsigned kv4_attn_launches(const Kv4AttnArgs &, unsigned) { return 1; }

cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, unsigned, cudaStream_t st) {
    if (a.n_rows == 0) return cudaSuccess;
    return launch_pdl(kv4_attn_simple, dim3(a.n_rows, a.n_head), dim3(32), 0, st, a);
}

}  // namespace b200q
