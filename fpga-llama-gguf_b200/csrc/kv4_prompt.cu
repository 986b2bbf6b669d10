// Attention over the paged 4-bit cache for prompts: requests with many rows, on the fifth-generation tensor cores.
//
// A CTA takes 128 query rows (token, head of the group) of one KV head and goes over the keys 64 at a time, with FP32
// sums and outputs as in kv4_attn.cu:
//   S = Q K^T        FP32 accuracy from FP16 products: q = qh + ql (22 bits; rows scaled by a power of two), and a value of
//                    the cache is d (c - 8), a multiple of FP16's smallest number of at most 15 bits, so kh + kl holds it
//                    exactly: S = qh kh + ql kh + qh kl (what ql kl would add is below 2^-22 of a product). ql and kl are
//                    held 2^11 times as large, so that a number of q has its 22 bits down to 2^28 below the row's largest
//   P = 2^(s - m)    the running maximum m of a row moves only when a score passes it
//   O += P V         the same way: ph vh + pl vh + ph vl, in tensor memory and, by turns, on to FP32 sums
// Values of 2^16 and more do not fit FP16: a token's K or V with a d of 2^13 or more is lowered by 2^e, e = 1 to 3, so that
// its largest d is below 2^13. All others enter as they are, whatever their magnitude and however far a token's blocks lie
// apart. (The largest d of every token raised to 1/2, as it was once, made subnormals of d 2^14 below it and lost their bits;
// now only such a token's d below 2^-11 lose some, 2^-37 of its largest one at most.) K's 2^e comes back in as a factor of the
// key's column of S; V's, e_t, moves into the weight: w_t = 2^(s_t + e_t - m), and the sum of the weights takes w_t / 2^e_t.
//
// Operands: qh, kh, kl, vh, vl in shared memory (no swizzle; K is K-major, V MN-major, both written 16 bytes = 8 dims of a
// key at a time by the same code), ql and P in tensor memory. kl lies behind kh, so that one product of N 128 forms qh kh and
// qh kl side by side and qh, whose reads bound the products of N 64, is read once for both. In a step 8 warps
//   unpack V    while the tensor cores form S
//   soften      S from tensor memory, P back into its place (lane = row; two warps share a row's 64 keys)
//   unpack the next K    while the tensor cores add P V
// A ninth warp issues the products (which holds it up while the tensor cores are busy) and the raw tiles' bulk copies.
//
// 4 requests of 200 to 2048 new tokens on up to 2560 keys, 16 heads of 256: 320 us, 200 TFLOP/s of the plain products, three times
// that on the tensor cores, which are busy a third of the time; of 128: 227 us, of 64: 196. Of a step of 64 keys at 256 dims S
// takes 2800 cycles, the softmax 1000 to 2000, P V 2100, one after another: O, S and ql fill tensor memory. With smaller
// heads they do not, and there it is the same order all the same.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv4.cuh"
#include "launch.h"
#include "serve.h"
#include "tcgen05.cuh"

namespace b200q {
namespace {

constexpr unsigned kRows = 128, kKeys = 64, kWork = 256, kThreads = kWork + 32;  // 8 warps, and one that issues products and copies
constexpr unsigned kBadMax = 96;  // values that are not numbers, remembered by (key, block)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLow = 2048.0f;  // ql and kl are 2^11 times what they stand for, so that they seldom are subnormal

__device__ __forceinline__ void tell(uint32_t *status, unsigned bit) {
    if (status) atomicOr(status, bit);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2(half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ half2 as_h2(uint32_t x) { return *reinterpret_cast<half2 *>(&x); }
// two FP32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(unsigned(127 + e) << 23); }

template <int NB>
struct Prompt {
    static constexpr int D = NB * 32, kTile = NB * 576;
    static constexpr int kQ = kRows * D * 2, kPart = kKeys * D * 2;
    static constexpr int kRaw = kQ + 4 * kPart, kSmem = kRaw + 4 * kTile;
    // columns of tensor memory: O, S (qh kh, then qh kl + ql kh: the sums in tensor memory drop what is below their last bit, so
    // that the small products go to a sum of their own; P takes the place of the former, 32 keys' upper and lower parts by
    // 16 columns), ql
    static constexpr unsigned kS = D, kQl = D + 128, kNeed = D + 128 + D / 2;
    static constexpr unsigned kCols = kNeed <= 256 ? 256 : 512;
    static_assert(kNeed <= 512 && kSmem <= 216 * 1024);
    // Tensor memory's sums drop what is below their last bit, half of it on average, 12 times a step. So O moves on to FP32 sums by
    // turns: in every step a thread adds kParts of its NB runs of 16 dims to them and clears the runs, while the tensor cores
    // form S, and each run is moved every kTurns steps. The sums of kHeld runs are in registers (with more, others spill), those
    // of the rest lie in y. Error of the result and us, 4 requests of 2048 on up to 2560 keys, 16 heads of 256 (of 128):
    //   all of O to y every 32 steps, before the softmax   3.1 10^-6  307  (2.9 10^-6  221)
    //   every 8                                            1.8        376  (1.5        246)
    //   by turns                                           1.4        320  (1.2        227)
    //   by turns, no run in registers                      1.4        328  (1.2        235)
    // and FP32 arithmetic is off by 1.0 (0.8) 10^-6.
    static constexpr unsigned kParts = (NB + 3) / 4, kTurns = (NB + kParts - 1) / kParts, kHeld = NB < 2 ? NB : 2;
};

__device__ __forceinline__ void work_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kWork) : "memory"); }
__device__ __forceinline__ bool work_sync_or(bool x) {
    uint32_t y;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(y)
                 : "r"(uint32_t(x)), "n"(kWork)
                 : "memory");
    return y;
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

template <int NB>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const Kv4AttnArgs a, unsigned least_rows) {
    using S = Prompt<NB>;
    constexpr int D = S::D;
    extern __shared__ __align__(1024) uint8_t smem[];
    // S formed, P V added, raw tiles there; K unpacked, V unpacked (and the raw tiles read), P stored: an arrival a warp
    __shared__ uint64_t bar_s, bar_o, bar_raw, bar_k, bar_v, bar_p;
    __shared__ uint32_t tm_base;
    __shared__ __align__(16) float k_scale[kKeys], v_log[kKeys], v_inv[kKeys];  // read four at a time
    __shared__ float row_top[2][kRows];
    __shared__ unsigned present, n_bad, bad[kBadMax];
    __shared__ unsigned whole_of[kThreads / 32], count_of[kThreads / 32], found_req, found_tile;
    const unsigned tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned per = a.n_head / a.c.n_kv, head = blockIdx.x % a.c.n_kv;
    pdl_wait();
    pdl_launch_dependents();

    // The CTA's tile: those of all requests with enough rows lie in one line, the last (which see the most keys) come first. A
    // thread counts some requests; one is left out as kv4_attn.cu says, when its rows or lengths lie outside the bounds.
    const unsigned each = (a.n_req + kThreads - 1) / kThreads, r0 = tid * each < a.n_req ? tid * each : a.n_req, r1 = r0 + each < a.n_req ? r0 + each : a.n_req;
    unsigned whole = a.n_req;  // the requests before the first whose rows run backwards
    for (unsigned r = r1; r > r0; --r)
        if (a.q_start[r - 1] > a.q_start[r]) whole = r - 1;
    whole = __reduce_min_sync(~0u, whole);
    if (lane == 0) whole_of[warp] = whole;
    __syncthreads();
    for (unsigned w = 0; w < kThreads / 32; ++w) whole = min(whole, whole_of[w]);
    auto tiles_of = [&](unsigned r) {
        const unsigned s = a.q_start[r], e = a.q_start[r + 1];
        if (r >= whole || e > a.n_rows || e - s > a.max_q || a.kv_len[r] > a.max_kv || (e - s) * per < least_rows) return 0u;
        return ((e - s) * per + kRows - 1) / kRows;
    };
    unsigned count = 0;
    for (unsigned r = r0; r < r1; ++r) count += tiles_of(r);
    unsigned upto = count;
    for (unsigned o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) count_of[warp] = upto;
    __syncthreads();
    unsigned total = 0;
    for (unsigned w = 0; w < kThreads / 32; ++w) {
        if (w < warp) upto += count_of[w];
        total += count_of[w];
    }
    const unsigned turn = blockIdx.x / a.c.n_kv, mine = total - 1 - turn;
    if (turn >= total) return;
    if (mine < upto && mine >= upto - count) {
        unsigned at = upto - count, r = r0;
        while (at + tiles_of(r) <= mine) at += tiles_of(r++);
        found_req = r;
        found_tile = mine - at;
    }
    __syncthreads();
    const unsigned req = found_req, row0 = found_tile * kRows;
    const unsigned start = a.q_start[req], end = a.q_start[req + 1], len = a.kv_len[req], all = (end - start) * per;
    const int base = int(len) - int(end - start);
    const unsigned last = row0 + kRows < all ? row0 + kRows - 1 : all - 1;
    const int hi = base + int(last / per), first_pos = base + int(row0 / per);
    const int lo = a.window && first_pos >= 0 && unsigned(first_pos) + 1 > a.window ? first_pos + 1 - int(a.window) : 0;

    // this thread's row (lane of tensor memory), and its half of the keys or dims
    const unsigned quarter = warp & 3, half_ = warp >> 2 & 1, row = quarter * 32 + lane, at_row = row0 + row;
    const bool real = at_row < all;
    const int pos = real ? base + int(at_row / per) : -1;
    const int low = a.window && pos >= 0 && unsigned(pos) + 1 > a.window ? pos + 1 - int(a.window) : 0;
    float *y = a.y + (start + (real ? at_row / per : 0)) * a.y_stride + size_t(head * per + (real ? at_row % per : 0)) * D;
    if (hi < 0) {  // no row of the tile sees anything
        if (real && warp < kWork / 32)
            for (unsigned d = 0; d < D / 2; ++d) y[half_ * (D / 2) + d] = 0.0f;
        return;
    }
    const unsigned step0 = unsigned(lo) / kKeys, steps = unsigned(hi) / kKeys + 1 - step0;

    if (warp == 0) tm_alloc(&tm_base, S::kCols);
    if (tid == 0) {
        mbar_init(&bar_s, 1);
        mbar_init(&bar_o, 1);
        mbar_init(&bar_raw, 1);
        mbar_init(&bar_k, kWork / 32);
        mbar_init(&bar_v, kWork / 32);
        mbar_init(&bar_p, kWork / 32);
        mbar_fence_init();
        n_bad = 0;
    }
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    const uint32_t tm = tm_base, tm_lane = tm + (quarter * 32 << 16);
    uint8_t *const kh = smem + S::kQ, *const kl = kh + S::kPart, *const vh = kl + S::kPart, *const vl = vh + S::kPart, *const raw = smem + S::kRaw;

    const uint32_t q_at = smem_addr(smem), kh_at = smem_addr(kh), vh_at = smem_addr(vh), vl_at = smem_addr(vl);
    bool fail = false;
    if (warp == kWork / 32) {
        // the warp that issues: raw tiles (a bulk copy each, those behind the last key or without a page left out) and products
        const unsigned tiles_per_page = a.c.page / kTileTokens;
        const uint8_t *src;
        auto look_up = [&](unsigned j) {
            const unsigned tile = (step0 + j) * (kKeys / kTileTokens) + lane;
            src = nullptr;
            if (j < steps && lane < kKeys / kTileTokens && int(tile * kTileTokens) <= hi) {
                const unsigned page = a.table[size_t(req) * a.stride + tile / tiles_per_page];
                if (page < a.c.n_pages)
                    src = a.c.base + ((size_t(page) * a.c.n_kv + head) * tiles_per_page + tile % tiles_per_page) * S::kTile;
                else tell(a.status, kServePage);
            }
        };
        auto fetch = [&] {
            const unsigned there = __ballot_sync(~0u, src != nullptr);
            if (lane == 0) {
                present = there;
                mbar_expect_tx(&bar_raw, __popc(there) * S::kTile);
            }
            __syncwarp();
            if (src)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                 smem_addr(raw + lane * S::kTile)),
                             "l"(src), "r"(S::kTile), "r"(smem_addr(&bar_raw))
                             : "memory");
        };
        auto reached = [&](uint64_t *bar, unsigned phase) { return __all_sync(~0u, mbar_wait(bar, phase & 1)); };
        look_up(0);
        fetch();
        for (unsigned j = 0; j < steps && !fail; ++j) {
            look_up(j + 1);
            if ((fail = !reached(&bar_k, j) || (j && !reached(&bar_o, j - 1)))) break;  // (S takes P's place)
            tm_fence_after();
            if (lane == 0) {
#pragma unroll 1
                for (unsigned k = 0; k < D / 16; ++k) {
                    const uint64_t kk = tm_operand(kh_at + k * 256, 128, D * 16);
                    tm_mma(tm + S::kS, tm_operand(q_at + k * 256, 128, D * 16), kk, tm_f16(2 * kKeys, false), k != 0);
                    tm_mma_t(tm + S::kS + kKeys, tm + S::kQl + k * 8, kk, tm_f16(kKeys, false), true);
                }
                tm_commit(&bar_s);
            }
            __syncwarp();
            if ((fail = !reached(&bar_v, j))) break;
            if (j + 1 < steps) fetch();
            if ((fail = !reached(&bar_p, j))) break;
            tm_fence_after();
            if (lane == 0) {
#pragma unroll 1
                for (unsigned k = 0; k < kKeys / 16; ++k) {
                    const uint64_t v = tm_operand(vh_at + k * (D * 32), D * 16, 128);
                    const uint32_t p = tm + S::kS + k / 2 * 32 + k % 2 * 8;
                    tm_mma_t(tm, p, v, tm_f16(D, true), j || k);
                    tm_mma_t(tm, p, tm_operand(vl_at + k * (D * 32), D * 16, 128), tm_f16(D, true), true);
                    tm_mma_t(tm, p + 16, v, tm_f16(D, true), true);
                }
                tm_commit(&bar_o);
            }
            __syncwarp();
        }
    } else {
    // Q: rows scaled to below 2^15; the upper parts to shared memory, the lower ones to tensor memory, by way of V's place.
    // A warp takes a row at a time, its lanes four dims each.
    float row_scale;
    {
        const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | a.q_stride * 4 | a.q_head_stride * 4) & 15) == 0;
        constexpr unsigned kTurns = (D / 4 + 31) / 32, kAhead = 4;  // rows whose loads are on their way together
        for (unsigned r0 = warp; r0 < kRows; r0 += kAhead * (kWork / 32)) {
            float4 v[kAhead][kTurns];
#pragma unroll
            for (unsigned i = 0; i < kAhead; ++i) {
                const unsigned at = row0 + r0 + i * (kWork / 32);
                const float *q = a.q + (start + (at < all ? at / per : 0)) * a.q_stride + (head * per + (at < all ? at % per : 0)) * a.q_head_stride;
#pragma unroll
                for (unsigned n = 0; n < kTurns; ++n) {
                    const unsigned d = (n * 32 + lane) * 4;
                    v[i][n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (at >= all || d >= D) continue;
                    if (wide) v[i][n] = *reinterpret_cast<const float4 *>(q + d);
                    else v[i][n] = make_float4(q[d], q[d + 1], q[d + 2], q[d + 3]);
                }
            }
#pragma unroll
            for (unsigned i = 0; i < kAhead; ++i) {
                const unsigned r = r0 + i * (kWork / 32);
                float top = 0.0f;
#pragma unroll
                for (unsigned n = 0; n < kTurns; ++n)
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(v[i][n].x), fabsf(v[i][n].y)), fmaxf(fabsf(v[i][n].z), fabsf(v[i][n].w))));
                for (unsigned x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
                int ex = int(__float_as_uint(top) >> 23) - 127 - 14;
                ex = ex < -110 ? -110 : ex > 113 ? 113 : ex;  // (NaN, infinity: what they are)
                const float down = pow2(-ex);
                if (lane == 0) row_top[0][r] = a.scale * kLog2e * pow2(ex);
#pragma unroll
                for (unsigned n = 0; n < kTurns; ++n) {
                    const unsigned d = (n * 32 + lane) * 4;
                    if (d >= D) continue;
                    const float4 y = make_float4(v[i][n].x * down, v[i][n].y * down, v[i][n].z * down, v[i][n].w * down);
                    const half2 p = __floats2half2_rn(y.x, y.y), q = __floats2half2_rn(y.z, y.w);
                    const float2 bp = __half22float2(p), bq = __half22float2(q);
                    const unsigned at = r / 8 * (D * 16) + d / 8 * 128 + r % 8 * 16 + d % 8 * 2;
                    *reinterpret_cast<uint2 *>(smem + at) = make_uint2(h2(p), h2(q));
                    *reinterpret_cast<uint2 *>(vh + at) = make_uint2(h2(__floats2half2_rn((y.x - bp.x) * kLow, (y.y - bp.y) * kLow)), h2(__floats2half2_rn((y.z - bq.x) * kLow, (y.w - bq.y) * kLow)));
                }
            }
        }
        work_sync();
        row_scale = row_top[0][row];
        for (unsigned d = half_ * (D / 2); d < (half_ + 1) * (D / 2); d += 16) {
            uint32_t low_part[8];
#pragma unroll
            for (unsigned g = 0; g < 2; ++g) {
                const uint4 x = *reinterpret_cast<const uint4 *>(vh + row / 8 * (D * 16) + (d / 8 + g) * 128 + row % 8 * 16);
                low_part[4 * g] = x.x, low_part[4 * g + 1] = x.y, low_part[4 * g + 2] = x.z, low_part[4 * g + 3] = x.w;
            }
            tm_store8(tm_lane + S::kQl + d / 2, low_part);
        }
        tm_wait_store();
        work_sync();  // (V's place and row_top are read)
    }

    // Raw tiles to FP16 pairs of operands. A warp takes 8 keys, a lane a key and every fourth block.
    const unsigned key = warp * 8 + lane % 8, token = key % kTileTokens;
    const uint8_t *const my_tile = raw + key / kTileTokens * S::kTile;
    auto unpack = [&](unsigned j, bool is_v, uint8_t *up, uint8_t *down) {
        const int at = int((step0 + j) * kKeys + key);
        const bool hidden = at > hi || !(present >> key / kTileTokens & 1);
        half d[(NB + 3) / 4];
        float top = 0.0f;
#pragma unroll
        for (int p = 0; p < (NB + 3) / 4; ++p) {
            const unsigned b = p * 4 + lane / 8;
            d[p] = __float2half_rn(0.0f);
            if (b < NB && !hidden) {
                d[p] = *reinterpret_cast<const half *>(my_tile + (is_v ? NB * 544 : NB * 512) + (token * NB + b) * 2);
                if (is_v && !(fabsf(__half2float(d[p])) <= 65504.0f)) {  // set apart, lest it reach rows that do not see the key
                    const unsigned n = atomicAdd(&n_bad, 1u);
                    if (n < kBadMax) bad[n] = unsigned(at) * 8 + b;
                    d[p] = __float2half_rn(0.0f);
                }
                top = fmaxf(top, fabsf(__half2float(d[p])));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
        const int over = int(__float_as_uint(fminf(top, 65504.0f)) >> 23) - 139, e = over > 0 ? over : 0;  // top / 2^e is below 2^13
        if (lane < 8) {
            if (is_v) v_log[key] = hidden ? -INFINITY : float(e), v_inv[key] = pow2(-e);
            else k_scale[key] = pow2(e);
        }
#pragma unroll
        for (int p = 0; p < (NB + 3) / 4; ++p) {
            const int nbp = NB - 4 * p < 4 ? NB - 4 * p : 4;
            const unsigned bq = lane / 8, b = p * 4 + bq;
            if (int(bq) >= nbp) continue;
            const half2 dd = __half2half2(__float2half_rn(__half2float(d[p]) * pow2(-e)));
            const uint8_t *words = my_tile + p * 1024 + (is_v ? NB * 256 + ((token / 8 * 2 + token % 2) * 16 + token / 2 % 4) * nbp * 4 : token * 16 * nbp) + bq * 4;
            const unsigned word_step = is_v ? 16 * nbp : 4 * nbp;
            uint8_t *const to = up + warp * (D * 16) + b * 512 + lane % 8 * 16, *const to_low = down + (to - up);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t hi_of[2][4], lo_of[2][4];  // low nibbles' 8 dims, high nibbles' 8 dims
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t w = hidden ? 0x88888888u : *reinterpret_cast<const uint32_t *>(words + (2 * u + i) * word_step);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t pair = __byte_perm(w, 0u, x ? 0x4342 : 0x4140);  // two bytes, 16 bits apart
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const half2 c = __hsub2(as_h2((pair >> (4 * n) & 0x000f000fu) | 0x64006400u), as_h2(0x64086408u));
                            const half2 v = __hmul2(c, dd);
                            hi_of[n][2 * i + x] = h2(v);
                            const half2 rest = __hfma2(c, dd, __hneg2(v));
                            lo_of[n][2 * i + x] = h2(is_v ? rest : __hmul2(rest, __float2half2_rn(kLow)));
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    *reinterpret_cast<uint4 *>(to + (2 * n + u) * 128) = make_uint4(hi_of[n][0], hi_of[n][1], hi_of[n][2], hi_of[n][3]);
                    *reinterpret_cast<uint4 *>(to_low + (2 * n + u) * 128) = make_uint4(lo_of[n][0], lo_of[n][1], lo_of[n][2], lo_of[n][3]);
                }
            }
        }
    };
    auto hand_over = [&](uint64_t *bar) {  // what this warp wrote, to the issuing warp and the tensor cores
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tm_fence_before();
        __syncwarp();
        if (lane == 0) arrive(bar);
    };

    // A wait that ran out, for the whole warp: its lanes stay together in what follows.
    auto missed = [&](uint64_t *bar, unsigned phase) { return !__all_sync(~0u, mbar_wait(bar, phase & 1)); };
    fail = missed(&bar_raw, 0);
    if (!fail) unpack(0, false, kh, kl);
    hand_over(&bar_k);
    float top = -INFINITY, sum = 0.0f;
    // The FP32 sums, and the maxima that each turn's were formed with (-inf: there is nothing in them yet)
    float moved[S::kHeld][16], moved_top[S::kTurns];
#pragma unroll
    for (unsigned i = 0; i < S::kTurns; ++i) moved_top[i] = -INFINITY;
#pragma unroll
    for (unsigned i = 0; i < S::kHeld; ++i)
#pragma unroll
        for (unsigned e = 0; e < 16; ++e) moved[i][e] = 0.0f;
    // y goes out and comes back by whole sectors of 32 bytes where it lies so (half a sector at a time takes twice as long)
    const unsigned y_align = unsigned(reinterpret_cast<uintptr_t>(a.y) | a.y_stride * 4);
    auto from_y = [&](unsigned c, float (&v)[16]) {
        const float *at = y + c;
        if (y_align % 32 == 0) {
#pragma unroll
            for (unsigned e = 0; e < 16; e += 8)
                asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=f"(v[e]), "=f"(v[e + 1]), "=f"(v[e + 2]), "=f"(v[e + 3]), "=f"(v[e + 4]), "=f"(v[e + 5]), "=f"(v[e + 6]), "=f"(v[e + 7])
                             : "l"(at + e)
                             : "memory");
        } else if (y_align % 16 == 0) {
#pragma unroll
            for (unsigned e = 0; e < 16; e += 4) {
                const float4 x = *reinterpret_cast<const float4 *>(at + e);
                v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
            }
        } else {
#pragma unroll
            for (unsigned e = 0; e < 16; ++e) v[e] = at[e];
        }
    };
    auto to_y = [&](unsigned c, const float (&v)[16]) {
        float *at = y + c;
        if (y_align % 32 == 0) {
#pragma unroll
            for (unsigned e = 0; e < 16; e += 8)
                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at + e), "f"(v[e]), "f"(v[e + 1]), "f"(v[e + 2]),
                             "f"(v[e + 3]), "f"(v[e + 4]), "f"(v[e + 5]), "f"(v[e + 6]), "f"(v[e + 7])
                             : "memory");
        } else if (y_align % 16 == 0) {
#pragma unroll
            for (unsigned e = 0; e < 16; e += 4) *reinterpret_cast<float4 *>(at + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
#pragma unroll
            for (unsigned e = 0; e < 16; ++e) at[e] = v[e];
        }
    };
    unsigned j = 0;
    for (; j < steps; ++j) {
        if (j && !fail) fail = missed(&bar_o, j - 1);  // V is free, O is there
        const bool move = j >= S::kTurns && !fail;
        const unsigned turn = j % S::kTurns;
        float last_top = -INFINITY, was[S::kParts][16];
#pragma unroll
        for (unsigned i = 0; i < S::kTurns; ++i) last_top = i == turn ? moved_top[i] : last_top;
        const bool held = move && last_top != -INFINITY;
        if (S::kHeld < NB) {
#pragma unroll
            for (unsigned i = 0; i < S::kParts; ++i) {
                const unsigned run = turn * S::kParts + i;
#pragma unroll
                for (unsigned e = 0; e < 16; ++e) was[i][e] = 0.0f;
                if (held && real && run >= S::kHeld && run < NB) from_y(half_ * (D / 2) + run * 16, was[i]);
            }
        }
        if (!fail) unpack(j, true, vh, vl);
        hand_over(&bar_v);
        if (move) {
            tm_fence_after();
            const float f = held ? exp2_fast(last_top - top) : 0.0f;
#pragma unroll
            for (unsigned i = 0; i < S::kParts; ++i) {
                const unsigned run = turn * S::kParts + i, c = half_ * (D / 2) + run * 16;
                if (run >= NB) continue;
                uint32_t o[16];
                tm_load16(tm_lane + c, o);
#pragma unroll
                for (unsigned r = 0; r < S::kHeld; ++r) {
                    if (r != run) continue;
#pragma unroll
                    for (unsigned e = 0; e < 16; ++e) moved[r][e] = fmaf(moved[r][e], f, __uint_as_float(o[e]));
                }
                if (run >= S::kHeld && real) {
#pragma unroll
                    for (unsigned e = 0; e < 16; ++e) was[i][e] = fmaf(was[i][e], f, __uint_as_float(o[e]));
                    to_y(c, was[i]);
                }
#pragma unroll
                for (unsigned e = 0; e < 16; ++e) o[e] = 0;
                tm_store16(tm_lane + c, o);
            }
#pragma unroll
            for (unsigned i = 0; i < S::kTurns; ++i) moved_top[i] = i == turn ? top : moved_top[i];
        }

        // scores of the row and 32 keys, in powers of two
        if (!fail) fail = missed(&bar_s, j);
        if ((fail = work_sync_or(fail))) break;  // (and all keys' scales are there)
        tm_fence_after();
        uint32_t s[32], s_low[32];
        tm_load32(tm_lane + S::kS + half_ * 32, s);
        tm_load32(tm_lane + S::kS + kKeys + half_ * 32, s_low);
        const int key0 = int((step0 + j) * kKeys + half_ * 32);
        float mx = -INFINITY;
        const bool edge = __any_sync(~0u, key0 < low || key0 + 31 > pos);
        const float2 scale2 = make_float2(row_scale, row_scale);
        float2 w[16];
#pragma unroll
        for (unsigned i = 0; i < 16; i += 2) {
            const float4 ks = *reinterpret_cast<const float4 *>(k_scale + half_ * 32 + 2 * i), vg = *reinterpret_cast<const float4 *>(v_log + half_ * 32 + 2 * i);
            const float2 f[2] = {make_float2(ks.x, ks.y), make_float2(ks.z, ks.w)}, g[2] = {make_float2(vg.x, vg.y), make_float2(vg.z, vg.w)};
#pragma unroll
            for (unsigned e = 0; e < 2; ++e) {
                const unsigned k = 2 * (i + e);
                const float2 x = fma2(make_float2(__uint_as_float(s_low[k]), __uint_as_float(s_low[k + 1])), make_float2(1.0f / kLow, 1.0f / kLow),
                                      make_float2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])));
                w[i + e] = fma2(mul2(x, f[e]), scale2, g[e]);  // (a hidden key: -inf)
            }
        }
        if (edge) {
#pragma unroll
            for (unsigned i = 0; i < 16; ++i) {
                const int key = key0 + int(2 * i);
                if (key < low || key > pos) w[i].x = -INFINITY;
                if (key + 1 < low || key + 1 > pos) w[i].y = -INFINITY;
            }
        }
#pragma unroll
        for (unsigned i = 0; i < 16; ++i) mx = fmaxf(mx, fmaxf(w[i].x, w[i].y));
        row_top[half_][row] = mx;
        work_sync();
        mx = fmaxf(mx, row_top[half_ ^ 1][row]);
        if (__any_sync(~0u, mx > top)) {  // a higher maximum: 4 above the score, so that it moves seldom
            const float nt = mx > top ? mx + 4.0f : top, f = top == nt ? 1.0f : exp2_fast(top - nt);
            sum *= f;
            top = nt;
            if (j) {
                tm_wait_store();  // (of runs that were cleared)
                for (unsigned c = half_ * (D / 2); c < (half_ + 1) * (D / 2); c += 16) {
                    uint32_t o[16];
                    tm_load16(tm_lane + c, o);
#pragma unroll
                    for (unsigned e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tm_store16(tm_lane + c, o);
                }
            }
        }
        const float lift = top == -INFINITY ? 0.0f : 14.0f - top;  // weights up to 2^14
        uint32_t ph[16], pl[16];
        float2 sum2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (unsigned i = 0; i < 16; i += 2) {
            const float4 vi = *reinterpret_cast<const float4 *>(v_inv + half_ * 32 + 2 * i);
            const float2 g[2] = {make_float2(vi.x, vi.y), make_float2(vi.z, vi.w)};
#pragma unroll
            for (unsigned e = 0; e < 2; ++e) {
                const float2 x = add2(w[i + e], make_float2(lift, lift)), y = make_float2(exp2_fast(x.x), exp2_fast(x.y));
                sum2 = fma2(y, g[e], sum2);
                const half2 h = __floats2half2_rn(y.x, y.y);
                const float2 b = __half22float2(h), z = add2(y, make_float2(-b.x, -b.y));
                ph[i + e] = h2(h);
                pl[i + e] = h2(__floats2half2_rn(z.x, z.y));
            }
        }
        sum += sum2.x + sum2.y;
        tm_store16(tm_lane + S::kS + half_ * 32, ph);
        tm_store16(tm_lane + S::kS + half_ * 32 + 16, pl);
        tm_wait_store();
        hand_over(&bar_p);
        if (j + 1 < steps) {
            fail = missed(&bar_raw, j + 1);
            if (!fail) unpack(j + 1, false, kh, kl);
            hand_over(&bar_k);
        }
    }
    if (!fail) fail = missed(&bar_o, steps - 1);
    tm_fence_after();
    work_sync();  // (the last maxima are read)
    row_top[half_][row] = sum;
    if (work_sync_or(fail)) {
        // some wait ran out: say so, let what is on its way land (each wait is bounded again), and give back what is held
        if (tid == 0) {
            tell(a.status, kServeWait);
            for (unsigned i = 0; i < 2; ++i) mbar_wait(&bar_raw, i), mbar_wait(&bar_s, i), mbar_wait(&bar_o, i);
        }
    } else {
        sum = row_top[0][row] + row_top[1][row];
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        // a value that is not a number makes its block's dims so, in the rows that see it
        unsigned nan_blocks = 0;
        const unsigned nb = n_bad < kBadMax ? n_bad : kBadMax;
        for (unsigned i = 0; i < nb; ++i)
            if (int(bad[i] / 8) >= low && int(bad[i] / 8) <= pos) nan_blocks |= 1u << bad[i] % 8;
        if (n_bad > kBadMax) {  // more than are remembered: the scales again, those of the keys this row sees
            const unsigned tiles_per_page = a.c.page / kTileTokens;
            for (int k = low; k <= pos; ++k) {
                const unsigned tile = unsigned(k) / kTileTokens, page = a.table[size_t(req) * a.stride + tile / tiles_per_page];
                if (page >= a.c.n_pages) continue;
                const auto *d = reinterpret_cast<const half *>(a.c.base + ((size_t(page) * a.c.n_kv + head) * tiles_per_page + tile % tiles_per_page) * S::kTile +
                                                               NB * 544 + unsigned(k) % kTileTokens * NB * 2);
                for (unsigned b = 0; b < NB; ++b)
                    if (!(fabsf(__half2float(d[b])) <= 65504.0f)) nan_blocks |= 1u << b;
            }
        }
        auto finish = [&](unsigned run, float (&v)[16], float back) {
            const unsigned c = half_ * (D / 2) + run * 16;
            uint32_t o[16];
            tm_load16(tm_lane + c, o);
            const bool bad_block = nan_blocks >> c / 32 & 1;
#pragma unroll
            for (unsigned e = 0; e < 16; ++e) {
                v[e] = fmaf(v[e], back, __uint_as_float(o[e])) * f;
                if (sum == 0.0f) v[e] = 0.0f;
                if (bad_block) v[e] = __uint_as_float(0x7fc00000u);
            }
            if (real) to_y(c, v);
        };
#pragma unroll
        for (unsigned run = 0; run < NB; ++run) {
            const float was_top = moved_top[run / S::kParts], back = was_top != -INFINITY ? exp2_fast(was_top - top) : 0.0f;
            if (run < S::kHeld) {
                finish(run, moved[run < S::kHeld ? run : 0], back);
            } else {
                float v[16] = {};
                if (real && was_top != -INFINITY) from_y(half_ * (D / 2) + run * 16, v);
                finish(run, v, back);
            }
        }
    }
    }
    tm_fence_before();
    __syncthreads();
    if (warp == 0) {
        tm_fence_after();
        tm_free(tm, S::kCols);
    }
}

// the most tiles that n_rows rows of requests of least_rows and more can make
unsigned long long prompt_tiles(const Kv4AttnArgs &a, unsigned least_rows) {
    const unsigned long long rows = (unsigned long long)a.n_rows * (a.n_head / a.c.n_kv), requests = rows / least_rows;
    return rows / kRows + (requests < a.n_req ? requests : a.n_req) + 1;
}

template <int NB>
cudaError_t launch_prompt(const Kv4AttnArgs &a, unsigned least_rows, cudaStream_t st) {
    using S = Prompt<NB>;
    const cudaError_t e = ensure_smem_attr(reinterpret_cast<const void *>(kv4_prompt_kernel<NB>), S::kSmem);
    if (e != cudaSuccess) return e;
    return launch_pdl(a.pdl, kv4_prompt_kernel<NB>, dim3(unsigned(prompt_tiles(a, least_rows)) * a.c.n_kv), dim3(kThreads), S::kSmem, st, a, least_rows);
}

}  // namespace

cudaError_t launch_kv4_prompt(const Kv4AttnArgs &a, unsigned least_rows, cudaStream_t st) {
    switch (a.c.dim / 32) {
    case 1: return launch_prompt<1>(a, least_rows, st);
    case 2: return launch_prompt<2>(a, least_rows, st);
    case 3: return launch_prompt<3>(a, least_rows, st);
    case 4: return launch_prompt<4>(a, least_rows, st);
    case 5: return launch_prompt<5>(a, least_rows, st);
    case 6: return launch_prompt<6>(a, least_rows, st);
    case 7: return launch_prompt<7>(a, least_rows, st);
    case 8: return launch_prompt<8>(a, least_rows, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace b200q
