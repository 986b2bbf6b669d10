// Shapes that the operators for several sequences take (include/b200q.h), for the entry points and the list planner. No CUDA.
#pragma once
#include <cstddef>
#include <cstdint>

namespace b200q {

constexpr unsigned kTileTokens = 16;  // tokens of one cache tile
constexpr unsigned kMaxKv4Dim = 256, kMaxPage = 4096, kMaxKvHeads = 256, kMaxBeams = 32, kMaxBeamOut = 64, kMaxVocab = 1u << 20;
constexpr unsigned kMaxMapReq = 65535, kMaxAttnReq = 4096, kMaxSelectReq = 2047;

// a tile: K codes, V codes (8 dim bytes each), K scales, V scales (dim bytes each) of 16 tokens of one KV head
#if defined(__CUDACC__)
__host__ __device__
#endif
inline unsigned kv4_tile_bytes(unsigned dim) { return 18 * dim; }

inline bool page_ok(unsigned page) { return page >= kTileTokens && page <= kMaxPage && page % kTileTokens == 0; }
inline bool kv4_shape_ok(unsigned n_pages, unsigned page, unsigned n_kv, unsigned dim) {
    return dim >= 32 && dim <= kMaxKv4Dim && dim % 32 == 0 && page_ok(page) && n_kv >= 1 && n_kv <= kMaxKvHeads && n_pages >= 1 &&
           (unsigned long long)n_pages * page < 0xFFFFFFFFull;
}
inline size_t kv4_layer_bytes(unsigned n_pages, unsigned page, unsigned n_kv, unsigned dim) {
    return size_t(n_pages) * n_kv * (page / kTileTokens) * kv4_tile_bytes(dim);
}
inline bool attn_shape_ok(unsigned n_head, unsigned n_kv, unsigned n_req, unsigned n_rows, unsigned max_q, unsigned max_kv) {
    return n_head >= 1 && n_head <= 1024 && n_head % n_kv == 0 && n_req >= 1 && n_req <= kMaxAttnReq && n_rows <= (1u << 24) && max_q >= 1 &&
           max_q <= (1u << 24) && max_kv >= 1 && max_kv <= (1u << 28);
}
inline bool select_shape_ok(unsigned n_req, unsigned beams, unsigned vocab, unsigned n_out) {
    return n_req >= 1 && n_req <= kMaxSelectReq && beams >= 1 && beams <= kMaxBeams && vocab >= 1 && vocab <= kMaxVocab && n_out >= 1 &&
           n_out <= kMaxBeamOut;
}

}  // namespace b200q
