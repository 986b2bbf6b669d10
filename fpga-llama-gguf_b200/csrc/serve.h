// The operators that serve several sequences from a paged 4-bit KV cache (include/b200q.h, "several sequences"): kernel
// arguments and launchers. The kernels take plain device pointers, so the context-free entry points (serve.cpp) and the
// command lists (api.cpp) run the same code.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "serve_limits.h"

namespace b200q {

// status bits (include/b200q.h, B200Q_SERVE_*)
constexpr unsigned kServeRequest = 1, kServePage = 2, kServeSlot = 4, kServeShort = 8, kServeParent = 16, kServeWait = 32;
constexpr unsigned kNoSlot = 0xFFFFFFFFu;  // a slot, page, parent or token that names nothing

// The cache of one layer: page p, head h, tile t at base + ((p * n_kv + h) * (page / 16) + t) * 18 dim.
struct Kv4View {
    uint8_t *base = nullptr;
    unsigned n_pages = 0, page = 0, n_kv = 0, dim = 0;
};

struct BlockMapArgs {
    unsigned n_req = 0, page = 0, stride = 0, n_free = 0, n_rows = 0;
    const uint32_t *past = nullptr, *fresh = nullptr, *free_pages = nullptr, *cursor_in = nullptr;
    uint32_t *table = nullptr, *cursor_out = nullptr, *kv_len = nullptr, *q_start = nullptr, *slots = nullptr, *positions = nullptr;
    uint32_t *status = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

struct Kv4RowsArgs {  // kv4_store (k, v read) / kv4_load (k, v written)
    Kv4View c;
    float *k = nullptr, *v = nullptr;
    size_t k_stride = 0, v_stride = 0;
    const uint32_t *slots = nullptr;
    unsigned n = 0;
    uint32_t *status = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

struct Kv4AttnArgs {
    Kv4View c;
    const float *q = nullptr;
    float *y = nullptr;
    size_t q_stride = 0, q_head_stride = 0, y_stride = 0;
    unsigned n_rows = 0, n_head = 0, n_req = 0, max_q = 0, max_kv = 0, window = 0, stride = 0;
    const uint32_t *table = nullptr, *q_start = nullptr, *kv_len = nullptr;
    float scale = 0.0f;
    uint8_t *room = nullptr;  // workspace of kv4_attn_room bytes
    uint32_t *status = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

struct BeamSelectArgs {
    const float *logits = nullptr, *scores = nullptr;
    size_t stride = 0;  // floats between the rows of logits
    unsigned n_req = 0, beams = 0, vocab = 0, n_out = 0;
    float *out = nullptr;
    uint32_t *parent = nullptr, *token = nullptr;
    uint8_t *room = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

struct BeamReorderArgs {
    const uint8_t *src = nullptr;
    uint8_t *dst = nullptr;
    const uint32_t *parent = nullptr;
    unsigned n_req = 0, beams = 0, layers = 0;
    size_t row_bytes = 0, src_layer = 0, dst_layer = 0;
    uint32_t *status = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

struct Kv4ReorderArgs {
    Kv4View c;
    unsigned layers = 0, stride = 0, n_req = 0, beams = 0;
    size_t layer_bytes = 0;
    uint32_t *table = nullptr;
    const uint32_t *kv_len = nullptr, *parent = nullptr;
    uint32_t *status = nullptr;
    bool pdl = true;  // programmatic dependent launch
};

cudaError_t launch_block_map(const BlockMapArgs &a, cudaStream_t st);
unsigned block_map_launches(const BlockMapArgs &a);
cudaError_t launch_kv4_store(const Kv4RowsArgs &a, cudaStream_t st);
cudaError_t launch_kv4_load(const Kv4RowsArgs &a, cudaStream_t st);
size_t kv4_attn_room(const Kv4AttnArgs &a, unsigned sms);  // 0: more work than one launch takes
cudaError_t launch_kv4_attn(const Kv4AttnArgs &a, unsigned sms, cudaStream_t st);
// requests of least_rows (token, head of the group) rows or more, on tcgen05; the others are left out
cudaError_t launch_kv4_prompt(const Kv4AttnArgs &a, unsigned least_rows, cudaStream_t st);
size_t beam_select_room(const BeamSelectArgs &a);
cudaError_t launch_beam_select(const BeamSelectArgs &a, unsigned sms, cudaStream_t st);
cudaError_t launch_beam_reorder(const BeamReorderArgs &a, cudaStream_t st);
cudaError_t launch_kv4_reorder(const Kv4ReorderArgs &a, cudaStream_t st);
// kernels that launch_kv4_attn starts (for launch counts; block_map_launches above likewise)
unsigned kv4_attn_launches(const Kv4AttnArgs &a, unsigned sms);

// A launch that may start while the previous kernel drains: every kernel here waits (griddepcontrol.wait) before it
// touches global memory.
template <typename... P, typename... A>
inline cudaError_t launch_pdl(bool pdl, void (*k)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

}  // namespace b200q
