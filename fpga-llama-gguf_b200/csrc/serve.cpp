// Entry points of the operators that serve several sequences from a paged 4-bit KV cache (include/b200q.h). They hold no
// context: the caller names the device, the stream and every buffer. Each call checks its arguments on the host before
// it launches: sizes, alignments, that every pointer is device (or managed) memory of the device with room for what the
// kernels touch, that outputs lie apart from inputs, and that the stream belongs to the device. What only the device
// knows (lengths, pages, slots, parents) the kernels check themselves: they leave out what does not fit and set a bit
// in the caller's status word. Nothing is allocated, nothing waits, and a call can be captured into a graph.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/b200q.h"
#include "serve.h"

using namespace b200q;

namespace {

struct Extent {
    const char *name;
    const void *p;
    size_t bytes;
    bool written;
};

class Call {
  public:
    Call(const char *name, int device, void *stream, char *msg, unsigned len)
        : name_(name), device_(device), stream_(static_cast<cudaStream_t>(stream)), msg_(msg), len_(len) {
        if (msg_ && len_) msg_[0] = '\0';
    }
    ~Call() {
        if (prev_ >= 0 && prev_ != device_) cudaSetDevice(prev_);
    }
    Call(const Call &) = delete;
    Call &operator=(const Call &) = delete;

    bool ok() const { return rc_ == B200Q_OK; }
    int rc() const { return rc_; }
    cudaStream_t stream() const { return stream_; }

    __attribute__((format(printf, 2, 3))) void refuse(const char *fmt, ...) {
        if (!ok()) return;
        rc_ = B200Q_ERR_ARG;
        char why[256];
        va_list ap;
        va_start(ap, fmt);
        std::vsnprintf(why, sizeof(why), fmt, ap);
        va_end(ap);
        if (msg_ && len_) std::snprintf(msg_, len_, "%s: %s", name_, why);
    }
    void need(bool good, const char *what) {
        if (!good) refuse("%s", what);
    }

    // the device becomes current (until the call returns), and the stream is one of its streams
    void enter() {
        if (!ok()) return;
        cudaError_t e = cudaGetDevice(&prev_);
        if (e == cudaSuccess && prev_ != device_) e = cudaSetDevice(device_);
        if (e != cudaSuccess) {
            cudaGetLastError();
            prev_ = -1;
            return cuda(e, "device");
        }
        int d = device_;
        if (!stream_ || stream_ == cudaStreamLegacy || stream_ == cudaStreamPerThread) return;
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        // a capturing stream is not asked for its device (the question would end the capture; a launch from the wrong
        // device fails by itself)
        if (cudaStreamIsCapturing(stream_, &cap) != cudaSuccess ||
            (cap == cudaStreamCaptureStatusNone && cudaStreamGetDevice(stream_, &d) != cudaSuccess)) {
            cudaGetLastError();
            refuse("stream is not a valid CUDA stream");
        } else if (d != device_) {
            refuse("stream belongs to device %d, not %d", d, device_);
        }
    }

    // p .. p + bytes is memory of the device, aligned, inside one allocation. bytes 0: p is not used.
    void memory(const char *name, const void *p, size_t bytes, unsigned align, bool written = false) {
        if (!ok() || bytes == 0) return;
        if (!p) return refuse("%s is null", name);
        if (reinterpret_cast<uintptr_t>(p) % align) return refuse("%s is not %u-byte aligned", name, align);
        if (n_ < kMaxExtents) ext_[n_++] = Extent{name, p, bytes, written};
    }

    // the pointers are looked up, and what is written meets nothing else
    void check_memory() {
        if (!ok()) return;
        static AttrFn attr = entry();
        CUdeviceptr start_of[kMaxExtents];
        size_t size_of[kMaxExtents];
        unsigned n_known = 0;
        for (unsigned i = 0; i < n_ && ok(); ++i) {
            const Extent &x = ext_[i];
            const CUdeviceptr p = reinterpret_cast<CUdeviceptr>(x.p);
            bool known = false;  // inside an allocation that an earlier pointer of this call lies in
            for (unsigned j = 0; j < n_known && !known; ++j)
                known = p >= start_of[j] && p - start_of[j] <= size_of[j] && x.bytes <= size_of[j] - (p - start_of[j]);
            if (known) continue;
            int type = 0, ordinal = -1, managed = 0;
            CUdeviceptr start = 0;
            size_t size = 0;
            CUpointer_attribute what[5] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                           CU_POINTER_ATTRIBUTE_IS_MANAGED, CU_POINTER_ATTRIBUTE_RANGE_START_ADDR,
                                           CU_POINTER_ATTRIBUTE_RANGE_SIZE};
            void *to[5] = {&type, &ordinal, &managed, &start, &size};
            if (!attr || attr(5, what, to, p) != CUDA_SUCCESS || (type != CU_MEMORYTYPE_DEVICE && !managed))
                refuse("%s is not device memory (it must be device memory of device %d)", x.name, device_);
            else if (!managed && ordinal != device_)
                refuse("%s is device memory of device %d, not of device %d", x.name, ordinal, device_);
            else if (p < start || p - start > size || x.bytes > size - (p - start))
                refuse("%s + %zu bytes runs past the end of its allocation", x.name, x.bytes);
            start_of[n_known] = start;
            size_of[n_known++] = size;
        }
        for (unsigned i = 0; i < n_ && ok(); ++i)
            for (unsigned j = 0; j < n_; ++j) {
                const Extent &w = ext_[i], &x = ext_[j];
                const uintptr_t a = reinterpret_cast<uintptr_t>(w.p), b = reinterpret_cast<uintptr_t>(x.p);
                if (w.written && i != j && a < b + x.bytes && b < a + w.bytes) refuse("%s overlaps %s", w.name, x.name);
            }
    }

    void cuda(cudaError_t e, const char *what) {
        if (e == cudaSuccess || !ok()) return;
        cudaGetLastError();
        rc_ = B200Q_ERR_CUDA;
        if (msg_ && len_) std::snprintf(msg_, len_, "%s: %s: %s", name_, what, cudaGetErrorString(e));
    }

    unsigned sms() {
        static std::mutex mu;
        static int known[64] = {};
        if (device_ < 0 || device_ >= 64) return 148;
        std::lock_guard<std::mutex> lock(mu);
        if (!known[device_] && cudaDeviceGetAttribute(&known[device_], cudaDevAttrMultiProcessorCount, device_) != cudaSuccess) {
            cudaGetLastError();
            return 148;
        }
        return unsigned(known[device_]);
    }

  private:
    typedef CUresult (*AttrFn)(unsigned, CUpointer_attribute *, void **, CUdeviceptr);
    static AttrFn entry() {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<AttrFn>(f);
    }
    static constexpr unsigned kMaxExtents = 16;
    const char *name_;
    int device_, prev_ = -1, rc_ = B200Q_OK;
    cudaStream_t stream_;
    char *msg_;
    unsigned len_, n_ = 0;
    Extent ext_[kMaxExtents];
};

// the pool's shape; its bytes over the layers used
size_t check_pool(Call &c, const b200q_kv4_pool *p, bool layers) {
    c.need(p != nullptr, "pool is null");
    if (!c.ok()) return 0;
    c.need(p->head_dim >= 32 && p->head_dim <= kMaxKv4Dim && p->head_dim % 32 == 0, "head_dim is not a multiple of 32 up to 256");
    c.need(p->page_tokens >= kTileTokens && p->page_tokens <= 4096 && p->page_tokens % kTileTokens == 0,
           "page_tokens is not a multiple of 16 up to 4096");
    c.need(p->n_kv_head >= 1 && p->n_kv_head <= 256, "n_kv_head is not 1 to 256");
    c.need(p->n_pages >= 1 && (unsigned long long)p->n_pages * p->page_tokens < 0xFFFFFFFFull, "n_pages x page_tokens is not 1 to 2^32 - 2 tokens");
    if (!c.ok()) return 0;
    const size_t layer = size_t(p->n_pages) * p->n_kv_head * (p->page_tokens / kTileTokens) * kv4_tile_bytes(p->head_dim);
    if (!layers) return layer;
    c.need(p->n_layers >= 1 && p->n_layers <= 65534, "n_layers is not 1 to 65534");
    c.need(p->n_layers <= 1 || (p->layer_bytes >= layer && p->layer_bytes % 16 == 0 && p->layer_bytes <= (size_t(1) << 46)),
           "layer_bytes is smaller than a layer or not a multiple of 16");
    return c.ok() ? size_t(p->n_layers - 1) * p->layer_bytes + layer : 0;
}

Kv4View view_of(const b200q_kv4_pool *p) {
    Kv4View v;
    v.base = static_cast<uint8_t *>(p->base);
    v.n_pages = p->n_pages;
    v.page = p->page_tokens;
    v.n_kv = p->n_kv_head;
    v.dim = p->head_dim;
    return v;
}

size_t rows_extent(size_t rows, size_t stride, size_t width) { return rows ? ((rows - 1) * stride + width) * 4 : 0; }

constexpr size_t kMaxStride = size_t(1) << 32, kMaxSpan = size_t(1) << 60;  // floats

int rows_call(const char *name, bool store, int device, const b200q_kv4_pool *pool, float *k, float *v, const uint32_t *slots, unsigned n,
              size_t k_stride, size_t v_stride, uint32_t *status, void *stream, char *err, unsigned err_len) {
    Call c(name, device, stream, err, err_len);
    const size_t bytes = check_pool(c, pool, false);
    if (!c.ok()) return c.rc();
    const size_t width = size_t(pool->n_kv_head) * pool->head_dim;
    if (k_stride == 0) k_stride = width;
    if (v_stride == 0) v_stride = width;
    c.need(k_stride >= width && v_stride >= width && k_stride <= kMaxStride && v_stride <= kMaxStride, "a row stride is smaller than n_kv_head x head_dim");
    // (n and the strides are below 2^32 and 2^32 + 1: their products fit 64 bits, and so do the rows' bytes)
    c.need(!c.ok() || (n * k_stride <= kMaxSpan && n * v_stride <= kMaxSpan), "rows and their stride pass 2^60 floats");
    c.enter();
    if (!c.ok() || n == 0) return c.rc();
    c.memory("pool", pool->base, bytes, 16, store);
    c.memory("k", k, rows_extent(n, k_stride, width), 4);
    c.memory("v", v, rows_extent(n, v_stride, width), 4);
    c.memory("slots", slots, size_t(n) * 4, 4);
    c.memory("status", status, status ? 4 : 0, 4, true);
    c.check_memory();
    if (!store && c.ok()) {  // k and v are written: rows of one buffer side by side are fine, anything else apart
        const uintptr_t kb = reinterpret_cast<uintptr_t>(k), vb = reinterpret_cast<uintptr_t>(v), pb = reinterpret_cast<uintptr_t>(pool->base),
                        sb = reinterpret_cast<uintptr_t>(slots);
        const size_t kn = rows_extent(n, k_stride, width), vn = rows_extent(n, v_stride, width);
        const auto meet = [](uintptr_t a, size_t an, uintptr_t b, size_t bn) { return a < b + bn && b < a + an; };
        c.need(!meet(kb, kn, pb, bytes) && !meet(vb, vn, pb, bytes), "k or v overlaps the pool");
        c.need(!meet(kb, kn, sb, size_t(n) * 4) && !meet(vb, vn, sb, size_t(n) * 4), "k or v overlaps slots");
        const uintptr_t gap = kb < vb ? vb - kb : kb - vb;
        const bool beside = k_stride == v_stride && gap % (k_stride * 4) >= width * 4 && gap % (k_stride * 4) + width * 4 <= k_stride * 4;
        c.need(!meet(kb, kn, vb, vn) || beside, "k overlaps v");
    }
    if (!c.ok()) return c.rc();
    Kv4RowsArgs a;
    a.c = view_of(pool);
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.slots = slots;
    a.n = n;
    a.status = status;
    c.cuda(store ? launch_kv4_store(a, c.stream()) : launch_kv4_load(a, c.stream()), "launch");
    return c.rc();
}

void check_attn(Call &c, const b200q_kv4_pool *pool, unsigned n_rows, unsigned n_head, unsigned n_req, unsigned max_q, unsigned max_kv) {
    c.need(n_head >= 1 && n_head <= 1024 && n_head % pool->n_kv_head == 0, "n_head is not a multiple of n_kv_head up to 1024");
    c.need(n_req >= 1 && n_req <= kMaxAttnReq, "n_req is not 1 to 4096");
    c.need(n_rows <= (1u << 24), "n_rows is over 2^24");
    c.need(max_q >= 1 && max_q <= (1u << 24), "max_q is not 1 to 2^24");
    c.need(max_kv >= 1 && max_kv <= (1u << 28), "max_kv is not 1 to 2^28");
}

Kv4AttnArgs attn_shape(const b200q_kv4_pool *pool, unsigned n_rows, unsigned n_head, unsigned n_req, unsigned max_q, unsigned max_kv) {
    Kv4AttnArgs a;
    a.c = view_of(pool);
    a.n_rows = n_rows;
    a.n_head = n_head;
    a.n_req = n_req;
    a.max_q = max_q;
    a.max_kv = max_kv;
    return a;
}

}  // namespace

extern "C" {

B200Q_API size_t b200q_kv4_page_bytes(unsigned page_tokens, unsigned n_kv_head, unsigned head_dim) {
    if (page_tokens == 0 || page_tokens % kTileTokens || page_tokens > 4096 || n_kv_head == 0 || n_kv_head > 256 || head_dim == 0 ||
        head_dim % 32 || head_dim > kMaxKv4Dim)
        return 0;
    return size_t(n_kv_head) * (page_tokens / kTileTokens) * kv4_tile_bytes(head_dim);
}

B200Q_API int b200q_block_map(int device, unsigned n_req, const uint32_t *past, const uint32_t *fresh, uint32_t *table, unsigned table_stride,
                              unsigned page_tokens, const uint32_t *free_pages, unsigned n_free, const uint32_t *cursor_in,
                              uint32_t *cursor_out, uint32_t *kv_len, uint32_t *q_start, uint32_t *slots, uint32_t *positions,
                              unsigned n_rows, uint32_t *status, void *stream, char *err, unsigned err_len) {
    Call c("block_map", device, stream, err, err_len);
    c.need(n_req >= 1 && n_req <= kMaxMapReq, "n_req is not 1 to 65535");
    c.need(table_stride >= 1, "table_stride is 0");
    c.need(page_tokens >= kTileTokens && page_tokens <= kMaxPage && page_tokens % kTileTokens == 0, "page_tokens is not a multiple of 16 up to 4096");
    c.need((unsigned long long)table_stride * page_tokens < 0xFFFFFFFFull, "table_stride x page_tokens is over 2^32 - 2 tokens");
    c.need(n_rows < 0x80000000u, "n_rows is over 2^31 - 1");
    c.enter();
    c.memory("past", past, size_t(n_req) * 4, 4);
    c.memory("fresh", fresh, size_t(n_req) * 4, 4);
    c.memory("table", table, size_t(n_req) * table_stride * 4, 4, true);
    c.memory("free_pages", free_pages, size_t(n_free) * 4, 4);
    if (cursor_in != cursor_out) c.memory("cursor_in", cursor_in, 4, 4);
    c.memory("cursor_out", cursor_out, 4, 4, true);
    c.memory("kv_len", kv_len, size_t(n_req) * 4, 4, true);
    c.memory("q_start", q_start, (size_t(n_req) + 1) * 4, 4, true);
    c.memory("slots", slots, size_t(n_rows) * 4, 4, true);
    c.memory("positions", positions, size_t(n_rows) * 4, 4, true);
    c.memory("status", status, status ? 4 : 0, 4, true);
    c.check_memory();
    if (!c.ok()) return c.rc();
    BlockMapArgs a;
    a.n_req = n_req;
    a.page = page_tokens;
    a.stride = table_stride;
    a.n_free = n_free;
    a.n_rows = n_rows;
    a.past = past;
    a.fresh = fresh;
    a.free_pages = free_pages;
    a.cursor_in = cursor_in;
    a.table = table;
    a.cursor_out = cursor_out;
    a.kv_len = kv_len;
    a.q_start = q_start;
    a.slots = slots;
    a.positions = positions;
    a.status = status;
    c.cuda(launch_block_map(a, c.stream()), "launch");
    return c.rc();
}

B200Q_API int b200q_kv4_store(int device, const b200q_kv4_pool *pool, const float *k, const float *v, const uint32_t *slots, unsigned n,
                              size_t k_stride, size_t v_stride, uint32_t *status, void *stream, char *err, unsigned err_len) {
    return rows_call("kv4_store", true, device, pool, const_cast<float *>(k), const_cast<float *>(v), slots, n, k_stride, v_stride, status,
                     stream, err, err_len);
}

B200Q_API int b200q_kv4_load(int device, const b200q_kv4_pool *pool, const uint32_t *slots, unsigned n, float *k, float *v, size_t k_stride,
                             size_t v_stride, uint32_t *status, void *stream, char *err, unsigned err_len) {
    return rows_call("kv4_load", false, device, pool, k, v, slots, n, k_stride, v_stride, status, stream, err, err_len);
}

B200Q_API size_t b200q_kv4_attn_workspace(int device, const b200q_kv4_pool *pool, unsigned n_rows, unsigned n_head, unsigned n_req,
                                          unsigned max_q, unsigned max_kv) {
    Call c("kv4_attn_workspace", device, nullptr, nullptr, 0);
    check_pool(c, pool, false);
    if (c.ok()) check_attn(c, pool, n_rows, n_head, n_req, max_q, max_kv);
    return c.ok() ? kv4_attn_room(attn_shape(pool, n_rows, n_head, n_req, max_q, max_kv), c.sms()) : 0;
}

B200Q_API int b200q_kv4_attn(int device, const b200q_kv4_pool *pool, const float *q, float *y, unsigned n_rows, unsigned n_head,
                             const uint32_t *table, unsigned table_stride, const uint32_t *q_start, const uint32_t *kv_len, unsigned n_req,
                             unsigned max_q, unsigned max_kv, float scale, void *workspace, size_t workspace_bytes, size_t q_stride,
                             size_t q_head_stride, size_t y_stride, unsigned window, uint32_t *status, void *stream, char *err,
                             unsigned err_len) {
    Call c("kv4_attn", device, stream, err, err_len);
    const size_t bytes = check_pool(c, pool, false);
    if (!c.ok()) return c.rc();
    check_attn(c, pool, n_rows, n_head, n_req, max_q, max_kv);
    if (!c.ok()) return c.rc();
    const size_t dim = pool->head_dim, width = n_head * dim;
    if (q_head_stride == 0) q_head_stride = dim;
    c.need(q_head_stride <= kMaxStride, "a stride of q or y is over 2^32 floats");  // (before it is multiplied)
    if (!c.ok()) return c.rc();
    const size_t q_width = (n_head - 1) * q_head_stride + dim;
    if (q_stride == 0) q_stride = n_head * q_head_stride;
    if (y_stride == 0) y_stride = width;
    c.need(q_stride <= kMaxStride && y_stride <= kMaxStride, "a stride of q or y is over 2^32 floats");
    c.need(q_head_stride >= dim && q_stride >= q_width && y_stride >= width, "a stride of q or y is smaller than what it steps over");
    c.need(table_stride >= 1 && (unsigned long long)table_stride * pool->page_tokens >= max_kv, "max_kv does not fit table_stride pages");
    c.need(std::isfinite(scale), "scale is not finite");
    c.enter();
    if (!c.ok() || n_rows == 0) return c.rc();
    Kv4AttnArgs a = attn_shape(pool, n_rows, n_head, n_req, max_q, max_kv);
    const size_t room = kv4_attn_room(a, c.sms());
    c.need(room != 0, "n_rows, n_req and max_kv allow for more than 2^31 tiles of work");
    if (workspace_bytes < room) c.refuse("the workspace holds %zu bytes, %zu are needed", workspace_bytes, room);
    c.memory("pool", pool->base, bytes, 16);
    c.memory("q", q, rows_extent(n_rows, q_stride, q_width), 4);
    c.memory("y", y, rows_extent(n_rows, y_stride, width), 4, true);
    c.memory("table", table, size_t(n_req) * table_stride * 4, 4);
    c.memory("q_start", q_start, (size_t(n_req) + 1) * 4, 4);
    c.memory("kv_len", kv_len, size_t(n_req) * 4, 4);
    c.memory("workspace", workspace, room, 16, true);
    c.memory("status", status, status ? 4 : 0, 4, true);
    c.check_memory();
    if (!c.ok()) return c.rc();
    a.q = q;
    a.y = y;
    a.q_stride = q_stride;
    a.q_head_stride = q_head_stride;
    a.y_stride = y_stride;
    a.window = window;
    a.stride = table_stride;
    a.table = table;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.scale = scale;
    a.room = static_cast<uint8_t *>(workspace);
    a.status = status;
    c.cuda(launch_kv4_attn(a, c.sms(), c.stream()), "launch");
    return c.rc();
}

static void check_select(Call &c, unsigned n_req, unsigned beams, unsigned vocab, unsigned n_out) {
    c.need(n_req >= 1 && n_req <= kMaxSelectReq, "n_req is not 1 to 2047");
    c.need(beams >= 1 && beams <= kMaxBeams, "beams is not 1 to 32");
    c.need(vocab >= 1 && vocab <= kMaxVocab, "vocab is not 1 to 2^20");
    c.need(n_out >= 1 && n_out <= kMaxBeamOut, "n_out is not 1 to 64");
}

B200Q_API size_t b200q_beam_select_workspace(int device, unsigned n_req, unsigned beams, unsigned vocab, unsigned n_out) {
    Call c("beam_select_workspace", device, nullptr, nullptr, 0);
    check_select(c, n_req, beams, vocab, n_out);
    BeamSelectArgs a;
    a.n_req = n_req;
    a.beams = beams;
    a.vocab = vocab;
    a.n_out = n_out;
    return c.ok() ? beam_select_room(a) : 0;
}

B200Q_API int b200q_beam_select(int device, const float *logits, unsigned vocab, const float *scores, unsigned n_req, unsigned beams,
                                unsigned n_out, float *out_scores, uint32_t *out_parent, uint32_t *out_token, void *workspace,
                                size_t workspace_bytes, size_t logits_stride, void *stream, char *err, unsigned err_len) {
    Call c("beam_select", device, stream, err, err_len);
    check_select(c, n_req, beams, vocab, n_out);
    if (logits_stride == 0) logits_stride = vocab;
    c.need(logits_stride >= vocab && logits_stride <= kMaxStride, "logits_stride is smaller than vocab");
    c.enter();
    if (!c.ok()) return c.rc();
    BeamSelectArgs a;
    a.logits = logits;
    a.scores = scores;
    a.stride = logits_stride;
    a.n_req = n_req;
    a.beams = beams;
    a.vocab = vocab;
    a.n_out = n_out;
    a.out = out_scores;
    a.parent = out_parent;
    a.token = out_token;
    a.room = static_cast<uint8_t *>(workspace);
    const size_t room = beam_select_room(a), rows = size_t(n_req) * beams, outs = size_t(n_req) * n_out;
    if (workspace_bytes < room) c.refuse("the workspace holds %zu bytes, %zu are needed", workspace_bytes, room);
    c.memory("logits", logits, rows_extent(rows, logits_stride, vocab), 4);
    c.memory("scores", scores, rows * 4, 4);
    c.memory("out_scores", out_scores, outs * 4, 4, true);
    c.memory("out_parent", out_parent, outs * 4, 4, true);
    c.memory("out_token", out_token, outs * 4, 4, true);
    c.memory("workspace", workspace, room, 16, true);
    c.check_memory();
    if (c.ok()) c.cuda(launch_beam_select(a, c.sms(), c.stream()), "launch");
    return c.rc();
}

B200Q_API int b200q_beam_reorder(int device, const void *src, void *dst, const uint32_t *parent, unsigned n_req, unsigned beams,
                                 size_t row_bytes, unsigned n_layers, size_t src_layer_bytes, size_t dst_layer_bytes, uint32_t *status,
                                 void *stream, char *err, unsigned err_len) {
    Call c("beam_reorder", device, stream, err, err_len);
    c.need(n_req >= 1 && n_req <= kMaxMapReq, "n_req is not 1 to 65535");
    c.need(beams >= 1 && beams <= kMaxBeams, "beams is not 1 to 32");
    c.need(row_bytes >= 1 && row_bytes <= (size_t(1) << 40), "row_bytes is not 1 to 2^40");
    c.need(n_layers >= 1 && n_layers <= 65535, "n_layers is not 1 to 65535");
    if (!c.ok()) return c.rc();
    const size_t layer = size_t(n_req) * beams * row_bytes;
    if (src_layer_bytes == 0) src_layer_bytes = layer;
    if (dst_layer_bytes == 0) dst_layer_bytes = layer;
    c.need(layer <= (size_t(1) << 46) && src_layer_bytes >= layer && dst_layer_bytes >= layer && src_layer_bytes <= (size_t(1) << 46) &&
               dst_layer_bytes <= (size_t(1) << 46),
           "a layer's bytes are fewer than its rows hold");
    c.need(src != dst || src_layer_bytes == dst_layer_bytes, "in place, both layer strides are the same");
    c.enter();
    if (!c.ok()) return c.rc();
    if (src != dst) c.memory("src", src, (n_layers - 1) * src_layer_bytes + layer, 1);
    c.memory("dst", dst, (n_layers - 1) * dst_layer_bytes + layer, 1, true);
    c.memory("parent", parent, size_t(n_req) * beams * 4, 4);
    c.memory("status", status, status ? 4 : 0, 4, true);
    c.check_memory();
    if (!c.ok()) return c.rc();
    BeamReorderArgs a;
    a.src = static_cast<const uint8_t *>(src);
    a.dst = static_cast<uint8_t *>(dst);
    a.parent = parent;
    a.n_req = n_req;
    a.beams = beams;
    a.layers = n_layers;
    a.row_bytes = row_bytes;
    a.src_layer = src_layer_bytes;
    a.dst_layer = dst_layer_bytes;
    a.status = status;
    c.cuda(launch_beam_reorder(a, c.stream()), "launch");
    return c.rc();
}

B200Q_API int b200q_kv4_reorder(int device, const b200q_kv4_pool *pool, uint32_t *table, unsigned table_stride, const uint32_t *kv_len,
                                const uint32_t *parent, unsigned n_req, unsigned beams, uint32_t *status, void *stream, char *err,
                                unsigned err_len) {
    Call c("kv4_reorder", device, stream, err, err_len);
    const size_t bytes = check_pool(c, pool, true);
    c.need(table_stride >= 1, "table_stride is 0");
    c.need(n_req >= 1 && n_req <= kMaxMapReq, "n_req is not 1 to 65535");
    c.need(beams >= 1 && beams <= kMaxBeams, "beams is not 1 to 32");
    c.enter();
    if (!c.ok()) return c.rc();
    const size_t rows = size_t(n_req) * beams;
    c.memory("pool", pool->base, bytes, 16, true);
    c.memory("table", table, rows * table_stride * 4, 4, true);
    c.memory("kv_len", kv_len, rows * 4, 4);
    c.memory("parent", parent, rows * 4, 4);
    c.memory("status", status, status ? 4 : 0, 4, true);
    c.check_memory();
    if (!c.ok()) return c.rc();
    Kv4ReorderArgs a;
    a.c = view_of(pool);
    a.layers = pool->n_layers;
    a.stride = table_stride;
    a.n_req = n_req;
    a.beams = beams;
    a.layer_bytes = pool->layer_bytes;
    a.table = table;
    a.kv_len = kv_len;
    a.parent = parent;
    a.status = status;
    c.cuda(launch_kv4_reorder(a, c.stream()), "launch");
    return c.rc();
}

}  // extern "C"
