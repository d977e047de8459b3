// pages.cpp -- the C ABI of the paged cache (include/bmo_attn.h): allocation,
// argument checking, error reporting.  Conventions as in api.cpp: nothing
// throws across the ABI, int entry points return a status and record a
// message, a failed create returns NULL and says why on stderr.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <exception>
#include <mutex>
#include <string>

#include "../../include/bmo_attn.h"
#include "pages.hpp"

static_assert(BMO_ATTN_F32 == bmo::kTypeF32 && BMO_ATTN_F16 == bmo::kTypeF16 && BMO_ATTN_BF16 == bmo::kTypeBF16 &&
                  BMO_ATTN_Q4_0 == bmo::kTypeQ4_0,
              "the header's element types");

struct bmo_kv_pages {
    bmo::PagesGeom g{};
    int device = 0;
    uint8_t *mem = nullptr;
    std::mutex mu;  // guards last_error
    std::string last_error;
};

namespace {

thread_local std::string t_create_error;

constexpr float kLog2e = 1.4426950408889634f;
// Positions a table row can hold: 64 rows' steps of 32 then sum up in 32 bits.
constexpr int64_t kMaxRoom = int64_t(1) << 30;

// What an entry point does: collects its name's errors and keeps the handle's
// device current.
struct Call {
    bmo_kv_pages_t *h;
    const char *fn;
    int prev = -1;
    bool switched = false;
    Call(bmo_kv_pages_t *h_, const char *fn_) : h(h_), fn(fn_) {}
    ~Call() {
        if (switched) (void) hipSetDevice(prev);
    }
    int fail(int code, const std::string &why) {
        std::lock_guard<std::mutex> lk(h->mu);
        h->last_error = std::string(fn) + ": " + why;
        return code;
    }
    int null() { return fail(BMO_ATTN_ERR_NULL, "null pointer argument"); }
    int arg(const std::string &why) { return fail(BMO_ATTN_ERR_ARG, why); }
    // Ends a call: the launch's own status.
    int done(hipError_t e) {
        if (e != hipSuccess) return fail(BMO_ATTN_ERR_HIP, hipGetErrorString(e));
        std::lock_guard<std::mutex> lk(h->mu);
        h->last_error.clear();
        return BMO_ATTN_OK;
    }
    void enter() {
        if (hipGetDevice(&prev) == hipSuccess && prev != h->device) switched = hipSetDevice(h->device) == hipSuccess;
    }
};

// Runs f(call) behind the NULL check and the exception barrier.
template <class F>
int guarded(bmo_kv_pages_t *h, const char *fn, F f) {
    if (!h) return BMO_ATTN_ERR_NULL;
    try {
        Call c(h, fn);
        return f(c);
    } catch (...) {
        return BMO_ATTN_ERR_INTERNAL;
    }
}

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows [heads][dim] of 32- or 16-bit elements, stride elements apart: 0 for
// an argument that is not checked here, else why it is refused.
const char *row_fault(const void *p, int64_t &stride, int64_t dense, int type) {
    if (stride == 0) stride = dense;
    if (stride < dense) return "a stride is shorter than its row";
    if (stride > (int64_t(1) << 40)) return "a stride is too long";
    if (!aligned(p, 16) || stride * bmo::type_bytes(type) % 16 != 0) return "rows must be aligned to 16 bytes";
    return nullptr;
}

int check_layer(Call &c, int layer) {
    return layer < 0 || layer >= c.h->g.n_layers ? c.arg("layer out of range") : BMO_ATTN_OK;
}

int check_heads(Call &c, int n_heads) {
    return n_heads <= 0 || n_heads % c.h->g.n_kv != 0 || n_heads > (1 << 20)
               ? c.arg("n_heads must be a positive multiple of n_kv_heads")
               : BMO_ATTN_OK;
}

int check_table(Call &c, int n_batch, int max_pages) {
    if (n_batch <= 0) return c.arg("n_batch must be positive");
    if (max_pages <= 0 || (int64_t) max_pages << c.h->g.page_shift > kMaxRoom)
        return c.arg("max_pages must be positive, and max_pages * page_size at most 2^30");
    return BMO_ATTN_OK;
}

int slots_call(bmo_kv_pages_t *h, const char *fn, bool append, int layer, int n_tok, const int *slots, int type, void *k,
               void *v, int64_t stride, void *stream) {
    return guarded(h, fn, [&](Call &c) {
        // (an empty tensor has no address)
        if (n_tok != 0 && (!slots || !k || !v)) return c.null();
        if (int rc = check_layer(c, layer)) return rc;
        if (n_tok < 0) return c.arg("n_tok must not be negative");
        if (type < bmo::kTypeF32 || type > bmo::kTypeQ4_0) return c.arg("unknown element type");
        const bmo::PagesGeom &g = c.h->g;
        if (type == bmo::kTypeQ4_0) {
            if (stride != 0) return c.arg("blocks have no stride");
            if (!aligned(k, 2) || !aligned(v, 2)) return c.arg("blocks must be aligned to 2 bytes");
        } else {
            const int64_t given = stride;
            if (const char *why = row_fault(k, stride, (int64_t) g.n_kv * g.dim, type)) return c.arg(why);
            stride = given;
            if (const char *why = row_fault(v, stride, (int64_t) g.n_kv * g.dim, type)) return c.arg(why);
        }
        // (four lanes a block: the grid's threads stay below 2^32)
        if ((int64_t) n_tok * g.n_kv * (g.dim / 32) > (1 << 29)) return c.arg("n_tok too large (2^29 blocks)");
        if (n_tok == 0) return c.done(hipSuccess);
        c.enter();
        bmo::SlotsParams p{};
        p.base = c.h->mem + layer * g.layer_bytes;
        p.g = g;
        p.slots = slots;
        p.n_tok = n_tok;
        p.type = type;
        p.k = k;
        p.v = v;
        p.stride = stride;
        return c.done(append ? bmo::launch_pages_append(p, (hipStream_t) stream)
                             : bmo::launch_pages_gather(p, (hipStream_t) stream));
    });
}

// What a plan was asked for and answered, of the calls that are told.
struct Granted {
    bool told;
    const int *n_new, *status;
};

int decode_call(bmo_kv_pages_t *h, const char *fn, bool append, Granted granted, int layer, int n_batch, const int *lens,
                const int *table, int max_pages, int n_heads, int type, const void *q, int64_t q_stride, const void *k_new,
                const void *v_new, int64_t kv_stride, void *out, float scale, int window, int max_len, void *work,
                int64_t work_bytes, void *stream) {
    return guarded(h, fn, [&](Call &c) {
        if (!lens || !table || !q || !out || (append && (!k_new || !v_new)) ||
            (granted.told && (!granted.n_new || !granted.status)))
            return c.null();
        if (int rc = check_layer(c, layer)) return rc;
        if (int rc = check_table(c, n_batch, max_pages)) return rc;
        if (int rc = check_heads(c, n_heads)) return rc;
        const bmo::PagesGeom &g = c.h->g;
        // (a workgroup of 256 a head at most: the grid's threads stay below 2^32)
        if ((int64_t) n_batch * n_heads > (1 << 23)) return c.arg("n_batch * n_heads must be at most 2^23");
        if (type < bmo::kTypeF32 || type > bmo::kTypeBF16) return c.arg("rows must be fp32, fp16 or bf16");
        if (const char *why = row_fault(q, q_stride, (int64_t) n_heads * g.dim, type)) return c.arg(why);
        if (append) {
            const int64_t given = kv_stride;
            if (const char *why = row_fault(k_new, kv_stride, (int64_t) g.n_kv * g.dim, type)) return c.arg(why);
            kv_stride = given;
            if (const char *why = row_fault(v_new, kv_stride, (int64_t) g.n_kv * g.dim, type)) return c.arg(why);
        }
        if (!aligned(out, 16) || !aligned(work, 16)) return c.arg("out and workspace must be aligned to 16 bytes");
        if (window < 0 || max_len < 0 || work_bytes < 0) return c.arg("window, max_len and sizes must not be negative");
        if (!(scale > 0.0f)) scale = 1.0f / std::sqrt((float) g.dim);
        if (!std::isfinite(scale)) return c.arg("scale must be finite");
        c.enter();
        bmo::PagesDecodeParams p{};
        p.base = c.h->mem + layer * g.layer_bytes;
        p.g = g;
        p.n_batch = n_batch;
        p.n_heads = n_heads;
        p.lens = lens;
        p.n_new = granted.n_new;
        p.status = granted.status;
        p.table = table;
        p.max_pages = max_pages;
        p.window = (int64_t) window >= (int64_t) max_pages << g.page_shift ? 0 : window;
        p.type = type;
        p.q = q;
        p.q_stride = q_stride;
        p.k_new = append ? k_new : nullptr;
        p.v_new = append ? v_new : nullptr;
        p.kv_stride = kv_stride;
        p.out = out;
        p.qscale = scale * kLog2e;
        p.max_len = max_len;
        p.work = static_cast<float *>(work);
        p.work_bytes = work_bytes;
        return c.done(bmo::launch_pages_decode(p, (hipStream_t) stream));
    });
}

int attend_call(bmo_kv_pages_t *h, const char *fn, Granted granted, int layer, int n_batch, const int *q_start,
                const int *lens, const int *table, int max_pages, int n_rows, int n_heads, int type, const void *q,
                int64_t q_stride, void *out, float scale, int causal, int window, int max_rows, int max_len,
                void *workspace, int64_t workspace_bytes, void *stream) {
    return guarded(h, fn, [&](Call &c) {
        if (!q_start || !lens || !table || (n_rows != 0 && (!q || !out)) || (granted.told && !granted.status))
            return c.null();
        if (int rc = check_layer(c, layer)) return rc;
        if (int rc = check_table(c, n_batch, max_pages)) return rc;
        if (int rc = check_heads(c, n_heads)) return rc;
        const bmo::PagesGeom &g = c.h->g;
        if (type != bmo::kTypeF16 && type != bmo::kTypeBF16) return c.arg("rows must be fp16 or bf16");
        if (n_rows < 0 || (int64_t) n_rows * n_heads > (1 << 30))
            return c.arg("n_rows must not be negative, n_rows * n_heads at most 2^30");
        // (tiles: 2^23 of rows and one an entry and kv head, 256 threads each)
        if ((int64_t) n_batch * g.n_kv > (1 << 22)) return c.arg("n_batch * n_kv_heads must be at most 2^22");
        if (const char *why = row_fault(q, q_stride, (int64_t) n_heads * g.dim, type)) return c.arg(why);
        if (!aligned(out, 16) || !aligned(workspace, 16)) return c.arg("out and workspace must be aligned to 16 bytes");
        if (window < 0 || max_rows < 0 || max_len < 0 || workspace_bytes < 0)
            return c.arg("window, max_rows, max_len and sizes must not be negative");
        if (!(scale > 0.0f)) scale = 1.0f / std::sqrt((float) g.dim);
        if (!std::isfinite(scale)) return c.arg("scale must be finite");
        if (n_rows == 0) return c.done(hipSuccess);
        c.enter();
        bmo::PagesAttendParams p{};
        p.base = c.h->mem + layer * g.layer_bytes;
        p.g = g;
        p.n_batch = n_batch;
        p.n_heads = n_heads;
        p.q_start = q_start;
        p.lens = lens;
        p.status = granted.status;
        p.table = table;
        p.max_pages = max_pages;
        p.n_rows = n_rows;
        p.causal = causal != 0;
        p.window = (int64_t) window >= (int64_t) max_pages << g.page_shift ? 0 : window;
        p.type = type;
        p.q = q;
        p.q_stride = q_stride;
        p.out = out;
        p.qscale = scale * kLog2e;
        p.max_rows = max_rows;
        p.max_len = max_len;
        p.work = static_cast<float *>(workspace);
        p.work_bytes = workspace_bytes;
        return c.done(bmo::launch_pages_attend(p, (hipStream_t) stream));
    });
}

}  // namespace

extern "C" {

bmo_kv_pages_t *bmo_kv_pages_create(int n_layers, int n_pages, int page_size, int n_kv_heads, int head_dim) {
    t_create_error.clear();
    auto reject = [](const std::string &m) -> bmo_kv_pages_t * {
        t_create_error = "bmo_kv_pages_create: " + m;
        std::fprintf(stderr, "[bmo_attn] %s\n", t_create_error.c_str());
        return nullptr;
    };
    bmo_kv_pages_t *h = nullptr;
    try {
        if (n_layers <= 0 || n_pages <= 0 || n_kv_heads <= 0)
            return reject("n_layers, n_pages and n_kv_heads must be positive");
        if (head_dim != 64 && head_dim != 128) return reject("head_dim must be 64 or 128");
        const int group = bmo::keys_per_group(head_dim);
        if (page_size < group || page_size > 1024 || (page_size & (page_size - 1)) != 0)
            return reject("page_size must be a power of two, from " + std::to_string(group) + " to 1024 at this head_dim");
        if ((int64_t) n_pages * page_size > INT_MAX || n_kv_heads > 65536)
            return reject("n_pages * page_size must be below 2^31, n_kv_heads at most 65536");
        const double total = (double) n_layers * n_pages * n_kv_heads * (page_size / group) * bmo::kGroupBytes;
        if (total > 1e15) return reject("too large");
        h = new bmo_kv_pages();
        h->g = bmo::make_pages_geom(n_layers, n_pages, page_size, n_kv_heads, head_dim);
        if (hipGetDevice(&h->device) != hipSuccess) {
            delete h;
            return reject("no HIP device");
        }
        const int64_t bytes = h->g.layer_bytes * n_layers;
        hipError_t e = hipMalloc(&h->mem, (size_t) bytes);
        if (e != hipSuccess) {
            delete h;
            return reject("hipMalloc of " + std::to_string(bytes) + " bytes failed: " + hipGetErrorString(e));
        }
        e = bmo::launch_pages_clear(h->mem, bytes, nullptr);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            (void) hipFree(h->mem);
            delete h;
            return reject(std::string("initialisation failed: ") + hipGetErrorString(e));
        }
        return h;
    } catch (...) {
        if (h && h->mem) (void) hipFree(h->mem);
        delete h;
        return reject("exception");
    }
}

void bmo_kv_pages_free(bmo_kv_pages_t *h) {
    if (!h) return;
    int prev = -1;
    const bool other = hipGetDevice(&prev) == hipSuccess && prev != h->device && hipSetDevice(h->device) == hipSuccess;
    (void) hipFree(h->mem);
    if (other) (void) hipSetDevice(prev);
    delete h;
}

int64_t bmo_kv_pages_bytes(const bmo_kv_pages_t *h) { return h ? h->g.layer_bytes * h->g.n_layers : 0; }

int bmo_kv_pages_device(const bmo_kv_pages_t *h) { return h ? h->device : -1; }

const char *bmo_kv_pages_last_error(const bmo_kv_pages_t *h) {
    if (!h) return t_create_error.empty() ? nullptr : t_create_error.c_str();
    thread_local std::string t_copy;
    auto *m = const_cast<bmo_kv_pages_t *>(h);
    {
        std::lock_guard<std::mutex> lk(m->mu);
        t_copy = m->last_error;
    }
    return t_copy.empty() ? nullptr : t_copy.c_str();
}

int bmo_kv_pages_list_init(bmo_kv_pages_t *h, int *free_list, void *stream) {
    return guarded(h, "bmo_kv_pages_list_init", [&](Call &c) {
        if (!free_list) return c.null();
        c.enter();
        return c.done(bmo::launch_list_init(free_list, c.h->g.n_pages, (hipStream_t) stream));
    });
}

int bmo_kv_pages_plan(bmo_kv_pages_t *h, int *free_list, int n_batch, const int *n_new, int *lens, int *table,
                      int max_pages, int *tok_start, int max_tok, int *tok_slot, int *tok_pos, int *tok_entry, int *status,
                      void *stream) {
    return guarded(h, "bmo_kv_pages_plan", [&](Call &c) {
        if (!free_list || !n_new || !lens || !table) return c.null();
        if (int rc = check_table(c, n_batch, max_pages)) return rc;
        if (max_tok < 0) return c.arg("max_tok must not be negative");
        c.enter();
        bmo::PlanParams p{};
        p.list = free_list;
        p.n_pages = c.h->g.n_pages;
        p.page_shift = c.h->g.page_shift;
        p.n_batch = n_batch;
        p.n_new = n_new;
        p.lens = lens;
        p.table = table;
        p.max_pages = max_pages;
        p.tok_start = tok_start;
        p.max_tok = max_tok;
        p.tok_slot = tok_slot;
        p.tok_pos = tok_pos;
        p.tok_entry = tok_entry;
        p.status = status;
        return c.done(bmo::launch_plan(p, (hipStream_t) stream));
    });
}

int bmo_kv_pages_append(bmo_kv_pages_t *h, int layer, int n_tok, const int *slots, int type, const void *k, const void *v,
                        int64_t stride, void *stream) {
    return slots_call(h, "bmo_kv_pages_append", true, layer, n_tok, slots, type, const_cast<void *>(k),
                      const_cast<void *>(v), stride, stream);
}

int bmo_kv_pages_gather(bmo_kv_pages_t *h, int layer, int n_tok, const int *slots, int type, void *k, void *v,
                        int64_t stride, void *stream) {
    return slots_call(h, "bmo_kv_pages_gather", false, layer, n_tok, slots, type, k, v, stride, stream);
}

int64_t bmo_kv_pages_workspace_bytes(const bmo_kv_pages_t *h, int n_heads) {
    if (!h || n_heads <= 0 || n_heads % h->g.n_kv != 0) return 0;
    return bmo::pages_work_bytes(h->g);
}

int bmo_kv_pages_decode(bmo_kv_pages_t *h, int layer, int n_batch, const int *lens, const int *table, int max_pages,
                        int n_heads, int type, const void *q, int64_t q_stride, void *out, float scale, int window,
                        int max_len, void *workspace, int64_t workspace_bytes, void *stream) {
    return decode_call(h, "bmo_kv_pages_decode", false, {}, layer, n_batch, lens, table, max_pages, n_heads, type, q, q_stride,
                       nullptr, nullptr, 0, out, scale, window, max_len, workspace, workspace_bytes, stream);
}

int bmo_kv_pages_append_decode(bmo_kv_pages_t *h, int layer, int n_batch, const int *lens, const int *table, int max_pages,
                               int n_heads, int type, const void *q, int64_t q_stride, const void *k_new,
                               const void *v_new, int64_t kv_stride, void *out, float scale, int window, int max_len,
                               void *workspace, int64_t workspace_bytes, void *stream) {
    return decode_call(h, "bmo_kv_pages_append_decode", true, {}, layer, n_batch, lens, table, max_pages, n_heads, type, q,
                       q_stride, k_new, v_new, kv_stride, out, scale, window, max_len, workspace, workspace_bytes, stream);
}

int bmo_kv_pages_append_decode_granted(bmo_kv_pages_t *h, int layer, int n_batch, const int *n_new, const int *status,
                                       const int *lens, const int *table, int max_pages, int n_heads, int type,
                                       const void *q, int64_t q_stride, const void *k_new, const void *v_new,
                                       int64_t kv_stride, void *out, float scale, int window, int max_len, void *workspace,
                                       int64_t workspace_bytes, void *stream) {
    return decode_call(h, "bmo_kv_pages_append_decode_granted", true, {true, n_new, status}, layer, n_batch, lens, table,
                       max_pages, n_heads, type, q, q_stride, k_new, v_new, kv_stride, out, scale, window, max_len,
                       workspace, workspace_bytes, stream);
}

int bmo_kv_pages_attend(bmo_kv_pages_t *h, int layer, int n_batch, const int *q_start, const int *lens, const int *table,
                        int max_pages, int n_rows, int n_heads, int type, const void *q, int64_t q_stride, void *out,
                        float scale, int causal, int window, int max_rows, int max_len, void *workspace,
                        int64_t workspace_bytes, void *stream) {
    return attend_call(h, "bmo_kv_pages_attend", {}, layer, n_batch, q_start, lens, table, max_pages, n_rows, n_heads, type,
                       q, q_stride, out, scale, causal, window, max_rows, max_len, workspace, workspace_bytes, stream);
}

int bmo_kv_pages_attend_granted(bmo_kv_pages_t *h, int layer, int n_batch, const int *status, const int *q_start,
                                const int *lens, const int *table, int max_pages, int n_rows, int n_heads, int type,
                                const void *q, int64_t q_stride, void *out, float scale, int causal, int window,
                                int max_rows, int max_len, void *workspace, int64_t workspace_bytes, void *stream) {
    return attend_call(h, "bmo_kv_pages_attend_granted", {true, nullptr, status}, layer, n_batch, q_start, lens, table,
                       max_pages, n_rows, n_heads, type, q, q_stride, out, scale, causal, window, max_rows, max_len,
                       workspace, workspace_bytes, stream);
}

}  // extern "C"
