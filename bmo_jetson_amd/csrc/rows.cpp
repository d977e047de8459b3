// rows.cpp -- the C ABI of the operators on rows (include/bmo_attn.h): norm,
// 8-bit rows, rotary positions, Q4_0 weights.  Conventions as in pages.cpp:
// nothing throws across the ABI, int entry points return a status and record a
// message, a failed create returns NULL and says why on stderr.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/bmo_attn.h"
#include "rows.hpp"
#include "spans.hpp"

static_assert(BMO_ATTN_SILU == bmo::kSilu && BMO_ATTN_GELU == bmo::kGelu, "the header's activations");

namespace bmo {

// What every handle of these operators has.
struct RowsHandle {
    int device = 0;
    std::mutex mu;  // guards last_error
    std::string last_error;
};

}  // namespace bmo

struct bmo_rope : bmo::RowsHandle {
    int dim = 0, rot = 0, interleaved = 0;
    float magnitude = 1.0f;
    double *rates = nullptr;
};

struct bmo_weights : bmo::RowsHandle {
    bmo::WeightsGeom g{};
    uint8_t *mem = nullptr;
};

namespace {

using Handle = bmo::RowsHandle;

thread_local std::string t_rows_error, t_rope_error, t_weights_error;

// What an entry point does: collects its name's errors (the handle's, or the
// thread's for calls without one) and keeps the handle's device current.
struct Call {
    Handle *h;
    const char *fn;
    int prev = -1;
    bool switched = false;
    Call(Handle *h_, const char *fn_) : h(h_), fn(fn_) {}
    ~Call() {
        if (switched) (void) hipSetDevice(prev);
    }
    int fail(int code, const std::string &why) {
        record(std::string(fn) + ": " + why);
        return code;
    }
    int null() { return fail(BMO_ATTN_ERR_NULL, "null pointer argument"); }
    int arg(const std::string &why) { return fail(BMO_ATTN_ERR_ARG, why); }
    // Ends a call: the launch's own status.
    int done(hipError_t e) {
        if (e != hipSuccess) return fail(BMO_ATTN_ERR_HIP, hipGetErrorString(e));
        record(std::string());
        return BMO_ATTN_OK;
    }
    void enter() {
        if (h && hipGetDevice(&prev) == hipSuccess && prev != h->device) switched = hipSetDevice(h->device) == hipSuccess;
    }

  private:
    void record(const std::string &m) {
        if (!h) {
            t_rows_error = m;
            return;
        }
        std::lock_guard<std::mutex> lk(h->mu);
        h->last_error = m;
    }
};

// Runs f(call) behind the exception barrier.
template <class F>
int guarded(Handle *h, const char *fn, F f) {
    try {
        Call c(h, fn);
        return f(c);
    } catch (...) {
        return BMO_ATTN_ERR_INTERNAL;
    }
}

const char *message(Handle *h, const std::string &of_create) {
    if (!h) return of_create.empty() ? nullptr : of_create.c_str();
    thread_local std::string t_copy;
    {
        std::lock_guard<std::mutex> lk(h->mu);
        t_copy = h->last_error;
    }
    return t_copy.empty() ? nullptr : t_copy.c_str();
}

bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr int64_t kMaxStride = int64_t(1) << 40;

// Rows of `dense` elements, stride elements apart (0: dense): nullptr, or why
// they are refused.
const char *row_fault(const void *p, int64_t &stride, int64_t dense, int type) {
    if (type < bmo::kTypeF32 || type > bmo::kTypeBF16) return "rows must be fp32, fp16 or bf16";
    if (stride == 0) stride = dense;
    if (stride < dense) return "a stride is shorter than its row";
    if (stride > kMaxStride) return "a stride is too long";
    if (!aligned(p, bmo::type_bytes(type))) return "rows must be aligned to their elements";
    return nullptr;
}

const char *rows8_fault(const void *codes, const void *scales) {
    return aligned(codes, 16) && aligned(scales, 2) ? nullptr
                                                    : "codes must be aligned to 16 bytes, scales to their elements";
}

using bmo::Span;
using bmo::meet;

Span span(const void *p, int64_t n, int64_t elements, int64_t stride, int size) {
    return {p, n, elements * size, stride * size};
}
Span span8(const void *codes, int64_t n, int64_t cols) { return {codes, 1, n * cols, 0}; }
Span span_scales(const void *scales, int64_t n, int64_t cols) { return {scales, 1, n * (cols / 32) * 2, 0}; }

// Whether anything written meets what else is written or read.
bool overlap(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (const Span *w = written.begin(); w != written.end(); ++w) {
        for (const Span *o = w + 1; o != written.end(); ++o)
            if (meet(*w, *o)) return true;
        for (const Span &r : read)
            if (meet(*w, r)) return true;
    }
    return false;
}

// A create that failed: says why and returns nullptr.
std::nullptr_t refused(std::string &error, const char *fn, const std::string &why) {
    error = std::string(fn) + ": " + why;
    std::fprintf(stderr, "[bmo_attn] %s\n", error.c_str());
    return nullptr;
}

// Frees device memory of a handle's device.
void release(Handle *h, void *mem) {
    int prev = -1;
    const bool other = hipGetDevice(&prev) == hipSuccess && prev != h->device && hipSetDevice(h->device) == hipSuccess;
    (void) hipFree(mem);
    if (other) (void) hipSetDevice(prev);
}

// Radians a position of each pair: theta^(-2i / rot), divided by factor; with
// a trained length by YaRN's blend (Peng, Quesnelle, Fan and Shippole, "YaRN:
// Efficient Context Window Extension of Large Language Models", 2023): pairs
// that turn fewer than beta_slow times over that length are divided by
// factor, those that turn more than beta_fast times are not.
std::vector<double> rope_rates(int rot, double theta, double factor, int trained, double beta_fast, double beta_slow,
                               const double *divisors) {
    const double pi = 3.14159265358979323846;
    auto pair_of = [&](double turns) { return rot * std::log(trained / (turns * 2 * pi)) / (2 * std::log(theta)); };
    double low = 0, high = 0;
    if (trained) {
        low = std::fmax(std::floor(pair_of(beta_fast)), 0.0);
        high = std::fmin(std::ceil(pair_of(beta_slow)), rot - 1.0);
    }
    std::vector<double> rates((size_t) rot / 2);
    for (int i = 0; i < rot / 2; ++i) {
        const double base = std::pow(theta, -2.0 * i / rot);
        const double slow = trained ? std::fmin(std::fmax((i - low) / std::fmax(high - low, 0.001), 0.0), 1.0) : 1.0;
        rates[(size_t) i] = (base * (1.0 - slow) + base / factor * slow) / (divisors ? divisors[i] : 1.0);
    }
    return rates;
}

int product_call(bmo_weights_t *h, const char *fn, bool gated, int n_rows, const void *codes, const void *scales,
                 int activation, int type, void *out, int64_t out_stride, void *out_codes, void *out_scales, void *stream) {
    if (!h) return BMO_ATTN_ERR_NULL;
    return guarded(h, fn, [&](Call &c) {
        // (an empty tensor has no address)
        if (n_rows != 0 && (!codes || !scales || (!gated && !out))) return c.null();
        if (!out_codes != !out_scales) return c.arg("codes and scales come together");
        if (gated && n_rows != 0 && !out && !out_codes) return c.null();
        if (n_rows < 0 || n_rows > (1 << 20)) return c.arg("n_rows must be at least 0 and at most 2^20");
        if (gated && h->g.rows % 64 != 0) return c.arg("a gated product needs gates and outputs in whole blocks of 32 rows");
        if (gated && activation != bmo::kSilu && activation != bmo::kGelu) return c.arg("unknown activation");
        const int n_out = gated ? h->g.rows / 2 : h->g.rows;
        if (out) {
            if (const char *why = row_fault(out, out_stride, n_out, type)) return c.arg(why);
        }
        if (const char *why = rows8_fault(codes, scales)) return c.arg(why);
        if (const char *why = rows8_fault(out_codes, out_scales)) return c.arg(why);
        if (n_rows == 0) return c.done(hipSuccess);
        if (overlap({span(out, n_rows, n_out, out_stride, bmo::type_bytes(type)), span8(out_codes, n_rows, n_out),
                     span_scales(out_scales, n_rows, n_out)},
                    {span8(codes, n_rows, h->g.cols), span_scales(scales, n_rows, h->g.cols)}))
            return c.arg("what is written overlaps what is read, or something else that is written");
        c.enter();
        bmo::ProductParams p{};
        p.w = h->mem;
        p.g = h->g;
        p.n_rows = n_rows;
        p.codes = static_cast<const int8_t *>(codes);
        p.scales = static_cast<const uint16_t *>(scales);
        p.activation = gated ? activation : bmo::kNoActivation;
        p.type = type;
        p.out = out;
        p.out_stride = out_stride;
        p.out_codes = static_cast<int8_t *>(out_codes);
        p.out_scales = static_cast<uint16_t *>(out_scales);
        return c.done(bmo::launch_product(p, (hipStream_t) stream));
    });
}

}  // namespace

extern "C" {

const char *bmo_rows_last_error(void) { return t_rows_error.empty() ? nullptr : t_rows_error.c_str(); }

int bmo_rms_norm(int n_rows, int dim, int type, const void *x, int64_t x_stride, int residual_type, void *residual,
                 int64_t residual_stride, int weight_type, const void *weight, float eps, int out_type, void *out,
                 int64_t out_stride, void *codes, void *scales, void *stream) {
    return guarded(nullptr, "bmo_rms_norm", [&](Call &c) {
        if (!weight || (n_rows != 0 && (!x || (!out && !codes)))) return c.null();
        if (!codes != !scales) return c.arg("codes and scales come together");
        // (a workgroup of up to 1024 a row: the grid's threads stay below 2^32)
        if (n_rows < 0 || n_rows >= (1 << 22)) return c.arg("n_rows must be at least 0 and below 2^22");
        if (dim <= 0 || dim > bmo::kNormMaxDim) return c.arg("dim must be positive and at most 32768");
        if (codes && dim % 32 != 0) return c.arg("8-bit rows need a dim that is a multiple of 32");
        if (!(eps >= 0.0f) || !std::isfinite(eps)) return c.arg("eps must be finite and not negative");
        int64_t w_stride = 0;
        if (const char *why = row_fault(x, x_stride, dim, type)) return c.arg(why);
        if (const char *why = row_fault(weight, w_stride, dim, weight_type)) return c.arg(why);
        if (residual) {
            if (const char *why = row_fault(residual, residual_stride, dim, residual_type)) return c.arg(why);
        }
        if (out) {
            if (const char *why = row_fault(out, out_stride, dim, out_type)) return c.arg(why);
        }
        if (const char *why = rows8_fault(codes, scales)) return c.arg(why);
        if (n_rows == 0) return c.done(hipSuccess);
        const Span rows = span(x, n_rows, dim, x_stride, bmo::type_bytes(type));
        const Span sums = span(residual, n_rows, dim, residual_stride, bmo::type_bytes(residual_type));
        const Span result = span(out, n_rows, dim, out_stride, bmo::type_bytes(out_type));
        const Span w = span(weight, 1, dim, dim, bmo::type_bytes(weight_type));
        const bool in_place = result == rows && out_type == type, doubled = sums == rows && residual_type == type;
        if (overlap({sums, result, span8(codes, n_rows, dim), span_scales(scales, n_rows, dim)}, {w}) ||
            overlap({span8(codes, n_rows, dim), span_scales(scales, n_rows, dim)}, {rows}) ||
            (!in_place && meet(result, rows)) || (!doubled && meet(sums, rows)))
            return c.arg("what is written overlaps what is read, or something else that is written");
        bmo::NormParams p{};
        p.n_rows = n_rows;
        p.dim = dim;
        p.type = type;
        p.x = x;
        p.x_stride = x_stride;
        p.res_type = residual_type;
        p.res = residual;
        p.res_stride = residual_stride;
        p.w_type = weight_type;
        p.w = weight;
        p.eps = eps;
        p.out_type = out_type;
        p.out = out;
        p.out_stride = out_stride;
        p.codes = static_cast<int8_t *>(codes);
        p.scales = static_cast<uint16_t *>(scales);
        return c.done(bmo::launch_norm(p, (hipStream_t) stream));
    });
}

int bmo_quantize_rows(int n_rows, int cols, int type, const void *x, int64_t stride, void *codes, void *scales,
                      void *stream) {
    return guarded(nullptr, "bmo_quantize_rows", [&](Call &c) {
        if (n_rows != 0 && (!x || !codes || !scales)) return c.null();
        if (n_rows < 0) return c.arg("n_rows must not be negative");
        if (cols <= 0 || cols % 32 != 0) return c.arg("cols must be a positive multiple of 32");
        // (a thread an octet: their number stays below 2^31)
        if ((int64_t) n_rows * (cols / 8) > (int64_t(1) << 30)) return c.arg("too large (2^33 elements)");
        if (const char *why = row_fault(x, stride, cols, type)) return c.arg(why);
        if (const char *why = rows8_fault(codes, scales)) return c.arg(why);
        if (n_rows == 0) return c.done(hipSuccess);
        if (overlap({span8(codes, n_rows, cols), span_scales(scales, n_rows, cols)},
                    {span(x, n_rows, cols, stride, bmo::type_bytes(type))}))
            return c.arg("what is written overlaps what is read, or something else that is written");
        bmo::QuantizeParams p{};
        p.n_rows = n_rows;
        p.cols = cols;
        p.type = type;
        p.x = x;
        p.stride = stride;
        p.codes = static_cast<int8_t *>(codes);
        p.scales = static_cast<uint16_t *>(scales);
        return c.done(bmo::launch_quantize_rows(p, (hipStream_t) stream));
    });
}

bmo_rope_t *bmo_rope_create(int head_dim, int rot_dim, int interleaved, double theta, double factor, int trained,
                            double beta_fast, double beta_slow, double magnitude, const double *divisors) {
    const char *fn = "bmo_rope_create";
    bmo_rope_t *h = nullptr;
    try {
        t_rope_error.clear();
        auto reject = [&](const std::string &why) -> bmo_rope_t * { return refused(t_rope_error, fn, why); };
        if (head_dim <= 0 || head_dim > 1024) return reject("head_dim must be positive and at most 1024");
        if (rot_dim <= 0 || rot_dim > head_dim || rot_dim % 2 != 0)
            return reject("rot_dim must be positive, even and at most head_dim");
        if (!(theta > 1.0) || !std::isfinite(theta)) return reject("theta must be above 1 and finite");
        if (!(factor > 0.0) || !std::isfinite(factor)) return reject("factor must be positive and finite");
        if (trained < 0) return reject("trained must not be negative");
        if (!(beta_fast > 0.0)) beta_fast = 32.0;
        if (!(beta_slow > 0.0)) beta_slow = 1.0;
        if (!std::isfinite(beta_fast) || !std::isfinite(beta_slow)) return reject("betas must be finite");
        if (!(magnitude > 0.0)) magnitude = trained && factor > 1.0 ? 0.1 * std::log(factor) + 1.0 : 1.0;
        if (!std::isfinite((float) magnitude)) return reject("magnitude must be finite in fp32");
        const std::vector<double> rates = rope_rates(rot_dim, theta, factor, trained, beta_fast, beta_slow, divisors);
        // (angles stay below 2^31 in magnitude, where the kernel's reduction holds)
        for (double r : rates)
            if (!(r >= 0.0 && r <= 1.0)) return reject("a pair would turn by more than a radian a position");
        h = new bmo_rope();
        h->dim = head_dim;
        h->rot = rot_dim;
        h->interleaved = interleaved != 0;
        h->magnitude = (float) magnitude;
        hipError_t e = hipGetDevice(&h->device);
        if (e == hipSuccess) e = hipMalloc(&h->rates, rates.size() * sizeof(double));
        if (e == hipSuccess) e = hipMemcpy(h->rates, rates.data(), rates.size() * sizeof(double), hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            if (h->rates) (void) hipFree(h->rates);
            delete h;
            return reject(hipGetErrorString(e));
        }
        return h;
    } catch (...) {
        if (h && h->rates) (void) hipFree(h->rates);
        delete h;
        return nullptr;
    }
}

void bmo_rope_free(bmo_rope_t *h) {
    if (!h) return;
    release(h, h->rates);
    delete h;
}

int bmo_rope_device(const bmo_rope_t *h) { return h ? h->device : -1; }

const char *bmo_rope_last_error(const bmo_rope_t *h) { return message(const_cast<bmo_rope_t *>(h), t_rope_error); }

int bmo_rope_apply(bmo_rope_t *h, int n_tok, const int *positions, int type, int n_heads, const void *q, int64_t q_stride,
                   void *q_out, int64_t q_out_stride, int n_kv_heads, const void *k, int64_t k_stride, void *k_out,
                   int64_t k_out_stride, void *stream) {
    if (!h) return BMO_ATTN_ERR_NULL;
    return guarded(h, "bmo_rope_apply", [&](Call &c) {
        if (n_tok != 0 && (!positions || !q || !q_out || (n_kv_heads != 0 && (!k || !k_out)))) return c.null();
        if (n_tok < 0) return c.arg("n_tok must not be negative");
        if (n_heads <= 0 || n_kv_heads < 0 || n_heads > 4096 || n_kv_heads > 4096)
            return c.arg("n_heads must be positive, n_kv_heads not negative, both at most 4096");
        // (a workgroup takes at least 512 elements, or a whole token: their number stays below 2^24)
        if ((int64_t) n_tok * (n_heads + n_kv_heads) * h->dim > (int64_t(1) << 32)) return c.arg("too large (2^32 elements)");
        const int64_t q_dense = (int64_t) n_heads * h->dim, k_dense = (int64_t) n_kv_heads * h->dim;
        if (const char *why = row_fault(q, q_stride, q_dense, type)) return c.arg(why);
        if (const char *why = row_fault(q_out, q_out_stride, q_dense, type)) return c.arg(why);
        if (n_kv_heads) {
            if (const char *why = row_fault(k, k_stride, k_dense, type)) return c.arg(why);
            if (const char *why = row_fault(k_out, k_out_stride, k_dense, type)) return c.arg(why);
        }
        if ((q == q_out && q_stride != q_out_stride) || (n_kv_heads && k == k_out && k_stride != k_out_stride))
            return c.arg("rows turned in place keep their stride");
        if (n_tok == 0) return c.done(hipSuccess);
        const int size = bmo::type_bytes(type);
        const Span qs = span(q, n_tok, q_dense, q_stride, size), qo = span(q_out, n_tok, q_dense, q_out_stride, size);
        const Span none = {nullptr, 0, 0, 0};
        const Span ks = n_kv_heads ? span(k, n_tok, k_dense, k_stride, size) : none;
        const Span ko = n_kv_heads ? span(k_out, n_tok, k_dense, k_out_stride, size) : none;
        if (overlap({qo, ko}, {{positions, 1, (int64_t) n_tok * 4, 0}}) || meet(qo, ks) || meet(ko, qs) ||
            (q != q_out && meet(qo, qs)) || (k != k_out && meet(ko, ks)))
            return c.arg("what is written overlaps what is read, or something else that is written");
        c.enter();
        bmo::RopeParams p{};
        p.rates = h->rates;
        p.magnitude = h->magnitude;
        p.dim = h->dim;
        p.rot = h->rot;
        p.interleaved = h->interleaved;
        p.n_tok = n_tok;
        p.positions = positions;
        p.type = type;
        p.part[0] = {n_heads, q, q_stride, q_out, q_out_stride};
        p.part[1] = {n_kv_heads, k, k_stride, k_out, k_out_stride};
        return c.done(bmo::launch_rope(p, (hipStream_t) stream));
    });
}

bmo_weights_t *bmo_weights_create(int rows, int cols) {
    const char *fn = "bmo_weights_create";
    bmo_weights_t *h = nullptr;
    try {
        t_weights_error.clear();
        auto reject = [&](const std::string &why) -> bmo_weights_t * { return refused(t_weights_error, fn, why); };
        if (rows <= 0 || rows > (1 << 24)) return reject("rows must be positive and at most 2^24");
        if (cols <= 0 || cols % 32 != 0 || cols > (1 << 24))
            return reject("cols must be a positive multiple of 32 and at most 2^24");
        h = new bmo_weights();
        h->g = bmo::make_weights_geom(rows, cols);
        hipError_t e = hipGetDevice(&h->device);
        const int64_t bytes = bmo::weights_bytes(h->g);
        if (e == hipSuccess) e = hipMalloc(&h->mem, (size_t) bytes);
        if (e == hipSuccess) e = bmo::launch_pages_clear(h->mem, bytes, nullptr);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            if (h->mem) (void) hipFree(h->mem);
            delete h;
            return reject(std::to_string(bytes) + " bytes: " + hipGetErrorString(e));
        }
        return h;
    } catch (...) {
        if (h && h->mem) (void) hipFree(h->mem);
        delete h;
        return nullptr;
    }
}

void bmo_weights_free(bmo_weights_t *h) {
    if (!h) return;
    release(h, h->mem);
    delete h;
}

int64_t bmo_weights_bytes(const bmo_weights_t *h) { return h ? bmo::weights_bytes(h->g) : 0; }

int bmo_weights_device(const bmo_weights_t *h) { return h ? h->device : -1; }

const char *bmo_weights_last_error(const bmo_weights_t *h) {
    return message(const_cast<bmo_weights_t *>(h), t_weights_error);
}

int bmo_weights_load(bmo_weights_t *h, int row, int n_rows, const void *blocks, void *stream) {
    if (!h) return BMO_ATTN_ERR_NULL;
    return guarded(h, "bmo_weights_load", [&](Call &c) {
        if (n_rows != 0 && !blocks) return c.null();
        if (row < 0 || n_rows < 0 || (int64_t) row + n_rows > h->g.rows) return c.arg("rows out of range");
        if (!aligned(blocks, 2)) return c.arg("blocks must be aligned to 2 bytes");
        if ((int64_t) n_rows * (h->g.cols / 32) > (int64_t(1) << 30)) return c.arg("n_rows too large (2^30 blocks)");
        if (n_rows == 0) return c.done(hipSuccess);
        c.enter();
        bmo::PackParams p{};
        p.w = h->mem;
        p.g = h->g;
        p.row0 = row;
        p.n_rows = n_rows;
        p.blocks = static_cast<const uint8_t *>(blocks);
        return c.done(bmo::launch_weights_pack(p, (hipStream_t) stream));
    });
}

int bmo_weights_product(bmo_weights_t *h, int n_rows, const void *codes, const void *scales, int type, void *out,
                        int64_t out_stride, void *stream) {
    return product_call(h, "bmo_weights_product", false, n_rows, codes, scales, 0, type, out, out_stride, nullptr, nullptr,
                        stream);
}

int bmo_weights_gated(bmo_weights_t *h, int n_rows, const void *codes, const void *scales, int activation, int type,
                      void *out, int64_t out_stride, void *out_codes, void *out_scales, void *stream) {
    return product_call(h, "bmo_weights_gated", true, n_rows, codes, scales, activation, type, out, out_stride, out_codes,
                        out_scales, stream);
}

}  // extern "C"
