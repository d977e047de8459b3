// rows_norm.hip -- RMS norm of rows with the residual's addition, and rows in
// 8 bits.
//
//   h = residual + x    (kept in the residual, rounded to its type; else h = x)
//   y = h / sqrt(mean(h^2) + eps) * w
//
// y leaves in 16 or 32 bits and as 8-bit rows for the products.  A team of T
// threads takes a row: eight elements a thread and step, NV steps, all loads
// (the weight's too) under way at once; the row stays in registers between the
// sum and the scaling, so that it is read once.
#include "kernels.hpp"
#include "rows_device.hpp"

namespace bmo {

namespace {

__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// Eight elements of a row: neighbours from 8 (i T + t) on, or, in rows that are
// not aligned for that, T apart from 8 i T + t on; those past the row's end as
// zeros.
template <int T, bool VEC>
struct Eight {
    int e;
    __device__ __forceinline__ Eight(int i, int t) : e(VEC ? (i * T + t) * 8 : i * T * 8 + t) {}
    __device__ __forceinline__ Raw8 load(const void *p, int64_t row, int dim, int type) const {
        Raw8 r = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if constexpr (VEC) {
            if (e < dim) r = load_raw8(p, row + e, type);
        } else {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = e + j * T < dim ? load1(p, row + e + j * T, type) : 0.0f;
            r.a = make_uint4(__builtin_bit_cast(uint32_t, x[0]), __builtin_bit_cast(uint32_t, x[1]),
                             __builtin_bit_cast(uint32_t, x[2]), __builtin_bit_cast(uint32_t, x[3]));
            r.b = make_uint4(__builtin_bit_cast(uint32_t, x[4]), __builtin_bit_cast(uint32_t, x[5]),
                             __builtin_bit_cast(uint32_t, x[6]), __builtin_bit_cast(uint32_t, x[7]));
        }
        return r;
    }
    static __device__ __forceinline__ void widen(const Raw8 &r, int type, float (&x)[8]) {
        widen8(r, VEC ? type : kTypeF32, x);
    }
    __device__ __forceinline__ void store(void *p, int64_t row, int dim, const float (&x)[8], int type) const {
        if constexpr (VEC) {
            if (e < dim) store8(p, row + e, x, type);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (e + j * T < dim) store1(p, row + e + j * T, x[j], type);
        }
    }
    // (dim is a multiple of 32: a block is four lanes' eights, or 32 lanes')
    __device__ __forceinline__ void store_codes(int8_t *codes, uint16_t *scales, int64_t row, int dim, const float (&y)[8]) const {
        if constexpr (VEC) {
            if (e >= dim) return;
            const Scale8 s = scale_of(quad_max(max_abs8(y)));
            *reinterpret_cast<uint2 *>(codes + row + e) = make_uint2(codes4(y, s.inv), codes4(y + 4, s.inv));
            if ((e & 31) == 0) scales[(row + e) >> 5] = (uint16_t) s.bits;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (e + j * T >= dim) break;
                const Scale8 s = scale_of(half_max(__builtin_fabsf(y[j])));
                codes[row + e + j * T] = (int8_t) code1(y[j], s.inv);
                if (((e + j * T) & 31) == 0) scales[(row + e + j * T) >> 5] = (uint16_t) s.bits;
            }
        }
    }
};

// Threads of a workgroup: teams of one wave share one.
constexpr int norm_threads(int t) { return t == 64 ? 256 : t; }

template <int T, int NV, bool VEC>
__global__ __launch_bounds__(norm_threads(T)) void norm_kernel(NormParams p) {
    constexpr int TEAMS = norm_threads(T) / T;
    using E = Eight<T, VEC>;
    const int t = threadIdx.x % T;
    const int64_t r = (int64_t) blockIdx.x * TEAMS + threadIdx.x / T;
    if (TEAMS > 1 && r >= p.n_rows) return;  // (teams of one wave meet at no barrier)
    Raw8 rx[NV], rr[NV], rw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const E e(i, t);
        rx[i] = e.load(p.x, r * p.x_stride, p.dim, p.type);
        if (p.res) rr[i] = e.load(p.res, r * p.res_stride, p.dim, p.res_type);
        rw[i] = e.load(p.w, 0, p.dim, p.w_type);
    }
    float h[NV][8], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        E::widen(rx[i], p.type, h[i]);
        if (p.res) {
            float b[8];
            E::widen(rr[i], p.res_type, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = round_to(h[i][j] + b[j], p.res_type);
            E(i, t).store(p.res, r * p.res_stride, p.dim, h[i], p.res_type);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(h[i][j], h[i][j], sum);
    }
    sum = wave_total(sum);
    if constexpr (T > 64) {
        __shared__ float s_sum[T / 64];
        if ((t & 63) == 0) s_sum[t >> 6] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) sum += s_sum[i];
    }
    const float inv = 1.0f / __builtin_sqrtf(sum / (float) p.dim + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const E e(i, t);
        float w[8], y[8];
        E::widen(rw[i], p.w_type, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = h[i][j] * inv * w[j];
        if (p.out) e.store(p.out, r * p.out_stride, p.dim, y, p.out_type);
        if (p.codes) e.store_codes(p.codes, p.scales, r * p.dim, p.dim, y);
    }
}

// Rows in 8 bits without a norm: a thread eight neighbours.
template <bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeParams p, FastDiv div_row) {
    const uint32_t per = (uint32_t) p.cols / 8;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= per * (uint32_t) p.n_rows) return;  // (whole quads: cols is a multiple of 32)
    const uint32_t r = div_row.div(i);
    const int e = (int) (i - r * per) * 8;
    float y[8];
    if constexpr (VEC) {
        widen8(load_raw8(p.x, r * p.stride + e, p.type), p.type, y);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = load1(p.x, r * p.stride + e + j, p.type);
    }
    const Scale8 s = scale_of(quad_max(max_abs8(y)));
    *reinterpret_cast<uint2 *>(p.codes + (int64_t) i * 8) = make_uint2(codes4(y, s.inv), codes4(y + 4, s.inv));
    if ((threadIdx.x & 3) == 0) p.scales[i >> 2] = (uint16_t) s.bits;
}

// Whether eight elements from any multiple of 8 on are aligned for 16-byte pieces.
bool wide(const void *p, int64_t stride, int type) {
    return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * type_bytes(type) % 16 == 0);
}

template <int T, int NV, bool VEC>
hipError_t run_norm(const NormParams &p, hipStream_t stream) {
    constexpr int TEAMS = norm_threads(T) / T;
    NormParams q = p;
    void *args[] = {&q};
    return hipLaunchKernel(reinterpret_cast<const void *>(norm_kernel<T, NV, VEC>),
                           dim3((unsigned) ((p.n_rows + TEAMS - 1) / TEAMS)), dim3(norm_threads(T)), args, 0, stream);
}

// One step a thread as far as a workgroup goes: 4096 elements in 512 threads 3.3 us
// for one row and 3.7 for 64 (fp32, residual, both outputs), in 256 x 2 steps 4.6
// and 5.1, in 64 x 8 12.3 and 13.5; 6000 rows the same but for 64 threads.  8192
// elements in 1024 x 1 or 512 x 2: 3.8 and 4.9 us for one row, 5.8 and 6.6 for 200
// (bf16 into an fp32 residual, 8-bit rows), 21.3 and 19.4 for 1000, 50.3 and 46.5 for
// 3000, but all in fp16 32.7 and 35.6: the rule stays with few rows.
template <bool VEC>
hipError_t pick_norm(const NormParams &p, hipStream_t stream) {
    const int octets = (p.dim + 7) / 8;
    if (octets <= 64) return run_norm<64, 1, VEC>(p, stream);
    if (octets <= 128) return run_norm<128, 1, VEC>(p, stream);
    if (octets <= 256) return run_norm<256, 1, VEC>(p, stream);
    if (octets <= 512) return run_norm<512, 1, VEC>(p, stream);
    if (octets <= 1024) return run_norm<1024, 1, VEC>(p, stream);
    if (octets <= 2048) return run_norm<1024, 2, VEC>(p, stream);
    return run_norm<1024, 4, VEC>(p, stream);
}

}  // namespace

hipError_t launch_norm(const NormParams &p, hipStream_t stream) {
    const bool vec = p.dim % 8 == 0 && wide(p.x, p.x_stride, p.type) && wide(p.res, p.res_stride, p.res_type) &&
                     wide(p.w, 0, p.w_type) && wide(p.out, p.out_stride, p.out_type);
    return vec ? pick_norm<true>(p, stream) : pick_norm<false>(p, stream);
}

hipError_t launch_quantize_rows(const QuantizeParams &p, hipStream_t stream) {
    QuantizeParams q = p;
    FastDiv div = make_fastdiv((uint32_t) p.cols / 8);
    void *args[] = {&q, &div};
    const bool vec = wide(p.x, p.stride, p.type);
    const int64_t octets = (int64_t) p.n_rows * (p.cols / 8);
    return hipLaunchKernel(vec ? reinterpret_cast<const void *>(quantize_rows_kernel<true>)
                               : reinterpret_cast<const void *>(quantize_rows_kernel<false>),
                           dim3((unsigned) ((octets + 255) / 256)), dim3(256), args, 0, stream);
}

}  // namespace bmo
