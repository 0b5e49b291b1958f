// RMS norm with the residual's addition whose rows come out in 8 bits, the
// same rows without a norm, and the values that such rows stand for
// (declarations: include/quant_studio.h).
#include <hip/hip_runtime.h>

#include "qs_device.h"
#include "qs_host.h"
#include "qs_launch_kernel.h"
#include "qs_rows.h"
#include "quant_studio.h"

namespace {

using namespace qsr;

struct NormArgs {
    const void* x;
    const void* residual;       // or null
    const float* weight;        // null: no norm, the rows as they are
    void* sum;                  // x + residual in the source type, or null
    int8_t* q;
    float* s;
    int64_t rows, k, stride, rstride;       // strides in values
    float eps;
};

// h = x + residual, u = h * w, and per 32 values a = max |u| / 127, codes
// rint(u / a), scale a / sqrt(mean(h^2) + eps).
// The row's factor 1 / sqrt(...) cancels in u / a, so the codes do not wait
// for the sum of squares: one pass over the row gives both, and only the K/32
// group steps are kept (in LDS, read back by the lane that wrote them) until
// the sum is known. P lanes share a row, eight values each at a time; four
// lanes make a group of 32. Many rows are bound by memory (8,191 x 2,560 bf16 with
// a residual, 149 MB read and written: 28 us, 5.3 TB/s, a copy's rate), a few by
// latency (a row of 2,560: 3.2 us).
// A NaN or an infinity makes its group's scale NaN, so its values are NaN, as
// the plain computation has them; an infinity's row has 1 / sqrt(inf) = 0 and
// its other groups 0.
template <int SRC, int P>
__global__ __launch_bounds__(P > 256 ? P : 256) void k_rms_norm_q8(NormArgs a) {
    extern __shared__ float steps[];
    constexpr int BLOCK = P > 256 ? P : 256, ROWS = BLOCK / P;
    const int lane = threadIdx.x % P, slot = threadIdx.x / P;
    const int64_t row = (int64_t)blockIdx.x * ROWS + slot;
    const bool live = row < a.rows;
    float* mine = steps + slot * (a.k / 32);
    float ss = 0.0f;
    if (live) {
        for (int64_t c = lane * 8; c < a.k; c += P * 8) {
            Eight<SRC> x, r;
            float h[8], u[8];
            load8<SRC>(a.x, row * a.stride + c, x);
            if (a.residual) load8<SRC>(a.residual, row * a.rstride + c, r);
            Eight<qs::SRC_F32> w;
            if (a.weight) load8<qs::SRC_F32>(a.weight, c, w);
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                h[i] = value8<SRC>(x, i);
                if (a.residual) h[i] += value8<SRC>(r, i);
                ss = __builtin_fmaf(h[i], h[i], ss);
                u[i] = a.weight ? h[i] * value8<qs::SRC_F32>(w, i) : h[i];
                const float m = fabsf(u[i]);
                top = m > top || m != m ? m : top;      // keeps a NaN
            }
            if (a.sum) store8<SRC>(a.sum, row * a.k + c, h);
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                const float m = __shfl_xor(top, o);
                top = m > top || m != m ? m : top;
            }
            const float step = top / 127.0f;
            const bool codes = step > 0.0f && step < __builtin_inff();
            uint32_t out[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                // a subnormal step is coarse: a quotient can pass 127
                const int v = codes ? (int)qs::clampf(rintf(u[i] / step), -127.0f, 127.0f) : 0;
                out[i >> 2] |= (uint32_t)(v & 255) << (8 * (i & 3));
            }
            *reinterpret_cast<uint2*>(a.q + row * a.k + c) = uint2{out[0], out[1]};
            if (lane % 4 == 0) mine[c / 32] = step;
        }
    }
    float f = 1.0f;
    if (a.weight) {     // the same for every lane
#pragma unroll
        for (int o = 1; o < (P < 64 ? P : 64); o *= 2) ss += __shfl_xor(ss, o);
        if constexpr (P > 64) {
            __shared__ float part[BLOCK / 64];
            if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = ss;
            __syncthreads();
            ss = 0.0f;
#pragma unroll
            for (int i = 0; i < P / 64; i++) ss += part[slot * (P / 64) + i];
        }
        f = 1.0f / sqrtf(ss / (float)a.k + a.eps);
    }
    if (live && lane % 4 == 0)
        for (int64_t c = lane * 8; c < a.k; c += P * 8) {
            const float step = mine[c / 32];
            // an infinite step stands for no values, with or without a norm
            a.s[row * (a.k / 32) + c / 32] = step < __builtin_inff() ? step * f : __builtin_nanf("");
        }
}

// the values q * s of 8-bit rows; 16 to a thread; bound by memory (8,191 x 2,560 to
// bf16, 65 MB: 12.5 us, 5.2 TB/s)
template <int DST>
__global__ __launch_bounds__(256) void k_q8_values(const int8_t* q, const float* s, void* dst, int64_t n16) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n16) return;
    const u32x4 c = reinterpret_cast<const u32x4*>(q)[i];
    const float sc = s[i >> 1];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)(int8_t)(c[2 * h + (j >> 2)] >> (8 * (j & 3))) * sc;
        store8<DST>(dst, 16 * i + 8 * h, v);
    }
}

// Rows of a launch: a wave to a row, the threads of a launch are under 2^32.
constexpr int64_t MOST_ROWS = INT64_C(1) << 24;

template <int SRC>
hipError_t launch_norm(const NormArgs& all, hipStream_t st) {
    // A wave per row where rows fill the 1,024 SIMDs several times (us with 64, 256
    // and 1,024 lanes, bf16 with a residual: 8,191 x 2,560 28, 31, 53; 4,096 x 1,024
    // 9.9, 11.7, 24.5), else a workgroup each (2,048 x 9,728 37, 28.5, 31; 1,024 x
    // 2,560 10.7, 8.0, 9.6), a large one where they are few and long (64 x 2,560 7.5,
    // 4.3, 3.8; 1 x 2,560 6.2, 3.8, 3.3; 333 x 1,024 5.0, 4.1, 4.3).
    const int p = all.rows >= 4096 ? 64 : all.rows <= 256 && all.k > 2048 ? 1024 : 256;
    const int rows = p > 256 ? 1 : 256 / p;
    const size_t lds = (size_t)rows * (all.k / 32) * 4;
    constexpr int64_t esz = SRC == qs::SRC_F32 ? 4 : 2;
    using qs_host::launch_kernel;
    for (int64_t first = 0; first < all.rows; first += MOST_ROWS) {
        NormArgs a = all;
        a.rows = all.rows - first < MOST_ROWS ? all.rows - first : MOST_ROWS;
        a.x = static_cast<const char*>(all.x) + first * all.stride * esz;
        if (all.residual) a.residual = static_cast<const char*>(all.residual) + first * all.rstride * esz;
        if (all.sum) a.sum = static_cast<char*>(all.sum) + first * all.k * esz;
        a.q = all.q + first * all.k;
        a.s = all.s + first * (all.k / 32);
        const dim3 grid((unsigned)((a.rows + rows - 1) / rows));
        const hipError_t e = p == 64    ? launch_kernel(k_rms_norm_q8<SRC, 64>, grid, dim3(256), lds, st, a)
                             : p == 256 ? launch_kernel(k_rms_norm_q8<SRC, 256>, grid, dim3(256), lds, st, a)
                                        : launch_kernel(k_rms_norm_q8<SRC, 1024>, grid, dim3(1024), lds, st, a);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

using qs_host::fail;

namespace {
constexpr int64_t kMaxValues = INT64_C(1) << 34, kMaxK = INT64_C(1) << 17, kMaxSpan = INT64_C(1) << 62;
bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }
}  // namespace

extern "C" {

int qs_rms_norm_q8(int src_type, const void* x, int64_t rows, int64_t k, int64_t x_row_stride_bytes,
                   const void* residual, int64_t residual_row_stride_bytes, const float* weight, float eps,
                   void* sum, int8_t* q, float* scales, void* hip_stream) {
    qs_host::clear_error();
    const int esz = src_type == QS_SRC_F32 ? 4 : (src_type == QS_SRC_F16 || src_type == QS_SRC_BF16) ? 2 : 0;
    if (!esz) return fail(QS_EINVAL, "unsupported source type %d (F32=0, F16=1, BF16=30)", src_type);
    if (rows < 0) return fail(QS_EINVAL, "rows %lld < 0", (long long)rows);
    if (k <= 0 || k % 32 || k > kMaxK)
        return fail(QS_EINVAL, "row length %lld is not a multiple of 32 in 32..%lld", (long long)k, (long long)kMaxK);
    if (rows > kMaxValues / k)
        return fail(QS_EINVAL, "%lld x %lld values exceed the 2^34 per call", (long long)rows, (long long)k);
    if (rows == 0) return 0;
    if (!x || !q || !scales) return fail(QS_EINVAL, "null x, q or scales");
    if (sum && !residual) return fail(QS_EINVAL, "a sum needs a residual");
    const int64_t strides[2] = {x_row_stride_bytes, residual ? residual_row_stride_bytes : x_row_stride_bytes};
    for (int64_t s : strides) {
        if (s < k * esz || s % 16)
            return fail(QS_EINVAL, "row stride %lld must be >= %lld and a multiple of 16", (long long)s,
                        (long long)(k * esz));
        if (rows > kMaxSpan / s)
            return fail(QS_EINVAL, "%lld rows of stride %lld bytes exceed a 2^62-byte span", (long long)rows,
                        (long long)s);
    }
    if (off16(x) || off16(residual) || off16(weight) || off16(sum) || off16(q) || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(QS_EINVAL, "x, residual, weight, sum and q must be 16-byte aligned, scales 4-byte");
    NormArgs a{x, residual, weight, sum, q, scales, rows, k, strides[0] / esz, strides[1] / esz, eps};
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = src_type == QS_SRC_F32   ? launch_norm<qs::SRC_F32>(a, st)
                         : src_type == QS_SRC_F16 ? launch_norm<qs::SRC_F16>(a, st)
                                                  : launch_norm<qs::SRC_BF16>(a, st);
    if (e != hipSuccess) return fail(QS_EIO, "rms_norm_q8: launch failed: %s", hipGetErrorString(e));
    return 0;
}

int qs_q8_values(const int8_t* q, const float* scales, int64_t rows, int64_t k, int dst_type, void* dst,
                 void* hip_stream) {
    qs_host::clear_error();
    if (dst_type != QS_SRC_F32 && dst_type != QS_SRC_F16 && dst_type != QS_SRC_BF16)
        return fail(QS_EINVAL, "unsupported destination type %d (F32=0, F16=1, BF16=30)", dst_type);
    if (rows < 0) return fail(QS_EINVAL, "rows %lld < 0", (long long)rows);
    if (k <= 0 || k % 32) return fail(QS_EINVAL, "row length %lld is not a positive multiple of 32", (long long)k);
    if (k > kMaxValues || rows > kMaxValues / k)
        return fail(QS_EINVAL, "%lld x %lld values exceed the 2^34 per call", (long long)rows, (long long)k);
    if (rows == 0) return 0;
    if (!q || !scales || !dst) return fail(QS_EINVAL, "null q, scales or dst");
    if (off16(q) || off16(dst) || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(QS_EINVAL, "q and dst must be 16-byte aligned, scales 4-byte");
    const int64_t n16 = rows * k / 16;
    const dim3 grid((unsigned)((n16 + 255) / 256));
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const auto kernel = dst_type == QS_SRC_F32   ? k_q8_values<qs::SRC_F32>
                        : dst_type == QS_SRC_F16 ? k_q8_values<qs::SRC_F16>
                                                 : k_q8_values<qs::SRC_BF16>;
    const hipError_t e = qs_host::launch_kernel(kernel, grid, dim3(256), 0, st, q, scales, dst, n16);
    if (e != hipSuccess) return fail(QS_EIO, "q8_values: launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // extern "C"
