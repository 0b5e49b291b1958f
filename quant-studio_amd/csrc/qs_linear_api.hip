// C ABI of the products with packed weights: argument checks, the adapters'
// first product and the dispatch over formats (declarations:
// include/quant_studio.h).
#include <hip/hip_runtime.h>

#include "qs_host.h"
#include "qs_launch_kernel.h"
#include "qs_linear.h"
#include "qs_linear_kernels.h"

namespace {

using qs_host::fail;
using qsl::LinearArgs;

struct ShrinkArgs {
    const int8_t* q;
    const float* s;
    const uint16_t* a;          // adapter i: rows off[i] .. off[i + 1] of k
    const int32_t *ids, *off;
    const float* scales;
    float* v;
    int64_t k, ldv;
    int32_t adapters;
    int type;
};

// v[t, r] = scale * sum over k of A[r, k] x[t, k] for the adapter of row t:
// a workgroup per row and 16 ranks, four to a wave.
__global__ __launch_bounds__(256) void k_adapter_rows(ShrinkArgs a) {
    const int64_t t = blockIdx.x;
    const int id = a.ids[t];
    if (id < 0 || id >= a.adapters) return;
    const int o = a.off[id], rank = a.off[id + 1] - o;
    const int r0 = blockIdx.y * 16 + threadIdx.x / 64 * 4, lane = threadIdx.x % 64;
    if (r0 >= rank) return;         // the ranks are multiples of 8: four rows or none
    const uint16_t* rows = a.a + (int64_t)(o + r0) * a.k;
    float sum[4] = {};
    for (int64_t c = lane * 8; c < a.k; c += 512) {
        const uint2 x = *reinterpret_cast<const uint2*>(a.q + t * a.k + c);
        const float s = a.s[t * (a.k / 32) + c / 32];
        float xv[8];
#pragma unroll
        for (int i = 0; i < 8; i++) xv[i] = (float)(int8_t)((i < 4 ? x.x : x.y) >> (8 * (i & 3)));
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint4 w = *reinterpret_cast<const uint4*>(rows + r * a.k + c);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
            float p = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++)
                p = __builtin_fmaf(xv[i], qsl::value16((ww[i >> 1] >> (16 * (i & 1))) & 0xffffu, a.type), p);
            sum[r] = __builtin_fmaf(s, p, sum[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int d = 1; d < 64; d *= 2) sum[r] += __shfl_xor(sum[r], d);
    if (lane < 4) a.v[t * a.ldv + r0 + lane] = a.scales[id] * (lane < 2 ? (lane ? sum[1] : sum[0]) : lane == 2 ? sum[2] : sum[3]);
}

template <int TYPE>
constexpr int64_t row_bytes_of(int64_t k) {
    return k % qsl::Format<TYPE>::BLK ? -1 : k / qsl::Format<TYPE>::BLK * qsl::Format<TYPE>::BYTES;
}

struct Entry {
    int type;
    hipError_t (*launch)(const LinearArgs&, void*, hipStream_t);
    int64_t (*row_bytes)(int64_t);
    int block_bytes;
};
#define QS_ENTRY(T) {T, qsl::launch_linear<T>, row_bytes_of<T>, qsl::Format<T>::BYTES}
constexpr Entry kEntries[] = {
    QS_ENTRY(QS_TYPE_Q4_0), QS_ENTRY(QS_TYPE_Q4_1), QS_ENTRY(QS_TYPE_Q5_0), QS_ENTRY(QS_TYPE_Q5_1),
    QS_ENTRY(QS_TYPE_Q8_0), QS_ENTRY(QS_TYPE_IQ4_NL), QS_ENTRY(QS_TYPE_Q2_K), QS_ENTRY(QS_TYPE_Q3_K),
    QS_ENTRY(QS_TYPE_Q4_K), QS_ENTRY(QS_TYPE_Q5_K), QS_ENTRY(QS_TYPE_Q6_K), QS_ENTRY(QS_TYPE_IQ4_XS),
    QS_ENTRY(QS_TYPE_IQ2_XXS), QS_ENTRY(QS_TYPE_IQ2_XS), QS_ENTRY(QS_TYPE_IQ2_S), QS_ENTRY(QS_TYPE_IQ3_XXS),
    QS_ENTRY(QS_TYPE_IQ3_S),
};

bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }
bool off4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0; }
constexpr int64_t kMaxValues = INT64_C(1) << 34, kMaxRows = INT64_C(1) << 24, kMaxRank = 4096;

const Entry* find(int type) {
    for (const Entry& c : kEntries)
        if (c.type == type) return &c;
    return nullptr;
}

int bad_sizes(const Entry& e, int64_t n, int64_t k, int64_t t) {
    if (n < 0 || t < 0 || t > kMaxRows) return fail(QS_EINVAL, "n %lld, t %lld: negative, or t over 2^24", (long long)n, (long long)t);
    if (k <= 0 || k > kMaxRows || e.row_bytes(k) < 0)
        return fail(QS_EINVAL, "row length %lld is not a positive multiple of the type's block, or over 2^24", (long long)k);
    if (n > kMaxValues / k || t > kMaxValues / k || (n && t > kMaxValues / n))
        return fail(QS_EINVAL, "%lld x %lld with %lld rows: over 2^34 values", (long long)n, (long long)k, (long long)t);
    return 0;
}

// the rows' products with the adapters' A, then the factors as laid out
int64_t adapter_bytes(int64_t t, int max_rank) { return (t * max_rank * 4 + 255) / 256 * 256; }
int64_t workspace_of(int type, int64_t n, int64_t k, int64_t t, int max_rank) {
    if (n == 0 || t == 0) return 0;
    int64_t bytes = adapter_bytes(t, max_rank);
    if (qsl::takes_matrix(t)) {
        const qsl::MatrixPlan p = qsl::matrix_plan(type, n, k, t);
        bytes += p.x_bytes + p.w_bytes;
    }
    return bytes;
}

}  // namespace

extern "C" {

int64_t qs_packed_linear_workspace(int ggml_type, int64_t n, int64_t k, int64_t t, int max_rank) {
    qs_host::clear_error();
    const Entry* e = find(ggml_type);
    if (!e) return fail(QS_ENOTSUP, "unknown ggml type %d", ggml_type);
    const int bad = bad_sizes(*e, n, k, t);
    if (bad) return bad;
    if (max_rank < 0 || max_rank > kMaxRank || max_rank % 8)
        return fail(QS_EINVAL, "max_rank %d must be a multiple of 8 in 0..%lld", max_rank, (long long)kMaxRank);
    return workspace_of(ggml_type, n, k, t, max_rank);
}

int qs_packed_linear(int ggml_type, const void* weight, int64_t n, int64_t k, const int8_t* q, const float* scales,
                     int64_t t, int dst_type, void* dst, int64_t dst_bytes, const qs_adapters* adapters,
                     const int32_t* ids, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    qs_host::clear_error();
    const Entry* e = find(ggml_type);
    if (!e) return fail(QS_ENOTSUP, "unknown ggml type %d", ggml_type);
    const int esz = dst_type == QS_SRC_F32 ? 4 : (dst_type == QS_SRC_F16 || dst_type == QS_SRC_BF16) ? 2 : 0;
    if (!esz) return fail(QS_EINVAL, "unsupported destination type %d (F32=0, F16=1, BF16=30)", dst_type);
    const int bad = bad_sizes(*e, n, k, t);
    if (bad) return bad;
    if (n == 0 || t == 0) return 0;
    if (!weight || !q || !scales || !dst) return fail(QS_EINVAL, "null weight, q, scales or dst");
    if (off16(q) || off4(scales) || reinterpret_cast<uintptr_t>(dst) % esz ||
        reinterpret_cast<uintptr_t>(weight) % (e->block_bytes % 4 ? 2 : 4))
        return fail(QS_EINVAL, "q must be 16-byte aligned, scales 4-byte, dst by its type, weight 4-byte (2-byte where "
                               "the type's blocks are not whole words)");
    if (dst_bytes < n * t * esz)
        return fail(QS_EINVAL, "dst holds %lld bytes, %lld needed", (long long)dst_bytes, (long long)(n * t * esz));
    LinearArgs a{};
    a.w = static_cast<const uint8_t*>(weight);
    a.q = q;
    a.s = scales;
    a.dst = dst;
    a.row_bytes = e->row_bytes(k);
    a.n = n;
    a.k = k;
    a.t = t;
    a.dst_type = dst_type;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if ((adapters != nullptr) != (ids != nullptr)) return fail(QS_EINVAL, "adapters and ids go together");
    const bool adapted = adapters && adapters->count > 0 && adapters->max_rank > 0;
    const int rank = adapted ? adapters->max_rank : 0;
    if (adapted) {
        if (adapters->type != QS_SRC_F16 && adapters->type != QS_SRC_BF16)
            return fail(QS_EINVAL, "unsupported adapter type %d (F16=1, BF16=30)", adapters->type);
        if (adapters->max_rank > kMaxRank || adapters->max_rank % 8)
            return fail(QS_EINVAL, "max_rank %d must be a multiple of 8 in 0..%lld", adapters->max_rank,
                        (long long)kMaxRank);
        if (!adapters->a || !adapters->b || !adapters->offsets || !adapters->scales)
            return fail(QS_EINVAL, "null adapter a, b, offsets or scales");
        if (off16(adapters->a) || off16(adapters->b) || off4(ids))
            return fail(QS_EINVAL, "adapter a and b must be 16-byte aligned, ids 4-byte");
    }
    const int64_t need = workspace_of(ggml_type, n, k, t, rank);
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < need))
        return fail(QS_EINVAL, "workspace holds %lld bytes at %p, %lld needed, 256-byte aligned",
                    (long long)workspace_bytes, workspace, (long long)need);
    if (adapted) {
        a.ids = ids;
        a.off = adapters->offsets;
        a.b = static_cast<const uint16_t*>(adapters->b);
        a.b_type = adapters->type;
        a.v = static_cast<const float*>(workspace);
        a.ldv = adapters->max_rank;
        a.adapters = adapters->count;
        const ShrinkArgs s{q, scales, static_cast<const uint16_t*>(adapters->a), ids, adapters->offsets,
                           adapters->scales, static_cast<float*>(workspace), k, a.ldv, a.adapters, a.b_type};
        const hipError_t r = qs_host::launch_kernel(k_adapter_rows, dim3((unsigned)t, (unsigned)((a.ldv + 15) / 16)),
                                                    dim3(256), 0, st, s);
        if (r != hipSuccess) return fail(QS_EIO, "packed_linear: launch failed: %s", hipGetErrorString(r));
    }
    void* layouts = static_cast<uint8_t*>(workspace) + adapter_bytes(t, rank);
    const hipError_t r = e->launch(a, layouts, st);
    if (r != hipSuccess) return fail(QS_EIO, "packed_linear: launch failed: %s", hipGetErrorString(r));
    return 0;
}

}  // extern "C"
