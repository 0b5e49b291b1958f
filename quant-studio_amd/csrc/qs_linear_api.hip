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

// bytes of a result's value; `dst`: QS_SRC_*, alone or with QS_EXACT
int dst_size(int dst) {
    const int type = dst & ~QS_EXACT;
    return type == QS_SRC_F32 ? 4 : (type == QS_SRC_F16 || type == QS_SRC_BF16) ? 2 : 0;
}

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

// The workspace: what the adapters' products leave for the weight's, then the
// factors as laid out.
struct Work {
    int64_t v, delta, lo, rest, unit, layouts, sums, bytes; // offsets; v is hi where there is a lo, sums a split product's
    int splits, parts;
    bool few, f16;
};
Work work_of(int type, int64_t row_bytes, int dst, int64_t n, int64_t k, int64_t t, int max_rank) {
    using qsl::round_up;
    Work w{};
    if (n == 0 || t == 0) return w;
    const bool matrix = qsl::takes_matrix(t, n, k), few = qsl::takes_few(row_bytes, t, k);
    w.few = few;
    const bool f16 = w.f16 = qsl::takes_f16(dst, t, n, k);
    if (max_rank > 0 && matrix) {
        w.lo = round_up(t * max_rank * 2, 256);
        w.rest = 2 * w.lo;
        w.unit = w.rest + (f16 ? 0 : w.lo);
        w.layouts = w.unit + round_up(t * ((max_rank + 31) / 32) * 4, 256);
        w.parts = qsl::adapter_parts(t, k, max_rank);
    } else if (max_rank > 0) {
        w.delta = round_up(t * max_rank * 4, 256);
        w.layouts = w.delta + (few ? 0 : round_up(t * n * 4, 256));
    }
    const qsl::MatrixPlan plan = qsl::matrix_plan(type, f16, n, k, t);
    w.splits = f16                                ? qsl::choose16(max_rank > 0, t, n, k, plan.slice < n ? 1 : qsl::MOST_PARTS).splits
               : matrix || few ? 1
                                                  : qsl::tile_splits(t, n, k);
    w.sums = w.layouts + (matrix ? qsl::round_up(plan.bytes(), 256) : 0);
    w.bytes = w.sums + (w.splits > 1 ? w.splits * t * n * 4 : 0);
    // the adapters' sums are read before the layouts are written, in their place
    const int64_t adapted = w.layouts + w.parts * t * max_rank * 4;
    w.bytes = w.bytes > adapted ? w.bytes : adapted;
    return w;
}

}  // namespace

extern "C" {

int64_t qs_packed_linear_workspace(int ggml_type, int64_t n, int64_t k, int64_t t, int dst_type, int max_rank) {
    qs_host::clear_error();
    const Entry* e = find(ggml_type);
    if (!e) return fail(QS_ENOTSUP, "unknown ggml type %d", ggml_type);
    const int bad = bad_sizes(*e, n, k, t);
    if (bad) return bad;
    if (max_rank < 0 || max_rank > kMaxRank || max_rank % 8)
        return fail(QS_EINVAL, "max_rank %d must be a multiple of 8 in 0..%lld", max_rank, (long long)kMaxRank);
    if (!dst_size(dst_type))
        return fail(QS_EINVAL, "unsupported destination type %d (F32=0, F16=1, BF16=30)", dst_type);
    return work_of(ggml_type, e->row_bytes(k), dst_type, n, k, t, max_rank).bytes;
}

int qs_packed_linear(int ggml_type, const void* weight, int64_t n, int64_t k, const int8_t* q, const float* scales,
                     int64_t t, int dst_type, void* dst, int64_t dst_bytes, const qs_adapters* adapters,
                     const int32_t* ids, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    qs_host::clear_error();
    const Entry* e = find(ggml_type);
    if (!e) return fail(QS_ENOTSUP, "unknown ggml type %d", ggml_type);
    const int esz = dst_size(dst_type);
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
    a.dst_type = dst_type & ~QS_EXACT;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    if ((adapters != nullptr) != (ids != nullptr)) return fail(QS_EINVAL, "adapters and ids go together");
    if (adapters && (adapters->count < 0 || adapters->max_rank < 0))
        return fail(QS_EINVAL, "adapter count %d or max_rank %d is negative", adapters->count, adapters->max_rank);
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
    const Work work = work_of(ggml_type, e->row_bytes(k), dst_type, n, k, t, rank);
    if (work.bytes && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < work.bytes))
        return fail(QS_EINVAL, "workspace holds %lld bytes at %p, %lld needed, 256-byte aligned",
                    (long long)workspace_bytes, workspace, (long long)work.bytes);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    if (adapted) {
        qsl::AdapterArgs s{};
        s.q = q;
        s.s = scales;
        s.a = static_cast<const uint16_t*>(adapters->a);
        s.b = static_cast<const uint16_t*>(adapters->b);
        s.ids = ids;
        s.off = adapters->offsets;
        s.scales = adapters->scales;
        s.k = k;
        s.n = n;
        s.t = t;
        s.ldv = rank;
        s.adapters = adapters->count;
        s.v = reinterpret_cast<float*>(base + work.v);
        s.delta = reinterpret_cast<float*>(base + work.delta);
        s.hi = reinterpret_cast<uint16_t*>(base + work.v);
        s.lo = reinterpret_cast<uint16_t*>(base + work.lo);
        s.rest = work.f16 ? nullptr : reinterpret_cast<uint16_t*>(base + work.rest);
        s.unit = reinterpret_cast<float*>(base + work.unit);
        s.sums = reinterpret_cast<float*>(base + work.layouts);
        s.parts = work.parts;
        s.few = work.few;
        const hipError_t r = qsl::launch_adapters(adapters->type, s, st);
        if (r != hipSuccess) return fail(QS_EIO, "packed_linear: launch failed: %s", hipGetErrorString(r));
        a.ids = ids;
        a.off = s.off;
        a.b = s.b;
        a.b_type = adapters->type;
        a.ldv = rank;
        a.adapters = s.adapters;
        if (qsl::takes_matrix(t, n, k)) a.v_hi = s.hi, a.v_lo = s.lo, a.v_rest = s.rest, a.v_unit = s.unit;
        else if (work.few) a.v = s.v;
        else a.delta = s.delta;
    }
    a.parts = reinterpret_cast<float*>(base + work.sums);
    a.splits = work.splits;
    a.f16 = work.f16;
    const hipError_t r = e->launch(a, base + work.layouts, st);
    if (r != hipSuccess) return fail(QS_EIO, "packed_linear: launch failed: %s", hipGetErrorString(r));
    return 0;
}

}  // extern "C"
