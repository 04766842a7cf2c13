// C-ABI entry points of a layer's operators around a checkpoint's weights: norms, products with an epilogue, experts' products.
// Declarations and the per-function contract live in include/lmz_b200.h.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/lmz_b200.h"
#include "epilogue.cuh"
#include "norm_kernels.cuh"
#include "product_kernel.cuh"

using namespace lmz;

static_assert(MAX_EXPERTS == LMZ_GPU_MAX_EXPERTS && ACT_SILU == LMZ_GPU_ACT_SILU && ACT_GELU_TANH == LMZ_GPU_ACT_GELU_TANH);

#define API extern "C" __attribute__((visibility("default")))

#include "host_error.inl"
#include "host_device.inl"
#include "host_launch.inl"

// ------------------------------------------------------------------ norms

static int check_norm(const lmz_norm *p)
{
    const uint32_t e = element_bytes(p->dtype);
    if (!e || !element_bytes(p->weight_dtype)) return fail_msg(LMZ_GPU_EUNSUPPORTED, "an element type other than BF16, F16 and F32");
    if (p->weight_dtype != p->dtype && p->weight_dtype != LMZ_GPU_F32) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a norm's weight is of the tensors' type or F32");
    if (p->tokens >= 1ull << 31) return fail_msg(LMZ_GPU_EUNSUPPORTED, "2^31 tokens and more");
    if (p->dim == 0 || p->dim >= 1ull << 24) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a row has between 1 and 2^24 - 1 elements");
    if (!(p->eps >= 0) || p->eps > 3.4e38f) return fail_msg(LMZ_GPU_EUNSUPPORTED, "eps is a number and not below zero");
    return LMZ_GPU_OK;
}

// f(type tag, weight's type tag, vector width tag).  The weight's vectors have as many elements as the tensors', so that its address counts for the
// width as the tensors' would there.
template <class F>
static int by_norm_types(const lmz_norm *p, std::initializer_list<uint64_t> at, F f)
{
    const uint64_t e = element_bytes(p->dtype), wide = p->weight && p->weight_dtype != p->dtype ? 2 : 1;
    uint64_t bits = address(p->weight) / wide | (address(p->weight) & (wide - 1) ? 1 : 0);
    for (uint64_t v : at) bits |= v;
    return by_type(p->dtype, vector_bytes(p->dim * e, {bits}), [&](auto type, auto vec) {
        using T = decltype(type);
        if constexpr (!std::is_same_v<T, float>)
            if (p->weight_dtype == LMZ_GPU_F32) return f(type, float{}, vec);
        return f(type, T{}, vec);
    });
}

// How a block's threads share rows of so many vectors.
struct NormShape {
    uint32_t lane_log = 0, threads;
    bool is_long;
    NormShape(uint32_t vectors, uint32_t elements)
    {
        const uint32_t each = NORM_EACH / elements;
        while ((1u << lane_log) < NORM_MOST && (each << lane_log) < vectors) lane_log++;
        is_long = (each << lane_log) < vectors;
        threads = std::max(NORM_THREADS, 1u << lane_log);
    }
};

API int lmz_gpu_norm_dev(const lmz_norm *p, void *cuda_stream)
{
    int rc = check_norm(p);
    if (rc || p->tokens == 0) return rc;
    rc = device_ready();
    if (rc) return rc;
    if (!p->weight && !p->q) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a norm has a weight");
    const uint64_t e = element_bytes(p->dtype);
    return by_norm_types(p, {address(p->x), address(p->residual), address(p->y), address(p->stream), p->x_stride * e, p->residual ? p->residual_stride * e : 0, p->q ? address(p->q) * e : 0},
                         [&](auto type, auto weight_type, auto vec) {
        using T = decltype(type);
        using W = decltype(weight_type);
        constexpr int VB = sizeof(vec.raw), N = VB / sizeof(T);
        NormArgs a{};
        a.x = p->x, a.residual = p->residual, a.weight = p->weight, a.y = p->y, a.stream = p->stream, a.q = static_cast<uint8_t *>(p->q);
        a.scale = p->scale, a.rstd = p->rstd, a.tokens = p->tokens, a.dim = p->dim, a.x_stride = p->x_stride, a.residual_stride = p->residual_stride;
        a.vectors = static_cast<uint32_t>(p->dim / N), a.eps = p->eps;
        const NormShape shape(a.vectors, N);
        a.lane_log = shape.lane_log;
        const uint32_t per = shape.threads >> shape.lane_log;
        const dim3 grid(static_cast<unsigned>((p->tokens + per - 1) / per));
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        if (p->q) return launch("launch k_norm", shape.is_long ? k_norm<T, W, VB, true, true> : k_norm<T, W, VB, true, false>, grid, shape.threads, 0, cs, a);
        return launch("launch k_norm", shape.is_long ? k_norm<T, W, VB, false, true> : k_norm<T, W, VB, false, false>, grid, shape.threads, 0, cs, a);
    });
}

// Blocks of the gradients' kernel: the shares of the weight's gradient are read again, so no more of them than keep the multiprocessors busy.
constexpr uint32_t NORM_GRAD_BLOCKS = 4 * 148;
static uint64_t norm_grad_shares(const lmz_norm *p, const NormShape &shape)
{
    const uint32_t per = shape.threads >> shape.lane_log;
    return std::min<uint64_t>((p->tokens + per - 1) / per, NORM_GRAD_BLOCKS) * per;
}

API size_t lmz_gpu_norm_grad_work_bytes(const lmz_norm *p)
{
    // (whatever the vectors' width, a thread has NORM_EACH elements or fewer, and a block NORM_THREADS threads or one row's)
    const uint64_t row = std::min<uint64_t>(NORM_MOST, (p->dim + NORM_EACH - 1) / NORM_EACH);
    uint64_t lanes = 1;
    while (lanes < row) lanes *= 2;
    const uint64_t per = std::max<uint64_t>(1, NORM_THREADS / lanes);
    return std::min<uint64_t>((p->tokens + per - 1) / per, NORM_GRAD_BLOCKS) * per * p->dim * sizeof(float);
}

API int lmz_gpu_norm_grad_dev(const lmz_norm *p, void *cuda_stream)
{
    int rc = check_norm(p);
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    if (p->tokens == 0) {
        if (p->dweight) CK("cudaMemsetAsync", cudaMemsetAsync(p->dweight, 0, p->dim * element_bytes(p->weight_dtype), cs));
        return LMZ_GPU_OK;
    }
    if (!p->dx && !p->dweight) return LMZ_GPU_OK;
    const uint64_t e = element_bytes(p->dtype);
    return by_norm_types(p, {address(p->x), address(p->dy), address(p->dstream), address(p->dx), p->x_stride * e}, [&](auto type, auto weight_type, auto vec) {
        using T = decltype(type);
        using W = decltype(weight_type);
        constexpr int VB = sizeof(vec.raw), N = VB / sizeof(T);
        NormGradArgs a{};
        a.s = p->x, a.weight = p->weight, a.dy = p->dy, a.ds = p->dstream, a.rstd = p->rstd, a.dx = p->dx;
        a.partial = p->dweight ? static_cast<float *>(p->work) : nullptr;
        a.tokens = p->tokens, a.dim = p->dim, a.s_stride = p->x_stride, a.vectors = static_cast<uint32_t>(p->dim / N);
        const NormShape shape(a.vectors, N);
        a.lane_log = shape.lane_log;
        const uint64_t shares = norm_grad_shares(p, shape);
        const dim3 grid(static_cast<unsigned>(shares / (shape.threads >> shape.lane_log)));
        int failed = launch("launch k_norm_grad", shape.is_long ? k_norm_grad<T, W, VB, true> : k_norm_grad<T, W, VB, false>, grid, shape.threads, 0, cs, a);
        if (!failed && p->dweight)
            failed = launch("launch k_join", k_join<W>, dim3(static_cast<unsigned>((p->dim + 31) / 32)), 32 * JOIN_WARPS, 0, cs, static_cast<const float *>(a.partial),
                            shares, p->dim, static_cast<W *>(p->dweight));
        return failed;
    });
}

// ------------------------------------------------------------------ products

static int check_product(const lmz_product *p)
{
    if (p->dtype != LMZ_GPU_BF16 && p->dtype != LMZ_GPU_F16 && p->dtype != LMZ_GPU_E4M3) return fail_msg(LMZ_GPU_EUNSUPPORTED, "products are of BF16, F16 or E4M3");
    if (p->result_dtype != LMZ_GPU_BF16 && p->result_dtype != LMZ_GPU_F16) return fail_msg(LMZ_GPU_EUNSUPPORTED, "results are of BF16 or F16");
    if (p->dtype != LMZ_GPU_E4M3 && p->result_dtype != p->dtype) return fail_msg(LMZ_GPU_EUNSUPPORTED, "the result of a product of 16-bit tensors is of their type");
    if (p->dtype == LMZ_GPU_E4M3 && (p->offsets || !p->x_scale || !p->weight_scale)) return fail_msg(LMZ_GPU_EUNSUPPORTED, "products in 8 bits have scales, and no experts");
    if (p->offsets && p->offset_bytes != 4 && p->offset_bytes != 8) return fail_msg(LMZ_GPU_EUNSUPPORTED, "offsets are int32 or int64");
    if (p->experts == 0 || p->experts > MAX_EXPERTS) return report(LMZ_GPU_EUNSUPPORTED, "between 1 and %d experts", (int)MAX_EXPERTS);
    if (!p->offsets && p->experts != 1) return fail_msg(LMZ_GPU_EUNSUPPORTED, "several experts without offsets");
    if (p->in == 0 || p->out == 0 || p->in >= 1u << 21 || p->out >= 1u << 21)
        return fail_msg(LMZ_GPU_EUNSUPPORTED, "a weight has between 1 and 2^21 - 1 rows and columns");
    if (p->rows >= 1ull << 31) return fail_msg(LMZ_GPU_EUNSUPPORTED, "2^31 rows and more");
    if (p->activation >= ACT_COUNT) return fail_msg(LMZ_GPU_EUNSUPPORTED, "an activation that there is not");
    return LMZ_GPU_OK;
}

static Groups groups_of(const lmz_product *p) { return {p->offsets, p->experts, p->offset_bytes == 8, p->rows}; }

// What a product's kernels leave each other.
struct ProductLayout {
    uint64_t dz, partial, end = 0;
    bool epilogue;                               // dz is not dy
    ProductLayout(const lmz_product *p, bool grad)
    {
        auto take = [&](bool on, uint64_t bytes) {
            const uint64_t r = end;
            if (on) end += up256(bytes);
            return r;
        };
        epilogue = p->activation != ACT_NONE || p->times;
        dz = take(grad && epilogue, p->rows * p->out * 2);
        partial = take(grad && p->dbias, ((p->rows + EG_ROWS - 1) / EG_ROWS + p->experts) * p->out * 4);
    }
};

API size_t lmz_gpu_product_work_bytes(const lmz_product *p, int grad) { return ProductLayout(p, grad).end; }

template <class T, class O>
static int launch_product(const ProductArgs<T> &a, cudaStream_t cs)
{
    const dim3 grid(static_cast<unsigned>((a.feats + S_TILE - 1) / S_TILE), static_cast<unsigned>(std::min<uint64_t>(1024, (a.cols + S_TILE - 1) / S_TILE)),
                    std::min(64u, a.groups.count));
    return launch("launch k_product", k_product<T, O>, grid, S_THREADS, 0, cs, a);
}

template <class T, class O>
static int product_as(const lmz_product *p, cudaStream_t cs)
{
    ProductArgs<T> a{};
    a.a = static_cast<const T *>(p->weight), a.b = static_cast<const T *>(p->x), a.out = p->y, a.z = p->z;
    a.bias = p->bias, a.times = p->times, a.residual = p->residual, a.a_scale = p->weight_scale, a.b_scale = p->x_scale;
    a.groups = groups_of(p), a.feats = p->out, a.cols = p->rows, a.depth = p->in;
    a.a_f = p->weight_stride, a.a_k = 1, a.b_c = p->x_stride, a.b_k = 1, a.a_plane = p->weight_plane;
    a.times_stride = p->times_stride, a.residual_stride = p->residual_stride, a.activation = p->activation;
    return launch_product<T, O>(a, cs);
}

template <class T>
static int launch_epilogue_grad(const lmz_product *p, const ProductLayout &l, void *dz, cudaStream_t cs)
{
    const uint64_t chunks = (p->rows + EG_ROWS - 1) / EG_ROWS;
    float *partial = p->dbias ? reinterpret_cast<float *>(static_cast<uint8_t *>(p->work) + l.partial) : nullptr;
    int rc = by_width<T>(vector_bytes(p->out * 2, {address(p->dy), address(p->z) / 2, address(p->times), p->times ? p->times_stride * 2 : 0, address(p->dtimes)}), [&](auto vec) {
        constexpr int VB = sizeof(vec.raw);
        EpilogueGradArgs a{};
        a.dy = p->dy, a.z = p->z, a.times = p->times, a.dz = dz, a.dtimes = p->dtimes, a.partial = partial, a.groups = groups_of(p);
        a.rows = p->rows, a.out = a.dz_stride = p->out, a.times_stride = p->times_stride, a.vectors = static_cast<uint32_t>(p->out * 2 / VB), a.activation = p->activation;
        return launch("launch k_epilogue_grad", k_epilogue_grad<T, VB>, dim3(static_cast<unsigned>(chunks), (a.vectors + EG_THREADS - 1) / EG_THREADS), EG_THREADS, 0, cs, a);
    });
    if (!rc && p->dbias)
        rc = launch("launch k_bias_join", k_bias_join<T>, dim3(static_cast<unsigned>((p->out + 31) / 32), p->experts), 256, 0, cs, static_cast<const float *>(partial),
                    groups_of(p), p->out, static_cast<T *>(p->dbias));
    return rc;
}

template <class T>
static int product_grad_as(const lmz_product *p, cudaStream_t cs)
{
    if (p->rows == 0) {
        if (p->dweight) CK("cudaMemsetAsync", cudaMemsetAsync(p->dweight, 0, 2ull * p->experts * p->out * p->in, cs));
        if (p->dbias) CK("cudaMemsetAsync", cudaMemsetAsync(p->dbias, 0, 2ull * p->experts * p->out, cs));
        return LMZ_GPU_OK;
    }
    const ProductLayout l(p, true);
    T *own = l.epilogue ? reinterpret_cast<T *>(static_cast<uint8_t *>(p->work) + l.dz) : nullptr;
    if (l.epilogue || p->dbias) {
        const int rc = launch_epilogue_grad<T>(p, l, own, cs);
        if (rc) return rc;
    }
    const T *dz = own ? own : static_cast<const T *>(p->dy), *w = static_cast<const T *>(p->weight), *x = static_cast<const T *>(p->x);
    ProductArgs<T> a{};
    a.groups = groups_of(p), a.feats = p->in;
    if (p->dx) {
        a.a = w, a.b = dz, a.out = p->dx, a.cols = p->rows, a.depth = p->out;
        a.a_f = 1, a.a_k = p->weight_stride, a.b_c = p->out, a.b_k = 1, a.a_plane = p->weight_plane;
        const int rc = launch_product<T, T>(a, cs);
        if (rc) return rc;
    }
    if (p->dweight) {
        a.a = x, a.b = dz, a.out = p->dweight, a.cols = p->out, a.depth = p->rows, a.by_k = true;
        a.a_f = 1, a.a_k = p->x_stride, a.b_c = 1, a.b_k = p->out, a.a_plane = 0;
        return launch_product<T, T>(a, cs);
    }
    return LMZ_GPU_OK;
}

API int lmz_gpu_product_dev(const lmz_product *p, void *cuda_stream)
{
    int rc = check_product(p);
    if (rc || p->rows == 0) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    if (p->dtype == LMZ_GPU_E4M3)
        return p->result_dtype == LMZ_GPU_BF16 ? product_as<__nv_fp8_e4m3, __nv_bfloat16>(p, cs) : product_as<__nv_fp8_e4m3, __half>(p, cs);
    return p->dtype == LMZ_GPU_BF16 ? product_as<__nv_bfloat16, __nv_bfloat16>(p, cs) : product_as<__half, __half>(p, cs);
}

API int lmz_gpu_product_grad_dev(const lmz_product *p, void *cuda_stream)
{
    int rc = check_product(p);
    if (!rc && p->dtype == LMZ_GPU_E4M3) rc = fail_msg(LMZ_GPU_EUNSUPPORTED, "products in 8 bits have no gradients");
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    return p->dtype == LMZ_GPU_BF16 ? product_grad_as<__nv_bfloat16>(p, cs) : product_grad_as<__half>(p, cs);
}
