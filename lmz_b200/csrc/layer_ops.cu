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

// Where this source's kernels say that one has given up waiting (lmz_gpu_ops_gave_up).
__attribute__((visibility("hidden"))) int layer_gave_up_word(void **word)
{
    CK("cudaGetSymbolAddress", cudaGetSymbolAddress(word, g_gave_up));
    return LMZ_GPU_OK;
}

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
    NormShape(uint32_t vectors, uint32_t elements, uint32_t vector_bytes)
    {
        const uint32_t each = norm_each(vector_bytes) / elements;
        while ((1u << lane_log) < NORM_MOST && (each << lane_log) < vectors) lane_log++;
        is_long = (each << lane_log) < vectors;
        threads = std::max(NORM_THREADS, 1u << lane_log);
    }
};

API int lmz_gpu_norm_dev(const lmz_norm *p, void *cuda_stream)
{
    int rc = check_norm(p);
    if (rc || p->tokens == 0) return rc;
    if (!p->x || (!p->weight && !p->q)) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a norm has x and a weight");
    if (p->q ? p->y || !p->scale : !p->y) return fail_msg(LMZ_GPU_EUNSUPPORTED, "either y, or q and scale");
    rc = device_ready();
    if (rc) return rc;
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
        const NormShape shape(a.vectors, N, VB);
        a.lane_log = shape.lane_log;
        const uint32_t per = shape.threads >> shape.lane_log;
        const dim3 grid(static_cast<unsigned>((p->tokens + per - 1) / per));
        const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        auto run = [&](auto bits8) {
            constexpr bool B = decltype(bits8)::value;
            if (shape.is_long) return launch("launch k_norm", k_norm<T, W, VB, B, true, false>, grid, shape.threads, 0, cs, a);
            if constexpr (VB == 16)
                if (p->dim == norm_each(VB) << shape.lane_log && p->tokens % per == 0)
                    return launch("launch k_norm", k_norm<T, W, VB, B, false, true>, grid, shape.threads, 0, cs, a);
            return launch("launch k_norm", k_norm<T, W, VB, B, false, false>, grid, shape.threads, 0, cs, a);
        };
        return p->q ? run(std::true_type{}) : run(std::false_type{});
    });
}

// Blocks of the gradients' kernel: a share of the weight's gradient each, which are read again.  As many as there is room for (four of 256
// threads to a multiprocessor), and where there are few tokens, no more than have two turns each.
static uint64_t norm_grad_blocks(uint64_t tokens, uint32_t per)
{
    const uint64_t rows = (tokens + per - 1) / per;
    return std::min<uint64_t>(rows, std::max<uint64_t>(148, std::min<uint64_t>(4 * 148, (rows + 1) / 2)));
}

API size_t lmz_gpu_norm_grad_work_bytes(const lmz_norm *p)
{
    uint64_t most = 0;                           // (of wide and of narrow vectors: how many threads share a row goes by its elements alone)
    for (uint32_t vb : {16u, 8u}) {
        const NormShape shape(static_cast<uint32_t>(p->dim), 1, vb);
        most = std::max(most, norm_grad_blocks(p->tokens, shape.threads >> shape.lane_log));
    }
    return most * p->dim * sizeof(float);
}

API int lmz_gpu_norm_grad_dev(const lmz_norm *p, void *cuda_stream)
{
    int rc = check_norm(p);
    if (!rc && p->tokens && (!p->x || !p->weight || !p->rstd || !p->dy || (p->dweight && !p->work)))
        rc = fail_msg(LMZ_GPU_EUNSUPPORTED, "a norm's gradients go by x, its weight, rstd and dy, the weight's by a workspace, too");
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
        const NormShape shape(a.vectors, N, VB);
        a.lane_log = shape.lane_log;
        const uint64_t shares = norm_grad_blocks(p->tokens, shape.threads >> shape.lane_log);
        auto run = [&](auto kernel) { return launch("launch k_norm_grad", kernel, dim3(static_cast<unsigned>(shares)), shape.threads, 0, cs, a); };
        int failed;
        if (shape.is_long) failed = run(k_norm_grad<T, W, VB, true, NORM_MOST, false>);
        else if (shape.threads > NORM_THREADS) failed = run(k_norm_grad<T, W, VB, false, NORM_MOST, false>);
        else if (VB == 16 && p->dim == norm_each(VB) << shape.lane_log) failed = run(k_norm_grad<T, W, VB, false, NORM_THREADS, VB == 16>);
        else failed = run(k_norm_grad<T, W, VB, false, NORM_THREADS, false>);
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

// Rows that TMA takes as they lie: they start on 16 bytes.  (A single row has no next one.)
static bool in_place(const void *p, uint64_t bytes, uint64_t cols, uint64_t rows, uint64_t stride)
{
    return address(p) % 16 == 0 && (rows <= 1 ? cols * bytes % 16 == 0 : stride * bytes % 16 == 0 && stride >= cols);
}

static uint64_t up16(uint64_t n) { return (n + 15) & ~15ull; }

// What a product's kernels read in place of tensors that do not lie on boundaries, and leave each other.
struct ProductLayout {
    uint64_t x, w, dz, partial, most, end = 0;
    bool pack_x, pack_w, own_dz, powers;         // own_dz: dz is not dy, or does not lie where TMA takes it; powers: it is written times powers of two
    // Rows of a chunk of the epilogue's gradients: as few as give every multiprocessor blocks enough.
    static uint32_t chunk(const lmz_product *p)
    {
        uint32_t rows = EG_MOST_ROWS;
        while (rows > EG_LEAST_ROWS && p->rows * p->out < 1024ull * EG_THREADS * 8 * rows) rows /= 2;
        return rows;
    }
    ProductLayout(const lmz_product *p, bool grad)
    {
        auto take = [&](bool on, uint64_t bytes) {
            const uint64_t r = end;
            if (on) end += up256(bytes);
            return r;
        };
        const uint64_t e = p->dtype == LMZ_GPU_E4M3 ? 1 : 2;
        pack_x = !in_place(p->x, e, p->in, p->rows, p->x_stride);
        pack_w = !in_place(p->weight, e, p->in, p->out, p->weight_stride) || (p->experts > 1 && (p->weight_plane * e % 16 || p->weight_plane < p->out * (p->out <= 1 ? p->in : p->weight_stride)));
        own_dz = p->activation != ACT_NONE || p->times || !in_place(p->dy, 2, p->out, 2, p->out);
        x = take(pack_x && (!grad || p->dweight), p->rows * up16(p->in) * e);
        w = take(pack_w && (!grad || p->dx), p->experts * p->out * up16(p->in) * e);
        dz = take(grad && own_dz, p->rows * up8(p->out) * 2);
        partial = take(grad && p->dbias, ((p->rows + chunk(p) - 1) / chunk(p) + p->experts) * p->out * 4);
        powers = p->dtype == LMZ_GPU_F16 && (p->activation != ACT_NONE || p->times) && (p->dx || p->dweight);
        most = take(grad && powers, p->experts * 4ull);
    }
};

API size_t lmz_gpu_product_z_bytes(const lmz_product *p) { return p->rows * p->out * sizeof(float); }
API size_t lmz_gpu_product_work_bytes(const lmz_product *p, int grad) { return ProductLayout(p, grad).end; }

// x and the weight as the kernels take them: where they lie, or in the workspace (in one launch).
template <class T>
struct ProductInputs {
    const T *x, *w;
    uint64_t x_stride, w_stride, w_plane;
    int rc = LMZ_GPU_OK;
    ProductInputs(const lmz_product *p, const ProductLayout &l, bool want_x, bool want_w, cudaStream_t cs)
        : x(static_cast<const T *>(p->x)), w(static_cast<const T *>(p->weight)), x_stride(p->rows <= 1 ? p->in : p->x_stride),
          w_stride(p->out <= 1 ? p->in : p->weight_stride), w_plane(p->experts <= 1 ? p->out * w_stride : p->weight_plane)
    {
        using E = std::conditional_t<sizeof(T) == 1, uint8_t, uint16_t>;
        AlignArgs args{};
        uint32_t jobs = 0;
        uint64_t most = 0;
        const uint64_t pitch = up16(p->in);
        auto job = [&](const T *&t, uint64_t plane_stride, uint64_t stride, uint64_t rows, uint64_t planes, uint64_t off) {
            T *to = reinterpret_cast<T *>(static_cast<uint8_t *>(p->work) + off);
            args.job[jobs++] = {t, to, plane_stride, stride, rows, p->in, pitch, rows * planes};
            most = std::max(most, rows * planes * pitch * sizeof(T) / 16);
            t = to;
        };
        if (want_x && l.pack_x) job(x, 0, p->x_stride, p->rows, 1, l.x), x_stride = pitch;
        if (want_w && l.pack_w) job(w, p->weight_plane, p->weight_stride, p->out, p->experts, l.w), w_stride = pitch, w_plane = p->out * pitch;
        if (jobs) rc = launch("launch k_align", k_align<E>, dim3(static_cast<unsigned>(std::min<uint64_t>((most + ALIGN_THREADS - 1) / ALIGN_THREADS, 1u << 20)), jobs), ALIGN_THREADS, 0, cs, args);
    }
};

constexpr uint32_t PRODUCT_SMEM = 217u << 10;
static_assert(PRODUCT_SMEM + sizeof(ProductShared) <= 227u << 10);

template <class T, class O, int P, bool PAIR>
static int launch_product_as(ProductArgs &a, unsigned grid, cudaStream_t cs)
{
    static bool done[64];
    const int rc = opt_in_smem(k_product<T, O, P, PAIR>, PRODUCT_SMEM, done);
    if (rc) return rc;
    a.stage_bytes = product_stage_bytes(a.nt, PAIR, P == WEIGHT_GRAD);
    const uint32_t rest = ATOM_BYTES + G_EPILOGUE / 32 * G_TURN_BYTES;
    a.stages = std::min<uint32_t>(G_MAX_STAGES, (PRODUCT_SMEM - rest) / a.stage_bytes);
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(grid), G_THREADS, a.stages * a.stage_bytes + rest, cs, PAIR ? 2 : a.split, attrs);
    CK("launch k_product", cudaLaunchKernelEx(&c, k_product<T, O, P, PAIR>, a));
    return LMZ_GPU_OK;
}

// One of the three products: A, B and their strides; `a` has the rest.  `depth`: k, of all groups where it has them.
template <class T, class O, int P>
static int launch_product(ProductArgs &a, const T *at, uint64_t a_stride, uint64_t a_plane, const T *bt, uint64_t b_stride, uint64_t depth, cudaStream_t cs)
{
    constexpr bool by_k = P == WEIGHT_GRAD;
    constexpr uint32_t step_elements = ROW_BYTES / sizeof(T);
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    const uint64_t groups = a.groups.count, used = by_k ? groups : std::min<uint64_t>(groups, std::max<uint64_t>(a.cols, 1));
    // (tiles of columns: as many as groups that end anywhere have on average, half a tile more each, and no fewer than there can be)
    auto col_tiles = [&](uint64_t nt) { return by_k ? (a.cols + nt - 1) / nt * groups : groups == 1 ? (a.cols + nt - 1) / nt : std::max(used, a.cols / nt + used / 2); };
    auto most_tiles = [&](uint64_t nt) { return by_k ? (a.cols + nt - 1) / nt * groups : groups == 1 ? (a.cols + nt - 1) / nt : a.cols / nt + used; };
    const uint64_t rows_each = std::max<uint64_t>(1, a.cols / used);
    const uint64_t all_steps = by_k ? std::max<uint64_t>(1, (depth / groups + STEP_K - 1) / STEP_K) : (depth + step_elements - 1) / step_elements;
    // Tiles of 256 features by 160 to 256 columns by pairs of CTAs, or of 128 by 16 to 128 by one, or by a cluster that shares k: by what they are
    // reckoned to take (in 10 ns).  A step of a pair takes 0.3 us at 256 columns, of a CTA 0.19 whatever they are; what a tile takes beside its steps is a
    // pair's 2.6 us and more, a CTA's 0.04 a column; a cluster's meeting 1.4 us and more; the launch and the first tiles 6.  The way in and
    // out and clusters' meetings have become faster than that since, for all tiles alike: the order stands, the sums are two to nine us too many.  One B200, us, rows x in
    // x out, reckoned and measured: 4096x4096x4096 pairs of 256 93 (94), of 192 94 (94); 2048x4096x4096 pairs of 256 50 (46), 128 a CTA 75 (66); 512x4096x4096 pairs of 160
    // 22 (19), of 256 28 (24), 128 a CTA 23 (19); 200x4096x4096 128 by two CTAs 19 (17), by one 23 (19); 1x4096x4096 by four CTAs 11 (10), by two 14 (12), by one 19 (17);
    // the weight's gradient of 5000x256x256 by eight 13 (9), by four 14 (12), by two 18 (17).
    uint64_t best = ~0ull;
    bool pair = false;
    a.split = 1;
    auto consider = [&](bool p2, uint32_t nt, uint32_t split) {
        const uint64_t feats = (a.feats + (p2 ? 2 : 1) * G_FEATS - 1) / ((p2 ? 2 : 1) * G_FEATS), places = p2 ? sms / 2 : sms;
        const uint64_t n = feats * col_tiles(nt) * split;
        if (split > 1 && feats * most_tiles(nt) * split > places) return;
        const uint64_t waves = (n + places - 1) / places, steps = (all_steps + split - 1) / split;
        const uint64_t tile = p2 ? 30 * nt * steps / 256 + 516 - nt : 19 * steps + 4 * nt + (split == 1 ? 0 : 100 + 20 * split);
        const uint64_t cost = waves * tile + 600;
        if (cost < best) best = cost, pair = p2, a.nt = nt, a.split = split;
    };
    // (columns side by side come in blocks of 64, so that pairs of fewer than 256 of them load as much)
    const uint64_t wide = by_k ? a.cols : rows_each;
    for (uint32_t nt = by_k ? 64 : G_GROUP; nt <= 128; nt *= 2)
        for (uint32_t split = 1; split <= 8 && 2 * split <= std::max<uint64_t>(2, all_steps); split *= 2)
            if (nt == (by_k ? 64 : G_GROUP) || nt < 2 * wide) consider(false, nt, split);
    for (uint32_t nt = 256; nt >= (by_k ? 256 : 160); nt -= 32)
        if (wide > nt / 2) consider(true, nt, 1);
    const uint64_t per = (pair ? 2 : 1) * G_FEATS, feat_tiles = (a.feats + per - 1) / per, most = feat_tiles * most_tiles(a.nt);
    if (most >= 1u << 28) return fail_msg(LMZ_GPU_EUNSUPPORTED, "too many rows for a weight of this size");
    a.feat_tiles = static_cast<uint32_t>(feat_tiles), a.col_tiles = static_cast<uint32_t>((a.cols + a.nt - 1) / a.nt);
    a.steps = static_cast<uint32_t>((depth + step_elements - 1) / step_elements);
    a.tmem_columns = tmem_columns(a.split > 1 ? a.nt : 2 * a.nt);
    for (a.split_log = 0; 1u << a.split_log < a.split;) a.split_log++;
    const CUtensorMapDataType type = sizeof(T) == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : std::is_same_v<T, __nv_bfloat16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint32_t cols_each = pair ? a.nt / 2 : a.nt;
    if (P == FORWARD) rc = tile_map(&a.a, at, type, sizeof(T), depth, a.feats, a_stride, G_FEATS, groups, a_plane);
    else if (P == ROWS_GRAD) rc = tile_map(&a.a, at, type, sizeof(T), a.feats, depth, a_stride, STEP_K, groups, a_plane);
    else rc = tile_map(&a.a, at, type, sizeof(T), a.feats, depth, a_stride, STEP_K, 0, 0);
    if (!rc && by_k) rc = tile_map(&a.b, bt, type, sizeof(T), a.cols, depth, b_stride, STEP_K, 0, 0);
    else if (!rc) rc = tile_map(&a.b, bt, type, sizeof(T), depth, a.cols, b_stride, cols_each, 0, 0);
    if (rc) return rc;
    if (pair) return launch_product_as<T, O, P, true>(a, static_cast<unsigned>(std::min<uint64_t>(most, sms / 2) * 2), cs);
    return launch_product_as<T, O, P, false>(a, static_cast<unsigned>(a.split > 1 ? most * a.split : std::min<uint64_t>(most, sms)), cs);
}

template <class T, class O>
static int product_as(const lmz_product *p, cudaStream_t cs)
{
    const ProductLayout l(p, false);
    const ProductInputs<T> in(p, l, true, true, cs);
    if (in.rc) return in.rc;
    ProductArgs a{};
    a.out = p->y, a.z = static_cast<float *>(p->z), a.bias = p->bias, a.times = p->times, a.residual = p->residual, a.a_scale = p->weight_scale, a.b_scale = p->x_scale;
    a.groups = groups_of(p), a.feats = p->out, a.cols = p->rows;
    a.times_stride = p->times_stride, a.residual_stride = p->residual_stride, a.activation = p->activation;
    a.vectors = vector_bytes(p->out * 2, {address(p->y), address(p->z), address(p->bias), address(p->times), p->times ? p->times_stride * 2 : 0, address(p->residual),
                                          p->residual ? p->residual_stride * 2 : 0}) == 16;
    a.plain = !p->z && !p->times && !p->residual && address(p->x_scale) % 16 == 0;
    return launch_product<T, O, FORWARD>(a, in.w, in.w_stride, in.w_plane, in.x, in.x_stride, p->in, cs);
}

template <class T>
static int launch_epilogue_grad(const lmz_product *p, const ProductLayout &l, T *dz, cudaStream_t cs)
{
    const uint32_t chunk = ProductLayout::chunk(p);
    const uint64_t chunks = (p->rows + chunk - 1) / chunk;
    float *partial = p->dbias ? reinterpret_cast<float *>(static_cast<uint8_t *>(p->work) + l.partial) : nullptr;
    uint32_t *most = l.powers ? reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p->work) + l.most) : nullptr;
    if (most) CK("cudaMemsetAsync", cudaMemsetAsync(most, 0, p->experts * 4ull, cs));
    int rc = by_width<T>(vector_bytes(p->out * 2, {address(p->dy), address(p->z) / 2, address(p->times), p->times ? p->times_stride * 2 : 0, address(p->dtimes)}), [&](auto vec) {
        constexpr int VB = sizeof(vec.raw);
        EpilogueGradArgs a{};
        a.dy = p->dy, a.z = p->activation != ACT_NONE || p->dtimes ? static_cast<const float *>(p->z) : nullptr, a.times = p->times, a.dz = dz, a.dtimes = p->dtimes, a.partial = partial, a.groups = groups_of(p);
        a.rows = p->rows, a.out = p->out, a.dz_stride = up8(p->out), a.times_stride = p->times_stride, a.vectors = static_cast<uint32_t>(p->out * 2 / VB), a.activation = p->activation, a.chunk = chunk;
        a.most = most;
        const dim3 grid(static_cast<unsigned>(chunks), (a.vectors + EG_THREADS - 1) / EG_THREADS);
        const int failed = launch("launch k_epilogue_grad", k_epilogue_grad<T, VB>, grid, EG_THREADS, 0, cs, a);
        if constexpr (std::is_same_v<T, __half>)
            if (!failed && most) return launch("launch k_dz_again", k_dz_again<T, VB>, grid, EG_THREADS, 0, cs, a);
        return failed;
    });
    if (!rc && p->dbias)
        rc = launch("launch k_bias_join", k_bias_join<T>, dim3(static_cast<unsigned>((p->out + 31) / 32), p->experts), 32 * BJ_WARPS, 0, cs, static_cast<const float *>(partial),
                    groups_of(p), p->out, chunk, static_cast<T *>(p->dbias));
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
    const bool products = p->dx || p->dweight;
    T *own = l.own_dz && products ? reinterpret_cast<T *>(static_cast<uint8_t *>(p->work) + l.dz) : nullptr;
    int rc = LMZ_GPU_OK;
    if (own || p->dbias || p->dtimes) rc = launch_epilogue_grad<T>(p, l, own, cs);
    if (rc || !products) return rc;
    const ProductInputs<T> in(p, l, p->dweight != nullptr, p->dx != nullptr, cs);
    if (in.rc) return in.rc;
    const T *dz = own ? own : static_cast<const T *>(p->dy);
    const uint64_t dz_stride = own ? up8(p->out) : p->out;
    auto args = [&](void *out, uint64_t cols) {
        ProductArgs a{};
        a.out = out, a.groups = groups_of(p), a.feats = p->in, a.cols = cols;
        a.vectors = vector_bytes(p->in * 2, {address(out)}) == 16, a.plain = true;
        a.most = own && l.powers ? reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(p->work) + l.most) : nullptr;
        return a;
    };
    if (p->dx) {
        ProductArgs a = args(p->dx, p->rows);
        rc = launch_product<T, T, ROWS_GRAD>(a, in.w, in.w_stride, in.w_plane, dz, dz_stride, p->out, cs);
    }
    if (!rc && p->dweight) {
        ProductArgs a = args(p->dweight, p->out);
        rc = launch_product<T, T, WEIGHT_GRAD>(a, in.x, in.x_stride, 0, dz, dz_stride, p->rows, cs);
    }
    return rc;
}

API int lmz_gpu_product_dev(const lmz_product *p, void *cuda_stream)
{
    int rc = check_product(p);
    if (rc || p->rows == 0) return rc;
    if (!p->x || !p->weight || !p->y || (!p->work && ProductLayout(p, false).end)) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a product goes by x, a weight, y, and the workspace that it asks for");
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
    if (!rc && p->rows && !p->work && ProductLayout(p, true).end) rc = fail_msg(LMZ_GPU_EUNSUPPORTED, "a product's gradients go by the workspace that they ask for");
    if (!rc && p->rows && (!p->dy || (p->dx && !p->weight) || (p->dweight && !p->x) || ((p->activation != ACT_NONE || p->dtimes) && !p->z)))
        rc = fail_msg(LMZ_GPU_EUNSUPPORTED, "a product's gradients go by dy, x and the weight, and z where there is an activation or `times`");
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    return p->dtype == LMZ_GPU_BF16 ? product_grad_as<__nv_bfloat16>(p, cs) : product_grad_as<__half>(p, cs);
}
