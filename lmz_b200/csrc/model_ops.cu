// C-ABI entry points of the operators on a checkpoint's tensors: rows of an embedding table, projections with low-rank
// adapters, merges.  Declarations and the per-function contract live in include/lmz_b200.h.
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/lmz_b200.h"
#include "adapter_kernels.cuh"
#include "factor_grad_kernel.cuh"
#include "hidden_kernel.cuh"
#include "merge_kernel.cuh"
#include "merge_wide_kernel.cuh"
#include "project_kernel.cuh"
#include "rows_kernels.cuh"
#include "sort_kernel.cuh"

using namespace lmz;

static_assert(M_MAX_PLACES == LMZ_GPU_MAX_RANK);

#define API extern "C" __attribute__((visibility("default")))

#include "host_error.inl"
#include "host_device.inl"
#include "host_gave_up.inl"

static uint32_t element_bytes(int dtype) { return dtype == LMZ_GPU_F32 ? 4 : dtype == LMZ_GPU_BF16 || dtype == LMZ_GPU_F16 ? 2 : 0; }

// The widest vector, of at most 16 bytes, that rows of `row_bytes` at the given addresses and strides are made of.
static uint32_t vector_bytes(uint64_t row_bytes, std::initializer_list<uint64_t> at)
{
    uint64_t bits = row_bytes | 16;
    for (uint64_t v : at) bits |= v;
    return static_cast<uint32_t>(bits & (~bits + 1));
}

static uint64_t address(const void *p) { return reinterpret_cast<uint64_t>(p); }

// f(type tag, vector width tag) for a type and width; EUNSUPPORTED for a width below the type's.
template <class T, class F>
static int by_width(uint32_t vb, F f)
{
    switch (vb) {
    case 16: return f(Vec<T, 16>{});
    case 8: return f(Vec<T, 8>{});
    case 4: return f(Vec<T, 4>{});
    case 2:
        if constexpr (sizeof(T) == 2) return f(Vec<T, 2>{});
        break;
    }
    return fail_msg(LMZ_GPU_EUNSUPPORTED, "a tensor does not start on a boundary of its elements");
}

template <class F>
static int by_type(int dtype, uint32_t vb, F f)
{
    if (dtype == LMZ_GPU_BF16) return by_width<__nv_bfloat16>(vb, [&](auto v) { return f(__nv_bfloat16{}, v); });
    if (dtype == LMZ_GPU_F16) return by_width<__half>(vb, [&](auto v) { return f(__half{}, v); });
    if (dtype == LMZ_GPU_F32) return by_width<float>(vb, [&](auto v) { return f(float{}, v); });
    return fail_msg(LMZ_GPU_EUNSUPPORTED, "an element type other than BF16, F16 and F32");
}

// A launch in clusters along x whose blocks may start before the kernel in front of it has ended: each of these kernels waits
// for that itself, before it reads or writes what another may have to do with.
static cudaLaunchConfig_t clustered(dim3 grid, unsigned threads, size_t smem, cudaStream_t cs, unsigned cluster, cudaLaunchAttribute (&attrs)[2])
{
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster, attrs[1].val.clusterDim.y = 1, attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = smem, c.stream = cs, c.attrs = attrs, c.numAttrs = cluster > 1 ? 2 : 1;
    return c;
}

// The same without clusters.
template <class K, class... A>
static int launch(const char *what, K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t cs, A... args)
{
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(grid, threads, smem, cs, 1, attrs);
    CK(what, cudaLaunchKernelEx(&c, kernel, args...));
    return LMZ_GPU_OK;
}

static uint32_t lanes_log(uint32_t vectors)
{
    uint32_t log = 0;
    while ((1u << log) < vectors && (1u << log) < ROW_THREADS) log++;
    return log;
}

static int check_rows(uint64_t rows, uint64_t dim, int dtype, int id_bytes, uint64_t n)
{
    const uint32_t e = element_bytes(dtype);
    if (!e) return fail_msg(LMZ_GPU_EUNSUPPORTED, "an element type other than BF16, F16 and F32");
    if (id_bytes != 4 && id_bytes != 8) return fail_msg(LMZ_GPU_EUNSUPPORTED, "ids are int32 or int64");
    if (rows >= 1ull << 31 || n >= 1ull << 31) return fail_msg(LMZ_GPU_EUNSUPPORTED, "2^31 rows or tokens and more");
    if (dim == 0 || dim >= 1ull << 24) return fail_msg(LMZ_GPU_EUNSUPPORTED, "a row has between 1 and 2^24 - 1 elements");
    return LMZ_GPU_OK;
}

API int lmz_gpu_rows_dev(const void *d_table, uint64_t rows, uint64_t dim, uint64_t row_stride, int dtype, const void *d_ids,
                         int id_bytes, uint64_t n, float scale, void *d_out, void *cuda_stream)
{
    int rc = check_rows(rows, dim, dtype, id_bytes, n);
    if (rc) return rc;
    if (n == 0) return LMZ_GPU_OK;
    rc = device_ready();
    if (rc) return rc;
    const uint64_t e = element_bytes(dtype), bytes = dim * e;
    const uint32_t vb = vector_bytes(bytes, {address(d_table), address(d_out), row_stride * e});
    return by_type(dtype, vb, [&](auto type, auto vec) {
        using T = decltype(type);
        constexpr int VB = sizeof(vec.raw);
        RowsArgs a{};
        a.table = static_cast<const uint8_t *>(d_table), a.ids = d_ids, a.out = static_cast<uint8_t *>(d_out);
        a.rows = rows, a.n = n, a.row_bytes = bytes, a.stride_bytes = row_stride * e;
        a.vectors = static_cast<uint32_t>(bytes / VB), a.lane_log = lanes_log(a.vectors);
        a.scale = scale, a.wide = id_bytes == 8;
        constexpr int U = 4;
        const uint32_t per = (ROW_THREADS >> a.lane_log) * U;
        return launch("launch k_rows", k_rows<T, VB, U>, dim3(static_cast<unsigned>((n + per - 1) / per)), ROW_THREADS, 0, static_cast<cudaStream_t>(cuda_stream), a);
    });
}

// Tokens of a window of the rows' gradient: 32, and in windows of more for more than 4096 windows' tokens.
static uint32_t rows_window(uint64_t n) { return static_cast<uint32_t>((std::max<uint64_t>(ROWS_STEP, (n + 4095) / 4096) + ROWS_STEP - 1) / ROWS_STEP * ROWS_STEP); }

struct RowsGradLayout {
    uint64_t keys[2], pos[2], partial, end;
    RowsGradLayout(uint64_t n, uint64_t dim)
    {
        uint64_t at = 0;
        auto take = [&](uint64_t bytes) { const uint64_t r = at; at += (bytes + 255) & ~255ull; return r; };
        for (int i = 0; i < 2; i++) keys[i] = take(n * 4), pos[i] = take(n * 4);
        const uint64_t w = rows_window(n);
        partial = take(n > w ? (n + w - 1) / w * 2 * dim * 4 : 0);
        end = at;
    }
};

// Sort ids; on return *side is where the result lies.
static int launch_sort(SortArgs &s, cudaStream_t cs, int *side)
{
    static bool done[64];
    const int rc = opt_in_smem(k_sort, sort_smem(SORT_DIGIT), done);
    if (rc) return rc;
    uint32_t bits = 1;
    while (bits < 32 && s.nkeys >> bits) bits++;
    s.passes = (bits + SORT_DIGIT - 1) / SORT_DIGIT, s.digit = std::max(5u, (bits + s.passes - 1) / s.passes);
    // (a thousand elements are sorted by one CTA before a cluster has met)
    const uint32_t ctas = s.n <= SORT_THREADS ? 1 : SORT_CTAS;
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(ctas), SORT_THREADS, sort_smem(s.digit), cs, ctas, attrs);
    CK("launch k_sort", cudaLaunchKernelEx(&c, k_sort, static_cast<const SortArgs>(s)));
    *side = (s.passes - 1) & 1;
    return LMZ_GPU_OK;
}

API size_t lmz_gpu_rows_grad_work_bytes(uint64_t n, uint64_t, uint64_t dim) { return RowsGradLayout(n, dim).end; }

API int lmz_gpu_rows_grad_dev(const void *d_dy, uint64_t n, uint64_t dim, int dtype, const void *d_ids, int id_bytes, uint64_t rows,
                              float scale, void *d_dtable, void *d_work, void *cuda_stream)
{
    int rc = check_rows(rows, dim, dtype, id_bytes, n);
    if (rc) return rc;
    if (rows == 0) return LMZ_GPU_OK;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    const uint64_t bytes = dim * element_bytes(dtype);
    if (n == 0) {
        CK("cudaMemsetAsync", cudaMemsetAsync(d_dtable, 0, rows * bytes, cs));
        return LMZ_GPU_OK;
    }
    const RowsGradLayout l(n, dim);
    uint8_t *work = static_cast<uint8_t *>(d_work);
    auto words = [&](uint64_t off) { return reinterpret_cast<uint32_t *>(work + off); };
    SortArgs s{};
    s.ids = d_ids, s.n = n, s.nkeys = rows, s.wide = id_bytes == 8;
    for (int i = 0; i < 2; i++) s.keys[i] = words(l.keys[i]), s.pos[i] = words(l.pos[i]);
    int side = 0;
    rc = launch_sort(s, cs, &side);
    const uint64_t total = rows * bytes, blocks = (total + CLEAR_BYTES - 1) / CLEAR_BYTES;
    if (!rc && blocks >= 1u << 30) rc = fail_msg(LMZ_GPU_EUNSUPPORTED, "a table of 64 TiB and more");
    if (!rc) rc = launch("launch k_clear", k_clear, dim3(static_cast<unsigned>(blocks)), CLEAR_THREADS, 0, cs, static_cast<uint8_t *>(d_dtable), total);
    if (rc) return rc;
    return by_type(dtype, vector_bytes(bytes, {address(d_dy), address(d_dtable)}), [&](auto type, auto vec) {
        using T = decltype(type);
        constexpr int VB = sizeof(vec.raw);
        RowsGradArgs a{};
        a.dy = static_cast<const uint8_t *>(d_dy), a.keys = s.keys[side], a.pos = s.pos[side];
        a.partial = reinterpret_cast<float *>(work + l.partial), a.out = static_cast<uint8_t *>(d_dtable);
        a.rows = static_cast<uint32_t>(rows), a.row_bytes = bytes, a.dim = dim, a.n = static_cast<uint32_t>(n), a.window = rows_window(n), a.scale = scale;
        a.vectors = static_cast<uint32_t>(bytes / VB), a.lane_log = std::max(5u, lanes_log(a.vectors));
        const uint32_t slices = (a.vectors + ROW_THREADS - 1) / ROW_THREADS, per = ROW_THREADS >> a.lane_log;
        // (a row of 2^24 elements less one, two bytes at a time, is 65536 slices: one more than a grid has along y)
        const dim3 grid(((a.n + a.window - 1) / a.window + per - 1) / per, std::min(slices, 32768u), (slices + 32767) / 32768);
        int failed = launch("launch k_rows_sums", k_rows_sums<T, VB>, grid, ROW_THREADS, 0, cs, a);
        if (!failed && a.n > a.window) failed = launch("launch k_rows_join", k_rows_join<T, VB>, grid, ROW_THREADS, 0, cs, a);
        return failed;
    });
}

// ------------------------------------------------------------------ adapters

static int check_projection(const lmz_projection *p)
{
    if (p->dtype != LMZ_GPU_BF16 && p->dtype != LMZ_GPU_F16) return fail_msg(LMZ_GPU_EUNSUPPORTED, "projections are of BF16 or F16");
    if (p->index && p->index_bytes != 4 && p->index_bytes != 8) return fail_msg(LMZ_GPU_EUNSUPPORTED, "an index is of int32 or int64");
    if (p->rank == 0 || p->rank > LMZ_GPU_MAX_RANK) return report(LMZ_GPU_EUNSUPPORTED, "ranks are between 1 and %d", LMZ_GPU_MAX_RANK);
    if (p->adapters == 0 || p->adapters > 65535) return fail_msg(LMZ_GPU_EUNSUPPORTED, "between 1 and 65535 adapters");
    if (p->in == 0 || p->out == 0 || p->in >= 1u << 21 || p->out >= 1u << 21)
        return fail_msg(LMZ_GPU_EUNSUPPORTED, "a weight has between 1 and 2^21 - 1 rows and columns");
    if (p->tokens >= 1ull << 31) return fail_msg(LMZ_GPU_EUNSUPPORTED, "2^31 tokens and more");
    return LMZ_GPU_OK;
}

static TokenIndex token_index(const lmz_projection *p)
{
    return {p->index, static_cast<const float *>(p->scales), p->scale, p->adapters, p->index_bytes == 8};
}

static uint64_t up8(uint64_t n) { return (n + 7) & ~7ull; }
static uint64_t up256(uint64_t n) { return (n + 255) & ~255ull; }

// Rows of 16-bit elements that TMA and 16-byte copies take as they lie.
static bool on_boundary(const void *p, uint64_t cols, uint64_t stride) { return address(p) % 16 == 0 && stride % 8 == 0 && stride >= cols; }

// A tensor map of planes x rows x cols 16-bit elements, a plane's rows behind those of the plane before: tiles of 64 columns
// with the 128-byte swizzle.
static int tensor_map(CUtensorMap *map, const void *p, bool bf16, uint64_t cols, uint64_t rows, uint64_t stride, uint32_t tile_rows, uint64_t planes = 0,
                      uint32_t tile_planes = 1)
{
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return fail_msg(LMZ_GPU_EUNSUPPORTED, "the driver makes no tensor maps");
    const cuuint64_t dims[3] = {cols, rows, planes}, strides[2] = {stride * 2, stride * rows * 2};
    const cuuint32_t box[3] = {STEP_K, tile_rows, tile_planes}, steps[3] = {1, 1, 1};
    const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, planes ? 3 : 2, const_cast<void *>(p), dims,
                              strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? LMZ_GPU_OK : report(LMZ_GPU_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// Whether a projection that finds more than a quarter of its sixteens of tokens with several adapters takes the tokens in the
// order of their adapters.  To find out costs 7 us, the order and the copy of x 10 and more, and without them the sixteens take
// some 2.4 us a feature tile and 16 places of the rank on a multiprocessor: from 30 us of that on, if sixteens of one adapter
// come of it.  One B200, tokens x in x out, adapters, rank, in any order and in runs, with it and without: 8192x4096x4096 of 30 r16 240
// and 219 against 505 and 213, 8000x512x512 of 8 r128 77 and 66 against 301 and 56, 2048x1024x2048 of 16 r16 52 and 40 against 75
// and 34, 1024x4096x1024 of 8 r32 42 and 34 against 47 and 27 (left without).
static bool worth_sorting(const lmz_projection *p, uint64_t feats, uint64_t rp) { return p->tokens >= 8ull * p->adapters && p->tokens * feats * rp >= 1ull << 26; }

// Adapters that can have a sixteen of tokens to themselves: places for the parts of an F16 factor.
static uint64_t parts_slots(const lmz_projection *p) { return std::min<uint64_t>(p->index ? p->adapters : 1, (p->tokens + 15) / 16); }

// What a projection's kernels read in place of tensors that do not lie on boundaries, and between each other.
struct ProjectLayout {
    uint64_t x, w, a, b, dy, g, keys[2], pos[2], start, hidden, scattered, in_order, thin, parts, slot, halves[2], scale[2], end = 0;
    bool pack_x, pack_w, pack_a, pack_b, pack_dy;
    bool sorts;                                // the projection takes scattered tokens by adapter
    ProjectLayout(const lmz_projection *p, bool grad)
    {
        auto take = [&](bool on, uint64_t bytes) {
            const uint64_t r = end;
            if (on) end += up256(bytes);
            return r;
        };
        pack_x = !on_boundary(p->x, p->in, p->x_stride);
        pack_w = !on_boundary(p->weight, p->in, p->weight_stride);
        pack_a = !on_boundary(p->a, p->in, p->in);
        pack_b = grad || !on_boundary(p->b, p->rank, p->rank);   // (the gradients' transposed: [adapter][rank][out])
        pack_dy = grad && !on_boundary(p->dy, p->out, p->out);
        x = take(pack_x, p->tokens * up8(p->in) * 2);
        w = take(pack_w, p->out * up8(p->in) * 2);
        a = take(pack_a, p->adapters * p->rank * up8(p->in) * 2);
        b = take(pack_b, 2 * p->adapters * (grad ? p->rank * up8(p->out) : p->out * up8(p->rank)));
        dy = take(pack_dy, p->tokens * up8(p->out) * 2);
        g = take(grad, p->tokens * 4 * up8(p->rank));
        const bool may_sort = p->index && p->adapters > 1 && worth_sorting(p, grad ? p->in : p->out, up8(p->rank));
        sorts = may_sort && (!grad || p->dx);                    // (the workspace is the same whichever gradients are wanted)
        const bool sorted = (grad && p->index) || may_sort;
        for (int i = 0; i < 2; i++) keys[i] = take(sorted, p->tokens * 4), pos[i] = take(sorted, p->tokens * 4);
        start = take(grad && p->index, (p->adapters + 1ull) * 4);
        hidden = take(!grad && !p->hidden, p->tokens * 4 * up8(p->rank));
        scattered = take(may_sort, 4);
        in_order = take(may_sort, p->tokens * up8(grad ? p->out : p->in) * 2);
        const bool f16 = p->dtype == LMZ_GPU_F16;
        thin = take((may_sort || f16) && (grad || p->hidden), p->tokens * 4 * up8(p->rank));
        parts = take(f16, 4 * parts_slots(p) * (grad ? p->rank * up8(p->in) : p->out * up8(p->rank)));
        slot = take(f16, p->adapters * 4ull);
        for (int i = 0; i < 2; i++) halves[i] = take(grad && f16, p->tokens * 4 * up8(p->rank)), scale[i] = take(grad && f16, p->adapters * 4ull);
    }
};

API size_t lmz_gpu_project_hidden_bytes(const lmz_projection *p) { return p->tokens * 4 * up8(p->rank); }
API size_t lmz_gpu_project_work_bytes(const lmz_projection *p, int grad) { return ProjectLayout(p, grad).end; }

constexpr uint32_t OPS_SMEM = 201u << 10;      // dynamic shared memory that the kernels below are laid out within
constexpr uint32_t PROJECT_SMEM = 222u << 10;
static_assert(PROJECT_SMEM + sizeof(ProjectShared) <= 227u << 10);

static uint32_t tmem_columns(uint32_t n)
{
    uint32_t c = 32;
    while (c < n) c *= 2;
    return c;
}

template <class T, bool MN, bool PAIR>
static int launch_project_as(ProjectArgs<T> &a, unsigned grid, cudaStream_t cs)
{
    static bool done[64];
    const int rc = opt_in_smem(k_project<T, MN, PAIR>, PROJECT_SMEM, done);
    if (rc) return rc;
    a.stage_bytes = project_stage_bytes(a.nt, PAIR);
    // A slot per group that may be mixed, where a pair's six stages leave room for three.
    a.slots = PAIR ? 3 : std::min(P_MAX_SLOTS, (a.nt / P_GROUP + a.split - 1) / a.split);
    const uint32_t rest = ATOM_BYTES + a.slots * P_SLOT_BYTES + (PAIR ? 1 : 2) * P_GROUP * P_PLACES * 4;
    a.stages = std::min<uint32_t>(P_MAX_STAGES, (PROJECT_SMEM - rest) / a.stage_bytes);
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(grid), P_THREADS, a.stages * a.stage_bytes + rest, cs, PAIR ? 2 : a.split, attrs);
    CK("launch k_project", cudaLaunchKernelEx(&c, k_project<T, MN, PAIR>, a));
    return LMZ_GPU_OK;
}

// Scattered tokens by adapter (launch_in_order), or nothing.
template <class T>
struct InOrder {
    SortedTokens sorted{};
    const T *x = nullptr;                        // rows of up8(k) elements
};

// An F16 factor's parts, behind the thin product and beside it.
static int launch_parts(const lmz_projection *p, const SortedTokens &sorted, const __half *factor, uint64_t each, Thin *parts, uint32_t *slot, cudaStream_t cs)
{
    const uint64_t slots = parts_slots(p);
    PartsArgs a{};
    a.in = factor, a.out = parts, a.slot = slot, a.index = token_index(p), a.sorted = sorted;
    a.each = each, a.tokens = p->tokens, a.sixteens = (p->tokens + 15) / 16;
    const uint64_t blocks = (each + PARTS_VALUES - 1) / PARTS_VALUES;          // (below 2^21 * 256 / 2^13)
    return launch("launch k_parts", k_parts, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(slots)), PARTS_THREADS, 0, cs, a);
}

// y[t][f] = sum of x[t][k] W(f, k) + sum of h[t][j] F_i(f, j) (MN: W and F with their f next to each other).
template <class T, bool MN>
static int launch_project(const lmz_projection *p, const InOrder<T> &o, const T *x, uint64_t x_stride, uint64_t k, const T *w, uint64_t w_stride, uint64_t feats, const T *factor,
                          uint64_t factor_rows, uint64_t factor_row, const Thin *hidden, const ProjectLayout &l, T *y, cudaStream_t cs)
{
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    ProjectArgs<T> a{};
    Thin *parts = reinterpret_cast<Thin *>(static_cast<uint8_t *>(p->work) + l.parts);
    if constexpr (std::is_same_v<T, __half>) {
        uint32_t *slot = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p->work) + l.slot);
        a.slot = slot;
        rc = launch_parts(p, o.sorted, factor, factor_rows * factor_row, parts, slot, cs);
        if (rc) return rc;
    }
    a.index = token_index(p), a.sorted = o.sorted, a.hidden = hidden, a.factor = factor, a.factor_each = factor_rows * factor_row, a.factor_row = factor_row;
    a.y = y, a.tokens = p->tokens, a.feats = feats, a.rank = p->rank, a.rp = static_cast<uint32_t>(up8(p->rank));
    a.steps = static_cast<uint32_t>((k + STEP_K - 1) / STEP_K), a.split = 1;
    auto tiles = [&](uint64_t f, uint64_t t) { return (feats + f - 1) / f * ((p->tokens + t - 1) / t); };
    // Tiles of 256 by 256 by pairs of CTAs, or of 128 features by 16 to 128 tokens by one, or by a cluster that shares K: by what
    // they are reckoned to take (in 10 ns).  A step of a pair takes 0.3 us, of a CTA 0.19 or what L2 gives all of them their tiles
    // in; a cluster's meeting 1.5 us and more.  One B200, rank 16, us in all, tokens x in x out: 512x4096x4096 pairs 35, 128 tokens a
    // CTA 34, 64 a CTA 38; 200x4096x4096 64 a CTA 23, 128 a CTA 26, pairs 33; 16x4096x4096 by two CTAs 15.5, by one 20, by four 18;
    // 2048x1024x1024 128 a CTA 21, pairs 26; 128x1024x4096 32 a CTA 12, 128 by four 21; 300x4096x14336 pairs 56, 128 a CTA 70.
    uint64_t best = ~0ull;
    bool pair = false;
    auto consider = [&](bool p2, uint32_t nt, uint32_t split) {
        const uint64_t n = tiles(p2 ? 2 * P_FEATS : P_FEATS, nt) * split, places = p2 ? sms / 2 : sms;
        if (split > 1 && n > places) return;
        const uint64_t waves = (n + places - 1) / places, steps = (a.steps + split - 1) / split;
        const uint64_t step = p2 ? 30 : std::max<uint64_t>(19, std::min(n, places) * (P_FEATS + nt) / 940);
        const uint64_t meeting = split == 1 ? 0 : split == 2 ? 150 + 5 * nt / 2 : 180 * split;
        const uint64_t cost = waves * (step * steps + (p2 ? 600 : 4 * nt + meeting)) + 600;
        if (cost < best) best = cost, pair = p2, a.nt = nt, a.split = split;
    };
    for (uint32_t nt = P_GROUP; nt < P_TOKENS; nt *= 2)
        for (uint32_t split = 1; split <= 8 && 2 * split <= std::max(2u, a.steps); split *= 2)
            if (nt == P_GROUP || nt < 2 * p->tokens) consider(false, nt, split);
    if (p->tokens > P_TOKENS / 2) consider(true, P_TOKENS, 1);
    const uint64_t count = tiles(pair ? 2 * P_FEATS : P_FEATS, a.nt);
    if (count >= 1u << 28) return fail_msg(LMZ_GPU_EUNSUPPORTED, "too many tokens for a weight of this size");
    a.feat_tiles = static_cast<uint32_t>((feats + (pair ? 2 : 1) * P_FEATS - 1) / ((pair ? 2 : 1) * P_FEATS));
    a.token_tiles = static_cast<uint32_t>((p->tokens + a.nt - 1) / a.nt);
    a.tmem_columns = tmem_columns(a.split > 1 ? a.nt : 2 * a.nt);
    constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
    rc = tensor_map(&a.x, x, bf16, k, p->tokens, x_stride, pair ? a.nt / 2 : a.nt);
    if (!rc && o.x) rc = tensor_map(&a.xs, o.x, bf16, k, p->tokens, up8(k), pair ? a.nt / 2 : a.nt);
    if (!rc) rc = MN ? tensor_map(&a.w, w, bf16, feats, k, w_stride, STEP_K) : tensor_map(&a.w, w, bf16, k, feats, w_stride, P_FEATS);
    if (!rc) rc = tensor_map(&a.h, hidden, true, a.rp, 2, a.rp, 1, p->tokens, pair ? a.nt / 2 : a.nt);
    const void *f = factor;
    if (!bf16) f = parts;
    const uint64_t planes = bf16 ? p->adapters : 2 * parts_slots(p);
    if (!rc) rc = MN ? tensor_map(&a.f, f, true, feats, factor_rows, factor_row, STEP_K, planes) : tensor_map(&a.f, f, true, a.rp, factor_rows, factor_row, P_FEATS, planes);
    if (rc) return rc;
    if (pair) return launch_project_as<T, MN, true>(a, static_cast<unsigned>(std::min<uint64_t>(count, sms / 2) * 2), cs);
    return launch_project_as<T, MN, false>(a, static_cast<unsigned>(a.split > 1 ? count * a.split : std::min<uint64_t>(count, sms)), cs);
}

// h = s x F^T for each token's own adapter; f: [adapter][rank][f_stride], its first k of each row.
template <class T>
static int launch_hidden(const lmz_projection *p, const InOrder<T> &o, const T *x, uint64_t x_stride, uint64_t k, const T *f, uint64_t f_stride, Thin *h, void *kept,
                         cudaStream_t cs)
{
    static bool done[64];
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    HiddenArgs<T> a{};
    a.index = token_index(p), a.sorted = o.sorted, a.h = h, a.kept = kept, a.tokens = p->tokens, a.rank = p->rank, a.rp = static_cast<uint32_t>(up8(p->rank));
    a.steps = static_cast<uint32_t>((k + STEP_K - 1) / STEP_K);
    const uint64_t tiles = (p->tokens + H_TOKENS - 1) / H_TOKENS;
    const uint32_t most = static_cast<uint32_t>(std::min<uint64_t>(p->index ? std::min(p->adapters, H_TOKENS) : 1, p->tokens));
    // As many adapters to a block as have room: the fewer blocks, the more multiprocessors the next kernel finds free for its
    // weight (one B200, 64 tokens of 48 adapters, 4096x14336: 24 blocks 60 us in all, 96 blocks 72).
    a.each = std::min(H_COLUMNS / a.rp, most);
    const uint32_t groups = (most + a.each - 1) / a.each, columns = (a.each * a.rp + 15) & ~15u;
    a.stage_bytes = (H_TOKENS + columns) * ROW_BYTES, a.tmem_columns = tmem_columns(columns);
    a.stages = std::min<uint32_t>(H_MAX_STAGES, (OPS_SMEM - ATOM_BYTES) / a.stage_bytes);
    a.split = 1;
    while (a.split < 8 && tiles * groups * a.split * 2 <= (uint64_t)sms && a.steps >= 4 * a.split) a.split *= 2;
    constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
    rc = tensor_map(&a.x, x, bf16, k, p->tokens, x_stride, H_TOKENS);
    if (!rc && o.x) rc = tensor_map(&a.xs, o.x, bf16, k, p->tokens, up8(k), H_TOKENS);
    if (!rc) rc = tensor_map(&a.f, f, bf16, k, p->rank, f_stride, p->rank, p->adapters);
    if (!rc) rc = opt_in_smem(k_hidden<T>, OPS_SMEM, done);
    if (rc) return rc;
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(static_cast<unsigned>(tiles * a.split), groups), H_THREADS, a.stages * a.stage_bytes + ATOM_BYTES, cs, a.split, attrs);
    CK("launch k_hidden", cudaLaunchKernelEx(&c, k_hidden<T>, a));
    return LMZ_GPU_OK;
}

// One factor's gradient: dF_i(f, j) = the sum over i's tokens of thin[t][j] z[t][f].
template <class T>
struct FactorGrad {
    const T *z;
    uint64_t stride, feats;
    const T *thin;
    T *out;
    uint64_t wide, place;
    const float *scale;                          // F16 (k_thin)
};

template <class T>
static int launch_factor_grad(const lmz_projection *p, const FactorGrad<T> *jobs, uint32_t count, const uint32_t *order, const uint32_t *start, cudaStream_t cs)
{
    static bool done[64];
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    FactorGradArgs<T> a{};
    a.order = order, a.start = start;
    a.tokens = static_cast<uint32_t>(p->tokens), a.rank = p->rank, a.rp = static_cast<uint32_t>(up8(p->rank));
    a.blocks = a.rp <= 128 ? 2 : 1;                              // (as many as TMEM has columns for)
    a.stage_bytes = factor_stage_bytes(a.blocks, a.rp), a.tmem_columns = tmem_columns(a.blocks * 2 * a.rp);
    a.stages = std::min<uint32_t>(FG_MAX_STAGES, (OPS_SMEM - ATOM_BYTES) / a.stage_bytes);
    constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
    uint32_t clusters = 0;
    for (uint32_t i = 0; i < count; i++) {
        const FactorGrad<T> &f = jobs[i];
        FactorGradJob<T> &g = a.job[i];
        g.out = f.out, g.scale = f.scale, g.feats = f.feats, g.each = f.feats * p->rank, g.wide = f.wide, g.place = f.place;
        g.clusters = static_cast<uint32_t>((f.feats + a.blocks * FG_FEATS - 1) / (a.blocks * FG_FEATS));
        clusters += g.clusters;
        rc = tensor_map(&g.z, f.z, bf16, f.feats, p->tokens, f.stride, STEP_K);
        if (!rc) rc = tensor_map(&g.z_rows, f.z, bf16, f.feats, p->tokens, f.stride, 1);
        if (!rc) rc = tensor_map(&g.thin, f.thin, bf16, 2 * a.rp, p->tokens, 2 * a.rp, STEP_K);
        if (!rc) rc = tensor_map(&g.thin_rows, f.thin, bf16, 2 * a.rp, p->tokens, 2 * a.rp, 1);
        if (rc) return rc;
    }
    a.split = 1;
    while (a.split < 8 && (uint64_t)clusters * p->adapters * a.split * 2 <= (uint64_t)sms && p->tokens >= 4ull * STEP_K * a.split) a.split *= 2;
    rc = opt_in_smem(k_factor_grad<T>, OPS_SMEM, done);
    if (rc) return rc;
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(clusters * a.split, p->adapters), FG_THREADS, a.stages * a.stage_bytes + ATOM_BYTES, cs, a.split, attrs);
    CK("launch k_factor_grad", cudaLaunchKernelEx(&c, k_factor_grad<T>, a));
    return LMZ_GPU_OK;
}

// A projection's tensors as the kernels take them: where they lie, or packed into the workspace (in one launch).
template <class T>
struct ProjectInputs {
    const T *x, *w, *a, *b, *dy;
    uint64_t x_stride, w_stride, a_stride, dy_stride;
    int rc;
    ProjectInputs(const lmz_projection *p, const ProjectLayout &l, bool grad, cudaStream_t cs)
        : x(static_cast<const T *>(p->x)), w(static_cast<const T *>(p->weight)), a(static_cast<const T *>(p->a)), b(static_cast<const T *>(p->b)),
          dy(static_cast<const T *>(p->dy)), x_stride(p->x_stride), w_stride(p->weight_stride), a_stride(p->in), dy_stride(p->out), rc(LMZ_GPU_OK)
    {
        PackArgs<T> args{};
        uint32_t jobs = 0;
        uint64_t most = 0;
        auto job = [&](const T *&t, uint64_t outer, uint64_t so, uint64_t rows, uint64_t sr, uint64_t cols, uint64_t sc, uint64_t off) {
            T *to = reinterpret_cast<T *>(static_cast<uint8_t *>(p->work) + off);
            args.job[jobs++] = {t, to, so, sr, sc, rows, cols, up8(cols), outer * rows};
            most = std::max(most, sc == 1 ? outer * rows * up8(cols) / 256 + 1 : outer * rows * ((up8(cols) + PACK_COLS - 1) / PACK_COLS));    // (warps)
            t = to;
        };
        const uint64_t r = p->rank;
        if (l.pack_x) job(x, 1, 0, p->tokens, x_stride, p->in, 1, l.x), x_stride = up8(p->in);
        if (l.pack_w) job(w, 1, 0, p->out, w_stride, p->in, 1, l.w), w_stride = up8(p->in);
        if (l.pack_a) job(a, 1, 0, p->adapters * r, p->in, p->in, 1, l.a), a_stride = up8(p->in);
        if (grad && l.pack_dy) job(dy, 1, 0, p->tokens, p->out, p->out, 1, l.dy), dy_stride = up8(p->out);
        if (grad) job(b, p->adapters, p->out * r, r, 1, p->out, r, l.b);
        else if (l.pack_b) job(b, 1, 0, p->adapters * p->out, r, r, 1, l.b);
        if (!jobs) return;
        const dim3 grid(static_cast<unsigned>(std::min<uint64_t>((most + PACK_WARPS - 1) / PACK_WARPS, 1u << 20)), jobs);
        rc = launch("launch k_pack", k_pack<T>, grid, 32 * PACK_WARPS, 0, cs, args);
    }
};

// The sort of the tokens by adapter; `order` is where it lies.  `start`: and where each adapter's begin.
static int launch_token_sort(const lmz_projection *p, const ProjectLayout &l, bool start, SortedTokens *sorted, cudaStream_t cs)
{
    uint8_t *work = static_cast<uint8_t *>(p->work);
    auto words = [&](uint64_t off) { return reinterpret_cast<uint32_t *>(work + off); };
    SortArgs s{};
    s.ids = p->index, s.n = p->tokens, s.nkeys = p->adapters, s.wide = p->index_bytes == 8;
    for (int i = 0; i < 2; i++) s.keys[i] = words(l.keys[i]), s.pos[i] = words(l.pos[i]);
    s.start = start ? words(l.start) : nullptr, s.scattered = l.sorts ? words(l.scattered) : nullptr;
    int side = 0;
    const int rc = launch_sort(s, cs, &side);
    *sorted = {s.scattered, s.pos[side], s.keys[side]};
    return rc;
}

// x's rows by adapter, if the sort has found them scattered.
template <class T>
static int launch_in_order(const lmz_projection *p, const ProjectLayout &l, const T *x, uint64_t x_stride, uint64_t k, InOrder<T> *o, cudaStream_t cs)
{
    T *to = reinterpret_cast<T *>(static_cast<uint8_t *>(p->work) + l.in_order);
    o->x = to;
    return launch("launch k_gather", k_gather<T>, dim3(static_cast<unsigned>((p->tokens + GATHER_WARPS - 1) / GATHER_WARPS)), 32 * GATHER_WARPS, 0, cs, o->sorted, x,
                  x_stride, static_cast<uint32_t>(k), p->tokens, to, up8(k));
}

template <class T>
static int project_as(const lmz_projection *p, cudaStream_t cs)
{
    const ProjectLayout l(p, false);
    const ProjectInputs<T> in(p, l, false, cs);
    auto work = [&](uint64_t off) -> void * { return static_cast<uint8_t *>(p->work) + off; };
    int rc = in.rc;
    InOrder<T> o;
    constexpr bool f16 = std::is_same_v<T, __half>;
    Thin *h = static_cast<Thin *>(p->hidden && !l.sorts && !f16 ? p->hidden : work(p->hidden ? l.thin : l.hidden));
    void *kept = h == p->hidden ? nullptr : p->hidden;
    if (!rc && l.sorts) {
        rc = launch_token_sort(p, l, false, &o.sorted, cs);
        if (!rc) rc = launch_in_order(p, l, in.x, in.x_stride, p->in, &o, cs);
    }
    if (!rc) rc = launch_hidden(p, o, in.x, in.x_stride, p->in, in.a, in.a_stride, h, kept, cs);
    if (!rc) rc = launch_project<T, false>(p, o, in.x, in.x_stride, p->in, in.w, in.w_stride, p->out, in.b, p->out, up8(p->rank), h, l, static_cast<T *>(p->y), cs);
    return rc;
}

// The halves of F16's thin products.
static int launch_thin(const lmz_projection *p, const ThinJob *jobs, uint32_t count, const uint32_t *order, const uint32_t *start, cudaStream_t cs)
{
    ThinArgs a{};
    for (uint32_t i = 0; i < count; i++) a.job[i] = jobs[i];
    a.order = order, a.start = start, a.tokens = static_cast<uint32_t>(p->tokens), a.rp = static_cast<uint32_t>(up8(p->rank));
    cudaLaunchAttribute attrs[2]{};
    const cudaLaunchConfig_t c = clustered(dim3(THIN_CTAS, p->adapters, count), THIN_THREADS, 0, cs, THIN_CTAS, attrs);
    CK("launch k_thin", cudaLaunchKernelEx(&c, k_thin, static_cast<const ThinArgs>(a)));
    return LMZ_GPU_OK;
}

template <class T>
static int project_grad_as(const lmz_projection *p, cudaStream_t cs)
{
    const uint64_t r = p->rank;
    if (p->tokens == 0) {
        if (p->da) CK("cudaMemsetAsync", cudaMemsetAsync(p->da, 0, 2ull * p->adapters * r * p->in, cs));
        if (p->db) CK("cudaMemsetAsync", cudaMemsetAsync(p->db, 0, 2ull * p->adapters * r * p->out, cs));
        return LMZ_GPU_OK;
    }
    const ProjectLayout l(p, true);
    const ProjectInputs<T> in(p, l, true, cs);
    auto work = [&](uint64_t off) -> void * { return static_cast<uint8_t *>(p->work) + off; };
    constexpr bool f16 = std::is_same_v<T, __half>;
    int rc = in.rc;
    InOrder<T> o;
    SortedTokens tokens{};
    void *g = work(l.g);                                         // what da needs of the thin product
    Thin *h = static_cast<Thin *>(l.sorts || f16 ? work(l.thin) : g);
    const bool factors = p->da || p->db;
    if (!rc && l.sorts) {
        rc = launch_token_sort(p, l, factors, &tokens, cs);
        o.sorted = tokens;
        if (!rc) rc = launch_in_order(p, l, in.dy, in.dy_stride, p->out, &o, cs);
    }
    if (!rc && (p->dx || p->da)) rc = launch_hidden(p, o, in.dy, in.dy_stride, p->out, in.b, up8(p->out), h, p->da && h != g ? g : nullptr, cs);
    if (!rc && p->dx) rc = launch_project<T, true>(p, o, in.dy, in.dy_stride, p->out, in.w, in.w_stride, p->in, in.a, r, in.a_stride, h, l, static_cast<T *>(p->dx), cs);
    if (rc || !factors) return rc;
    if (p->index && !l.sorts) rc = launch_token_sort(p, l, true, &tokens, cs);
    if (rc) return rc;
    const uint32_t *start = p->index ? static_cast<const uint32_t *>(work(l.start)) : nullptr;
    FactorGrad<T> jobs[2]{};
    uint32_t count = 0;
    if (p->db) jobs[count++] = {in.dy, in.dy_stride, p->out, static_cast<const T *>(p->hidden), static_cast<T *>(p->db), r, 1};
    if (p->da) jobs[count++] = {in.x, in.x_stride, p->in, static_cast<const T *>(g), static_cast<T *>(p->da), 1, p->in};
    if constexpr (f16) {
        ThinJob thin[2]{};
        for (uint32_t i = 0; i < count; i++) {
            thin[i] = {reinterpret_cast<const float *>(jobs[i].thin), static_cast<__half *>(work(l.halves[i])), static_cast<float *>(work(l.scale[i]))};
            jobs[i].thin = thin[i].to, jobs[i].scale = thin[i].scale;
        }
        rc = launch_thin(p, thin, count, tokens.order, start, cs);
        if (rc) return rc;
    }
    return launch_factor_grad<T>(p, jobs, count, tokens.order, start, cs);
}

API int lmz_gpu_ops_gave_up(void)
{
    const int rc = device_ready();
    if (rc) return rc;
    void *word = nullptr;
    CK("cudaGetSymbolAddress", cudaGetSymbolAddress(&word, g_gave_up));
    return taken_word(word);
}

API int lmz_gpu_project_dev(const lmz_projection *p, void *cuda_stream)
{
    int rc = check_projection(p);
    if (rc || p->tokens == 0) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    return p->dtype == LMZ_GPU_BF16 ? project_as<__nv_bfloat16>(p, cs) : project_as<__half>(p, cs);
}

API int lmz_gpu_project_grad_dev(const lmz_projection *p, void *cuda_stream)
{
    int rc = check_projection(p);
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    return p->dtype == LMZ_GPU_BF16 ? project_grad_as<__nv_bfloat16>(p, cs) : project_grad_as<__half>(p, cs);
}

template <class T>
static int merge_as(const void *w, uint64_t out, uint64_t in, uint64_t stride, const void *a, const void *b, unsigned rank, float scale, void *to,
                    cudaStream_t cs)
{
    MergeArgs<T> m{};
    m.w = static_cast<const T *>(w), m.a = static_cast<const T *>(a), m.b = static_cast<const T *>(b), m.out = static_cast<T *>(to);
    m.rows = out, m.cols = in, m.w_stride = stride, m.rank = rank, m.places = (rank + 15) & ~15u, m.scale = scale;
    m.a_even = on_boundary(a, in, in), m.b_even = on_boundary(b, rank, rank);
    return by_width<T>(vector_bytes(in * 2, {address(w), address(to), stride * 2}), [&](auto vec) {
        constexpr int VB = sizeof(vec.raw);
        static bool done[64];
        const int rc = opt_in_smem(k_merge<T, VB>, merge_smem_most(), done);
        if (rc) return rc;
        int sms = 0;
        const int failed = sm_count(&sms);
        if (failed) return failed;
        const uint64_t tiles = ((in + M_COLS - 1) / M_COLS) * ((out + M_ROWS - 1) / M_ROWS), room = (uint64_t)sms * (merge_smem(m.places) <= 113u << 10 ? 2 : 1);
        return launch("launch k_merge", k_merge<T, VB>, dim3(static_cast<unsigned>(std::min(tiles, room))), M_THREADS, merge_smem(m.places), cs, m);
    });
}

template <class T>
static int merge_wide_as(const void *w, uint64_t out, uint64_t in, uint64_t stride, const float *a, const float *b, unsigned rank, float scale, void *to,
                         cudaStream_t cs)
{
    const MergeWideArgs<T> m{static_cast<const T *>(w), a, b, static_cast<T *>(to), out, in, stride, rank, scale};
    const uint64_t tiles = ((in + MW_TILE - 1) / MW_TILE) * ((out + MW_TILE - 1) / MW_TILE);       // (below 2^28)
    const bool four = in % 4 == 0 && stride % 4 == 0 && (address(w) | address(to)) % (4 * sizeof(T)) == 0;
    return launch("launch k_merge_wide", four ? k_merge_wide<T, true> : k_merge_wide<T, false>, dim3(static_cast<unsigned>(tiles)), MW_THREADS, 0, cs, m);
}

API int lmz_gpu_merge_wide_dev(const void *d_weight, uint64_t out, uint64_t in, uint64_t weight_stride, const float *d_a, const float *d_b, unsigned rank,
                               float scale, int dtype, void *d_out, void *cuda_stream)
{
    lmz_projection p{};
    p.dtype = dtype == LMZ_GPU_F32 ? LMZ_GPU_BF16 : dtype, p.rank = rank, p.adapters = 1, p.in = in, p.out = out;
    int rc = check_projection(&p);
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    if (dtype == LMZ_GPU_F32) return merge_wide_as<float>(d_weight, out, in, weight_stride, d_a, d_b, rank, scale, d_out, cs);
    return dtype == LMZ_GPU_BF16 ? merge_wide_as<__nv_bfloat16>(d_weight, out, in, weight_stride, d_a, d_b, rank, scale, d_out, cs)
                                 : merge_wide_as<__half>(d_weight, out, in, weight_stride, d_a, d_b, rank, scale, d_out, cs);
}

API int lmz_gpu_merge_dev(const void *d_weight, uint64_t out, uint64_t in, uint64_t weight_stride, const void *d_a, const void *d_b, unsigned rank,
                          float scale, int dtype, void *d_out, void *cuda_stream)
{
    lmz_projection p{};
    p.dtype = dtype, p.rank = rank, p.adapters = 1, p.in = in, p.out = out;
    int rc = check_projection(&p);
    if (rc) return rc;
    rc = device_ready();
    if (rc) return rc;
    const cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
    return dtype == LMZ_GPU_BF16 ? merge_as<__nv_bfloat16>(d_weight, out, in, weight_stride, d_a, d_b, rank, scale, d_out, cs)
                                 : merge_as<__half>(d_weight, out, in, weight_stride, d_a, d_b, rank, scale, d_out, cs);
}
