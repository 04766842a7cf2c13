// Launches, element types, alignments and tensor maps, as the operators' entry points need them (included by model_ops.cu and
// layer_ops.cu).
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

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

static uint64_t up8(uint64_t n) { return (n + 7) & ~7ull; }
static uint64_t up256(uint64_t n) { return (n + 255) & ~255ull; }

// Rows of 16-bit elements that TMA and 16-byte copies take as they lie.
static bool on_boundary(const void *p, uint64_t cols, uint64_t stride) { return address(p) % 16 == 0 && stride % 8 == 0 && stride >= cols; }

// A tensor map of planes x rows x cols elements (planes 0: of rows x cols): tiles of 128 bytes of a row with the 128-byte swizzle.
static int tile_map(CUtensorMap *map, const void *p, CUtensorMapDataType type, uint32_t bytes, uint64_t cols, uint64_t rows, uint64_t stride, uint32_t tile_rows,
                    uint64_t planes, uint64_t plane_stride, uint32_t tile_planes = 1)
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
    const cuuint64_t dims[3] = {cols, rows, planes}, strides[2] = {stride * bytes, plane_stride * bytes};
    const cuuint32_t box[3] = {ROW_BYTES / bytes, tile_rows, tile_planes}, steps[3] = {1, 1, 1};
    auto make = [&] {
        return encode(map, type, planes ? 3 : 2, const_cast<void *>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = make();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {                       // a thread that has launched nothing yet (autograd's): the driver asks for its context
        int dev = 0;
        CK("cudaGetDevice", cudaGetDevice(&dev));
        CK("cudaSetDevice", cudaSetDevice(dev));
        r = make();
    }
    return r == CUDA_SUCCESS ? LMZ_GPU_OK : report(LMZ_GPU_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// The same of 16-bit elements, a plane's rows behind those of the plane before.
static int tensor_map(CUtensorMap *map, const void *p, bool bf16, uint64_t cols, uint64_t rows, uint64_t stride, uint32_t tile_rows, uint64_t planes = 0,
                      uint32_t tile_planes = 1)
{
    return tile_map(map, p, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, cols, rows, stride, tile_rows, planes, stride * rows, tile_planes);
}

static uint32_t tmem_columns(uint32_t n)
{
    uint32_t c = 32;
    while (c < n) c *= 2;
    return c;
}
