// fp8_linear.cu -- dense linear over e4m3 weights with one fp32 scale for each
// 128 x 128 block:
//   y[r, n] = bias[n] + sum over groups g of 128 columns of
//             s_x[r, g] * s_w[n / 128, g] * sum_{k in g} q_x[r, k] * q_w[n, k]
// with x quantised by row and group inside the call (or given as e4m3 with its
// scales).  The inner sum is exact products accumulated in fp32 by tcgen05
// (kind::f8f6f4); its scales differ from group to group, so each group's 128
// columns are one accumulation in TMEM that is read back, scaled and added to
// fp32 registers while the next group's runs into another TMEM buffer.
//
// Few rows (fp8_stream_kernel): bound by the weights' bytes.  The weights are
// the M operand -- a 128-row tile of W is exactly one row of scale blocks, and
// it goes from HBM through TMA into swizzled shared memory and from there to
// the tensor core without touching a register -- and the rows of x are N.
// A cluster of CTAs splits k; its partial sums meet in distributed shared
// memory in rank order, so there is no workspace, no counter and no atomic,
// and results do not depend on timing.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "fp8.cuh"
#include "host.hpp"

namespace exl3 {

// Status bits of the fp8 linear kernels on this device (exl3_fp8_status).
__device__ uint32_t g_fp8_status = 0u;

constexpr int kFsEpiWarps = 4;       // warps 0-3: TMEM lanes 32 w ..
constexpr int kFsXWarps = 4;         // warps 4-7: quantise x into the ring
constexpr int kFsProducerWarp = 8;
constexpr int kFsMmaWarp = 9;
constexpr int kFsThreads = 320;
constexpr int kFsMaxStages = 12;
constexpr int kFsMaxBufs = 8;
constexpr int kFsMaxCluster = 8;

struct FsParams {
    CUtensorMap wmap;            // W [n][k] bytes, box [128 k, 128 n], 128-byte swizzle
    const void* x;
    int64_t ldx;
    const float* xs;             // scales of an e4m3 x [rows][groups], else null
    const float* ws;             // [ceil(n / 128)][groups]
    const void* bias;
    void* y;
    int64_t ldy;
    int x_dtype, y_dtype, bias_dtype, pow2, xvec;
    int rows, n, k, groups;
    int stages, cluster;
};

template <int NT>
struct FsLayout {
    static constexpr int kXBytes = NT * 128;
    static constexpr int kStage = (int) kFp8WTile + kXBytes;
    static constexpr int kBufs = NT <= 16 ? 8 : NT <= 32 ? 4 : 2;
    static constexpr int kTmemCols = NT * kBufs;           // 128
};

template <int NT>
struct FsHead {
    uint64_t full[kFsMaxStages];
    uint64_t empty[kFsMaxStages];
    uint64_t tfull[kFsMaxBufs];
    uint64_t tempty[kFsMaxBufs];
    uint32_t tmem;
    uint32_t pad[3];
    float fac[kFsMaxStages][NT];          // s_x * s_w of the stage's rows
};

template <int NT>
__global__ void __launch_bounds__(kFsThreads, NT <= 32 ? 2 : 1) fp8_stream_kernel(const __grid_constant__ FsParams p) {
    using L = FsLayout<NT>;
    extern __shared__ uint8_t fs_raw[];
    uint8_t* ring = fs_raw + ((1024u - (smem_u32(fs_raw) & 1023u)) & 1023u);
    FsHead<NT>& H = *reinterpret_cast<FsHead<NT>*>(ring + p.stages * L::kStage);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = p.cluster, rank = S > 1 ? (int) cluster_rank() : 0;
    const int tile = (int) blockIdx.x / S;
    const int n0 = tile * 128, row0 = (int) blockIdx.y * NT;
    const int rows = min(NT, p.rows - row0);
    const int ncols = (rows + 15) & ~15;                   // MMA N
    const int kbeg = rank * p.groups / S, nsteps = (rank + 1) * p.groups / S - kbeg;
    uint32_t* status = &g_fp8_status;

    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&H.full[s], 1 + rows);
            mbar_init(&H.empty[s], 1 + kFsEpiWarps);
        }
        for (int b = 0; b < L::kBufs; ++b) { mbar_init(&H.tfull[b], 1); mbar_init(&H.tempty[b], kFsEpiWarps); }
        fence_barrier_init();
    }
    if (warp == kFsMmaWarp) tmem_alloc(&H.tmem, L::kTmemCols);
    // L2 prefetch ahead of the wait for the previous kernel: it brings no value
    // into this SM, so weights that kernel may have written are still read later.
    if (warp == kFsProducerWarp && lane < min(nsteps, p.stages)) tma_prefetch_2d(&p.wmap, (kbeg + lane) * 128, n0);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = H.tmem;
    pdl_wait();

    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.f;

    if (warp == kFsProducerWarp) {
        if (lane == 0) {
            int issued = 0;
            for (int s = 0; s < nsteps; ++s) {
                const int st = s % p.stages;
                if (!mbar_wait(&H.empty[st], ((s / p.stages) + 1u) & 1u, status)) break;
                mbar_arrive_expect_tx(&H.full[st], kFp8WTile);
                tma_load_2d(ring + st * L::kStage, &p.wmap, (kbeg + s) * 128, n0, &H.full[st]);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - p.stages); i < issued; ++i)
                if (!mbar_wait(&H.full[i % p.stages], (i / p.stages) & 1u, status)) break;
        }
    } else if (warp == kFsMmaWarp) {
        if (lane == 0) {
            const uint32_t id = idesc_f16(128, ncols);
            const uint64_t desc0 = sdesc_sw128(smem_u32(ring));
            for (int s = 0; s < nsteps; ++s) {
                const int st = s % p.stages, b = s % L::kBufs;
                if (!mbar_wait(&H.full[st], (s / p.stages) & 1u, status)) break;
                if (!mbar_wait(&H.tempty[b], ((s / L::kBufs) + 1u) & 1u, status)) break;
                tc_fence_after();
                const uint64_t wd = desc0 + (uint64_t) (st * (L::kStage >> 4)), xd = wd + (kFp8WTile >> 4);
#pragma unroll
                for (int q = 0; q < 4; ++q) tc_mma_f8(tmem + b * NT, wd + 2 * q, xd + 2 * q, id, q);
                tc_commit(&H.empty[st]);
                tc_commit(&H.tfull[b]);
            }
        }
    } else if (warp >= kFsEpiWarps) {
        // x: one warp for each (step, row), four elements a lane.  Rows of the B
        // operand behind the last one hold whatever the stage held: each is a
        // column of D of its own, and those columns are never used.
        const int xw = warp - kFsEpiWarps, items = nsteps * rows, k4 = lane * 4;
        auto fetch = [&](int i) {
            const int col = (kbeg + i / rows) * 128 + k4;
            const int64_t at = (int64_t) (row0 + i % rows) * p.ldx + col;
            if (p.xvec) return col < p.k ? load_raw4(p.x, p.x_dtype, at) : make_uint4(0u, 0u, 0u, 0u);
            return load_raw4_tail(p.x, p.x_dtype, at, p.k - col);
        };
        uint4 next = xw < items ? fetch(xw) : make_uint4(0u, 0u, 0u, 0u);
        for (int i = xw; i < items; i += kFsXWarps) {
            const uint4 raw = next;
            if (i + kFsXWarps < items) next = fetch(i + kFsXWarps);
            const int s = i / rows, r = i % rows, st = s % p.stages;
            float sx;
            uint32_t q;
            if (p.x_dtype == kDtE4M3) {
                q = raw.x;
                sx = __ldg(p.xs + (int64_t) (row0 + r) * p.groups + kbeg + s);
            } else {
                float v[4];
                unpack4(raw, p.x_dtype, v);
                sx = fp8_scale(__reduce_max_sync(0xffffffffu, abs_bits4(v)), p.pow2);
                q = fp8_quant4(v, sx, __frcp_rn(sx), p.pow2);
            }
            const float f = sx * __ldg(p.ws + (int64_t) tile * p.groups + kbeg + s);
            if (!mbar_wait_lanes(&H.empty[st], ((s / p.stages) + 1u) & 1u, status)) break;
            *reinterpret_cast<uint32_t*>(ring + st * L::kStage + kFp8WTile + sw128_byte(r, k4)) = q;
            if (lane == 0) H.fac[st][r] = f;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&H.full[st]);
        }
    } else {
        // scale and add: thread = weight row, registers = rows of x
        for (int s = 0; s < nsteps; ++s) {
            const int st = s % p.stages, b = s % L::kBufs;
            if (!mbar_wait_lanes(&H.tfull[b], (s / L::kBufs) & 1u, status)) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < NT / 16; ++c) {
                if (c * 16 >= ncols) break;
                float v[16];
                tc_ld16(tmem + ((uint32_t) (warp * 32) << 16) + (uint32_t) (b * NT + c * 16), v);
                const float4* f4 = reinterpret_cast<const float4*>(&H.fac[st][c * 16]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 f = f4[q];
                    acc[c * 16 + q * 4 + 0] = fmaf(v[q * 4 + 0], f.x, acc[c * 16 + q * 4 + 0]);
                    acc[c * 16 + q * 4 + 1] = fmaf(v[q * 4 + 1], f.y, acc[c * 16 + q * 4 + 1]);
                    acc[c * 16 + q * 4 + 2] = fmaf(v[q * 4 + 2], f.z, acc[c * 16 + q * 4 + 2]);
                    acc[c * 16 + q * 4 + 3] = fmaf(v[q * 4 + 3], f.w, acc[c * 16 + q * 4 + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&H.tempty[b]);
                mbar_arrive(&H.empty[st]);
            }
        }
    }

    // ---------------------------------------------------------------- output
    auto put = [&](int j, int i, float v) {
        const int col = n0 + i;
        if (col >= p.n) return;
        if (p.bias != nullptr) v += load_f32(p.bias, p.bias_dtype, col);
        store_out(p.y, p.y_dtype, (int64_t) (row0 + j) * p.ldy + col, v);
    };
    if (S == 1) {
        if (warp < kFsEpiWarps) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (j < rows) put(j, tid, acc[j]);
        }
        __syncthreads();
    } else {
        __syncthreads();                                   // every stage has been read: the ring is free
        float* part = reinterpret_cast<float*>(ring);       // [rows][128]
        if (warp < kFsEpiWarps) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (j < rows) part[j * 128 + tid] = acc[j];
        }
        cluster_sync_all();
        const int total = rows * 128, per = (total + S - 1) / S;
        for (int i = rank * per + tid; i < min(total, (rank + 1) * per); i += kFsThreads) {
            float v = 0.f;
            for (int c = 0; c < S; ++c) v += ld_dsmem(smem_u32(part + i), (uint32_t) c);
            put(i >> 7, i & 127, v);
        }
        cluster_sync_all();                                // no CTA leaves while its sums are being read
    }
    if (warp == kFsMmaWarp) {
        tc_fence_after();
        tmem_free(tmem, L::kTmemCols);
    }
}

// ------------------------------------------------------------------ host side
namespace {

PFN_cuTensorMapEncodeTiled_v12000 fp8_encoder() {
    static std::once_flag once;
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    });
    return fn;
}

}  // namespace

// [rows][cols] bytes of pitch ld; box 128 columns x box_rows, 128-byte swizzle;
// what lies outside reads as zero.
int fp8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, const char* what) {
    auto encode = fp8_encoder();
    EXL3_REQUIRE(encode != nullptr, EXL3_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available", what);
    const cuuint64_t dims[2] = {(cuuint64_t) cols, (cuuint64_t) rows};
    const cuuint64_t strides[1] = {(cuuint64_t) ld};
    const cuuint32_t box[2] = {128u, (cuuint32_t) box_rows};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    EXL3_REQUIRE(r == CUDA_SUCCESS, EXL3_ERR_CUDA, "%s: tensor map failed (%d)", what, (int) r);
    return EXL3_OK;
}

namespace {

// CTAs that split k: the largest power of two (a portable cluster) that keeps
// the grid within about two CTAs an SM and leaves every CTA two groups.
int fs_cluster(int64_t tiles, int groups) {
    int s = 1;
    while (s < kFsMaxCluster && tiles * s * 2 <= 296 && groups >= s * 4) s *= 2;
    return s;
}

template <int NT>
int fs_launch(FsParams& p, cudaStream_t stream) {
    using L = FsLayout<NT>;
    const int64_t tiles = ((int64_t) p.n + 127) / 128, rtiles = ((int64_t) p.rows + NT - 1) / NT;
    p.cluster = fs_cluster(tiles * rtiles, p.groups);
    const int steps = (p.groups + p.cluster - 1) / p.cluster;
    // two CTAs share an SM: at most about 112 KB each; at least the partial sums' room
    const int head = 1024 + (int) sizeof(FsHead<NT>);
    int stages = (112 * 1024 - head) / L::kStage;
    if (stages > kFsMaxStages) stages = kFsMaxStages;
    const int least = (NT * 512 + L::kStage - 1) / L::kStage;
    if (stages > steps) stages = steps < least ? least : steps;
    p.stages = stages;
    const int smem = head + stages * L::kStage;
    static std::once_flag once[64];
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    cudaError_t attr = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr = cudaFuncSetAttribute(fp8_stream_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 116 * 1024);
    });
    EXL3_CUDA(attr);
    EXL3_REQUIRE(tiles * p.cluster <= INT32_MAX && rtiles <= 65535, EXL3_ERR_UNSUPPORTED, "exl3_fp8_linear: matrix too large");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (tiles * p.cluster), (unsigned) rtiles);
    cfg.blockDim = dim3(kFsThreads);
    cfg.dynamicSmemBytes = (size_t) smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned) p.cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, fp8_stream_kernel<NT>, p));
    return EXL3_OK;
}

}  // namespace
}  // namespace exl3

extern "C" int exl3_fp8_linear(const void* x, int x_dtype, int64_t ldx, const float* x_scale, int64_t rows, int64_t k,
                               int64_t n, const void* w, int64_t ldw, const float* w_scale, const void* bias,
                               int bias_dtype, void* y, int y_dtype, int64_t ldy, int pow2, void* scratch,
                               int64_t scratch_bytes, void* stream) {
    using namespace exl3;
    EXL3_REQUIRE(rows >= 0 && k >= 1 && n >= 1 && rows <= INT32_MAX / 2 && k <= INT32_MAX / 2 && n <= INT32_MAX / 2,
                 EXL3_ERR_ARG, "exl3_fp8_linear: rows must be >= 0, k and n >= 1, each below 2^30");
    EXL3_REQUIRE(x_dtype >= 0 && x_dtype <= 3 && y_dtype >= 0 && y_dtype <= 2 && (bias == nullptr || (bias_dtype >= 0 && bias_dtype <= 2)),
                 EXL3_ERR_ARG, "exl3_fp8_linear: dtypes must be fp16, bf16 or fp32 (x: e4m3 too)");
    EXL3_REQUIRE(ldx >= k && ldw >= k && ldy >= n, EXL3_ERR_ARG, "exl3_fp8_linear: leading dimensions are too small");
    if (rows == 0) return EXL3_OK;
    EXL3_REQUIRE(x && w && w_scale && y, EXL3_ERR_ARG, "exl3_fp8_linear: null pointer");
    EXL3_REQUIRE((x_dtype == EXL3_DTYPE_E4M3) == (x_scale != nullptr), EXL3_ERR_ARG,
                 "exl3_fp8_linear: x_scale goes with an e4m3 x, and only with one");
    EXL3_REQUIRE(aligned16(w) && ldw % 16 == 0, EXL3_ERR_ARG, "exl3_fp8_linear: weight rows must be 16-byte aligned");
    (void) scratch;
    (void) scratch_bytes;
    FsParams p{};
    const int rc = fp8_map(&p.wmap, w, n, k, ldw, 128, "exl3_fp8_linear");
    if (rc != EXL3_OK) return rc;
    p.x = x; p.ldx = ldx; p.xs = x_scale; p.ws = w_scale; p.bias = bias; p.y = y; p.ldy = ldy;
    p.x_dtype = x_dtype; p.y_dtype = y_dtype; p.bias_dtype = bias_dtype; p.pow2 = pow2 != 0;
    p.rows = (int) rows; p.n = (int) n; p.k = (int) k; p.groups = (int) ((k + 127) / 128);
    const int es = x_dtype == 2 ? 4 : x_dtype == 3 ? 1 : 2;
    p.xvec = k % 4 == 0 && ldx % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * es) == 0;
    auto s = static_cast<cudaStream_t>(stream);
    if (rows <= 16) return fs_launch<16>(p, s);
    if (rows <= 32) return fs_launch<32>(p, s);
    return fs_launch<64>(p, s);
}

extern "C" int64_t exl3_fp8_linear_scratch_bytes(int64_t rows, int64_t k, int64_t n, int x_dtype) {
    if (rows < 0 || k < 1 || n < 1 || x_dtype < 0 || x_dtype > 3) return -1;
    return 0;
}

extern "C" int exl3_fp8_status(int clear, uint32_t* status, void* stream) {
    using namespace exl3;
    EXL3_REQUIRE(status, EXL3_ERR_ARG, "exl3_fp8_status: null pointer");
    auto s = static_cast<cudaStream_t>(stream);
    EXL3_CUDA(cudaMemcpyFromSymbolAsync(status, g_fp8_status, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, s));
    EXL3_CUDA(cudaStreamSynchronize(s));
    if (clear) {
        const uint32_t zero = 0u;
        EXL3_CUDA(cudaMemcpyToSymbolAsync(g_fp8_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s));
        EXL3_CUDA(cudaStreamSynchronize(s));
    }
    return EXL3_OK;
}
