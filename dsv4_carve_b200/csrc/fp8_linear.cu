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
// Few rows (fp8_stream_kernel, fp8_rows_kernel): bound by the weights' bytes.  The weights are
// the M operand -- a 128-row tile of W is exactly one row of scale blocks, and
// it goes from HBM through TMA into swizzled shared memory and from there to
// the tensor core without touching a register -- and the rows of x are N.
// A cluster of CTAs splits k; its partial sums meet in distributed shared
// memory in rank order, so there is no counter and no atomic, and results do
// not depend on timing.
//
// Many rows (fp8_gemm_kernel): bound by the tensor cores.  x is quantised by a
// kernel of its own (launched just before, overlapped) and its rows are the M
// operand of a pair of CTAs (cta_group::2, 256 rows x NW weight rows), so the
// factor s_x * s_w is one number a thread for each group of 128 columns and
// the scaling is one FMA a value.  8192 x 4096 x 4096: 126 us without the
// quantiser, 2.18 PFLOP/s, held by L2 -> shared memory (8.4 TB/s) and power.
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
constexpr int kFsMaxCluster = 8;

struct FsParams {
    CUtensorMap wmap;            // W [n][k] bytes, box [128 k, 128 n], 128-byte swizzle
    CUtensorMap xmap;            // e4m3 x [rows][k], box [128 k, NT] (fp8_rows_kernel)
    const void* x;
    int64_t ldx;
    const float* xs;             // scales of an e4m3 x: xs[row * xsr + group * xsg], else null
    int64_t xsr, xsg;
    const float* ws;             // [ceil(n / 128)][groups]
    const void* bias;
    void* y;
    int64_t ldy;
    int x_dtype, y_dtype, bias_dtype, pow2, xvec;
    int rows, n, k, groups;
    int stages, cluster;
    int early;                   // nothing still running can write the weights
};

// Sums of a cluster's partial tiles part[rows][128], in rank order; this CTA's
// share of the outputs goes to `put`, four columns a thread or, where that would
// leave most threads idle, one.
template <bool WIDE, typename Put>
__device__ __forceinline__ void cluster_reduce(const float* part, int rows, int S, int rank, int tid, int threads, Put&& put) {
    cluster_sync_all();
    constexpr int V = WIDE ? 4 : 1;
    const int total = rows * 128 / V, per = (total + S - 1) / S;
    for (int i = rank * per + tid; i < min(total, (rank + 1) * per); i += threads) {
        const uint32_t at = smem_u32(part + V * i);
        if constexpr (WIDE) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f), w[kFsMaxCluster];
#pragma unroll
            for (int c = 0; c < kFsMaxCluster; ++c) w[c] = c < S ? ld_dsmem4(at, (uint32_t) c) : v;
#pragma unroll
            for (int c = 0; c < kFsMaxCluster; ++c) { v.x += w[c].x; v.y += w[c].y; v.z += w[c].z; v.w += w[c].w; }
            put(i >> 5, (i & 31) * 4, v.x);
            put(i >> 5, (i & 31) * 4 + 1, v.y);
            put(i >> 5, (i & 31) * 4 + 2, v.z);
            put(i >> 5, (i & 31) * 4 + 3, v.w);
        } else {
            float v = 0.f;
            for (int c = 0; c < S; ++c) v += ld_dsmem(at, (uint32_t) c);
            put(i >> 7, i & 127, v);
        }
    }
    cluster_sync_all();                                    // no CTA leaves while its sums are being read
}

// ------------------------------------------------------------------ up to 8 rows
// x is quantised inside the kernel: warps 4-7 write it into the ring beside the
// weights.  One launch, 6.4 us for one row x 4096 x 4096 back to back (2.6 TB/s);
// what it takes is the chain of one launch (x from L2, quantising, MMA, the
// cluster's sum), not the weights' time.
struct FsLayout {
    static constexpr int NT = 16;                          // MMA N
    static constexpr int kStage = (int) kFp8WTile + NT * 128;
    static constexpr int kBufs = 8;
    static constexpr int kTmemCols = NT * kBufs;
};

struct FsHead {
    uint64_t full[kFsMaxStages];
    uint64_t empty[kFsMaxStages];
    uint64_t tfull[FsLayout::kBufs];
    uint64_t tempty[FsLayout::kBufs];
    uint32_t tmem;
    alignas(16) float fac[kFsMaxStages][FsLayout::NT];     // s_x * s_w of the stage's rows
};

__global__ void __launch_bounds__(kFsThreads, 2) fp8_stream_kernel(const __grid_constant__ FsParams p) {
    using L = FsLayout;
    constexpr int NT = L::NT;
    extern __shared__ uint8_t fs_raw[];
    uint8_t* ring = fs_raw + ((1024u - (smem_u32(fs_raw) & 1023u)) & 1023u);
    FsHead& H = *reinterpret_cast<FsHead*>(ring + p.stages * L::kStage);
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const int S = p.cluster, rank = S > 1 ? (int) cluster_rank() : 0;
    const int tile = (int) blockIdx.x / S;
    const int n0 = tile * 128, row0 = (int) blockIdx.y * NT;
    const int rows = min(NT, p.rows - row0);
    const int ncols = (rows + 15) & ~15;                   // MMA N
    const int kbeg = rank * p.groups / S, nsteps = (rank + 1) * p.groups / S - kbeg;
    uint32_t* status = &g_fp8_status;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&H.full[s], 1 + (rows + 3) / 4);
            mbar_init(&H.empty[s], 1 + kFsEpiWarps);
        }
        for (int b = 0; b < L::kBufs; ++b) { mbar_init(&H.tfull[b], 1); mbar_init(&H.tempty[b], kFsEpiWarps); }
        fence_barrier_init();
    }
    if (warp == kFsMmaWarp) tmem_alloc(&H.tmem, L::kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, H.tmem, 0);

    float acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = 0.f;

    if (warp == kFsProducerWarp) {
        const int ahead = min(nsteps, p.stages);
        auto weights = [&](int s) {
            const int st = s % p.stages;
            mbar_arrive_expect_tx(&H.full[st], kFp8WTile);
            tma_load_2d(ring + st * L::kStage, &p.wmap, (kbeg + s) * 128, n0, &H.full[st]);
        };
        // Ahead of the wait for the previous kernel, which may write the weights:
        // a prefetch into L2, which brings no value into this SM.
        if (lane < ahead) tma_prefetch_2d(&p.wmap, (kbeg + lane) * 128, n0);
        pdl_wait();
        if (lane == 0) {
            pdl_launch_dependents();
            int issued = 0;
            for (int s = 0; s < nsteps; ++s) {
                if (s >= p.stages && !mbar_wait(&H.empty[s % p.stages], ((s / p.stages) + 1u) & 1u, status)) break;
                weights(s);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - p.stages); i < issued; ++i)
                if (!mbar_wait(&H.full[i % p.stages], (i / p.stages) & 1u, status)) break;
        }
    } else if (warp == kFsMmaWarp) {
        pdl_wait();
        const uint32_t id = idesc_f16(128, ncols);
        const uint64_t desc0 = sdesc_sw128(smem_u32(ring));
        for (int s = 0; s < nsteps; ++s) {
            const int st = s % p.stages, b = s % L::kBufs;
            if (!mbar_poll2_lanes(&H.full[st], (s / p.stages) & 1u, &H.tempty[b], ((s / L::kBufs) + 1u) & 1u, status)) break;
            tc_fence_after();
            const uint64_t wd = desc0 + (uint64_t) (st * (L::kStage >> 4)), xd = wd + (kFp8WTile >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int q = 0; q < 4; ++q) tc_mma_f8(tmem + b * NT, wd + 2 * q, xd + 2 * q, id, q);
                tc_commit(&H.empty[st]);
                tc_commit(&H.tfull[b]);
            }
        }
    } else if (warp >= kFsEpiWarps) {
        // x: one warp for each step and four rows.  Rows of the B operand behind
        // the last one hold whatever the stage held: each is a column of D of its
        // own, and those columns are never used.
        pdl_wait();
        const int xw = warp - kFsEpiWarps, quads = (rows + 3) >> 2, items = nsteps * quads;
        XRows next;
        auto fetch = [&](int i) {
            const int r = (i % quads) * 4, cnt = min(4, rows - r), lr = XRows::row(cnt, lane);
            const int col = (kbeg + i / quads) * 128 + XRows::col(cnt, lane);
            next.load(cnt, p.x, p.x_dtype, (int64_t) (row0 + r + lr) * p.ldx + col, lr < cnt ? p.k - col : 0, p.xvec);
        };
        if (xw < items) fetch(xw);
        for (int i = xw; i < items; i += kFsXWarps) {
            const XRows cur = next;
            if (i + kFsXWarps < items) fetch(i + kFsXWarps);
            const int s = i / quads, r = (i % quads) * 4, cnt = min(4, rows - r), lr = XRows::row(cnt, lane), st = s % p.stages;
            const float ws = __ldg(p.ws + (int64_t) tile * p.groups + kbeg + s);
            const bool head = lr < cnt && (cnt == 1 ? lane == 0 : (lane & 7) == 0);
            float sx = 0.f;
            uint4 q = cur.r[0];
            if (p.x_dtype != kDtE4M3) q = cur.quantize(cnt, p.x_dtype, p.pow2, sx);
            else if (head) sx = __ldcg(p.xs + (row0 + r + lr) * p.xsr + (kbeg + s) * p.xsg);
            if (!mbar_wait_lanes(&H.empty[st], ((s / p.stages) + 1u) & 1u, status)) break;
            if (lr < cnt) XRows::store(cnt, ring + st * L::kStage + kFp8WTile, r + lr, lane, q);
            if (head) H.fac[st][r + lr] = sx * ws;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&H.full[st]);
        }
    } else {
        // scale and add: thread = weight row, registers = rows of x
        pdl_wait();
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
        cluster_reduce<false>(part, rows, S, rank, tid, kFsThreads, put);
    }
    if (warp == kFsMmaWarp) {
        tc_fence_after();
        tmem_free(tmem, L::kTmemCols);
    }
}

// ------------------------------------------------------------------ up to some hundred rows
// x comes in e4m3 through TMA beside the weights.  Eight epilogue warps (four for
// 16 rows) share the columns, i.e. the rows of x; each keeps its columns' factors
// in shared memory of its own, loaded two steps ahead.
constexpr int kFrProducerWarp = 8;
constexpr int kFrMmaWarp = 9;
constexpr int kFrThreads = 320;

template <int NT>
struct FrLayout {
    static constexpr int kHalves = NT >= 32 ? 2 : 1;
    static constexpr int kCols = NT / kHalves;             // columns of an epilogue warp: 16, 16, 32, 64
    static constexpr int kStage = (int) kFp8WTile + NT * 128;
    static constexpr int kBufs = NT <= 32 ? 4 : 2;
    static constexpr int kTmemCols = NT * kBufs;           // 64 .. 256
    static constexpr int kCtas = NT <= 64 ? 2 : 1;         // that share an SM
};

template <int NT>
struct FrHead {
    uint64_t full[kFsMaxStages];
    uint64_t done[kFsMaxStages];                           // the stage's MMAs: it may be refilled, and its sums be read
    uint64_t tempty[4];
    uint32_t tmem;
    alignas(16) float fac[8][2][FrLayout<NT>::kCols];
};

template <int NT>
__global__ void __launch_bounds__(kFrThreads, FrLayout<NT>::kCtas) fp8_rows_kernel(const __grid_constant__ FsParams p) {
    using L = FrLayout<NT>;
    extern __shared__ uint8_t fr_raw[];
    uint8_t* ring = fr_raw + ((1024u - (smem_u32(fr_raw) & 1023u)) & 1023u);
    FrHead<NT>& H = *reinterpret_cast<FrHead<NT>*>(ring + p.stages * L::kStage);
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const int S = p.cluster, rank = S > 1 ? (int) cluster_rank() : 0;
    const int tile = (int) blockIdx.x / S;
    const int n0 = tile * 128, row0 = (int) blockIdx.y * NT;
    const int rows = min(NT, p.rows - row0);
    const int ncols = (rows + 15) & ~15;                   // MMA N
    const int kbeg = rank * p.groups / S, nsteps = (rank + 1) * p.groups / S - kbeg;
    uint32_t* status = &g_fp8_status;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) { mbar_init(&H.full[s], 1); mbar_init(&H.done[s], 1); }
        for (int b = 0; b < L::kBufs; ++b) mbar_init(&H.tempty[b], 4 * L::kHalves);
        fence_barrier_init();
    }
    if (warp == kFrMmaWarp) tmem_alloc(&H.tmem, L::kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, H.tmem, 0);
    const int half = warp >> 2, lg = warp & 3, j0 = half * L::kCols;   // epilogue warps
    float acc[L::kCols];
#pragma unroll
    for (int j = 0; j < L::kCols; ++j) acc[j] = 0.f;

    if (warp == kFrProducerWarp) {
        const int ahead = min(nsteps, p.stages);
        auto weights = [&](int s) {
            const int st = s % p.stages;
            mbar_arrive_expect_tx(&H.full[st], L::kStage);
            tma_load_2d(ring + st * L::kStage, &p.wmap, (kbeg + s) * 128, n0, &H.full[st]);
        };
        // Ahead of the wait for the previous kernel: the weights themselves when it
        // is the quantiser of this call, behind whose own wait this kernel started;
        // otherwise it may write them, and a prefetch into L2 has to do.
        if (p.early) {
            if (lane == 0) for (int s = 0; s < ahead; ++s) weights(s);
        } else if (lane < ahead) {
            tma_prefetch_2d(&p.wmap, (kbeg + lane) * 128, n0);
        }
        pdl_wait();
        if (lane == 0) {
            pdl_launch_dependents();
            fence_proxy_async_global();
            int issued = 0;
            for (int s = 0; s < nsteps; ++s) {
                const int st = s % p.stages;
                if (s >= p.stages && !mbar_wait(&H.done[st], ((s / p.stages) + 1u) & 1u, status)) break;
                if (s >= ahead || !p.early) weights(s);
                tma_load_2d(ring + st * L::kStage + kFp8WTile, &p.xmap, (kbeg + s) * 128, row0, &H.full[st]);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - p.stages); i < issued; ++i)
                if (!mbar_wait(&H.full[i % p.stages], (i / p.stages) & 1u, status)) break;
        }
    } else if (warp == kFrMmaWarp) {
        pdl_wait();
        const uint32_t id = idesc_f16(128, ncols);
        const uint64_t desc0 = sdesc_sw128(smem_u32(ring));
        for (int s = 0; s < nsteps; ++s) {
            const int st = s % p.stages, b = s % L::kBufs;
            if (!mbar_poll2_lanes(&H.full[st], (s / p.stages) & 1u, &H.tempty[b], ((s / L::kBufs) + 1u) & 1u, status)) break;
            tc_fence_after();
            const uint64_t wd = desc0 + (uint64_t) (st * (L::kStage >> 4)), xd = wd + (kFp8WTile >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int q = 0; q < 4; ++q) tc_mma_f8(tmem + b * NT, wd + 2 * q, xd + 2 * q, id, q);
                tc_commit(&H.done[st]);
            }
        }
    } else if (half < L::kHalves) {
        // scale and add: thread = weight row, registers = rows of x
        pdl_wait();
        constexpr int NF = (L::kCols + 31) / 32;
        struct Fac { float f[NF], w; };
        auto load = [&](int s) {
            Fac v;
            v.w = s < nsteps ? __ldg(p.ws + (int64_t) tile * p.groups + kbeg + s) : 0.f;
#pragma unroll
            for (int h = 0; h < NF; ++h) {
                const int j = h * 32 + lane;
                v.f[h] = s < nsteps && j < L::kCols && j0 + j < rows ? __ldcg(p.xs + (row0 + j0 + j) * p.xsr + (kbeg + s) * p.xsg) : 0.f;
            }
            return v;
        };
        Fac v0 = load(0), v1 = load(1);
        const uint32_t tcol = tmem + ((uint32_t) (lg * 32) << 16) + (uint32_t) j0;
        for (int s = 0; s < nsteps; ++s) {
            const int st = s % p.stages, b = s % L::kBufs;
            float* fac = H.fac[warp][s & 1];               // the other one may still be read by slower lanes
#pragma unroll
            for (int h = 0; h < NF; ++h)
                if (h * 32 + lane < L::kCols) fac[h * 32 + lane] = v0.f[h] * v0.w;
            v0 = v1;
            v1 = load(s + 2);
            __syncwarp();
            if (!mbar_wait_lanes(&H.done[st], (s / p.stages) & 1u, status)) break;
            tc_fence_after();
            const float4* f4 = reinterpret_cast<const float4*>(fac);
            if constexpr (L::kCols == 16) {
                if (j0 < ncols) {
                    float v[16];
                    tc_ld16(tcol + (uint32_t) (b * NT), v);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 f = f4[q];
                        acc[4 * q] = fmaf(v[4 * q], f.x, acc[4 * q]);
                        acc[4 * q + 1] = fmaf(v[4 * q + 1], f.y, acc[4 * q + 1]);
                        acc[4 * q + 2] = fmaf(v[4 * q + 2], f.z, acc[4 * q + 2]);
                        acc[4 * q + 3] = fmaf(v[4 * q + 3], f.w, acc[4 * q + 3]);
                    }
                }
            } else {
                constexpr int NC = L::kCols / 32;
                if (j0 < ncols) {
                    uint32_t v[NC][32];
#pragma unroll
                    for (int c = 0; c < NC; ++c) tc_ld32_issue(tcol + (uint32_t) (b * NT + c * 32), v[c]);
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        tc_ld_wait(v[c]);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const float4 f = f4[c * 8 + q];
                            float* o = &acc[c * 32 + 4 * q];
                            o[0] = fmaf(__uint_as_float(v[c][4 * q]), f.x, o[0]);
                            o[1] = fmaf(__uint_as_float(v[c][4 * q + 1]), f.y, o[1]);
                            o[2] = fmaf(__uint_as_float(v[c][4 * q + 2]), f.z, o[2]);
                            o[3] = fmaf(__uint_as_float(v[c][4 * q + 3]), f.w, o[3]);
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&H.tempty[b]);
        }
    } else {
        pdl_wait();
    }

    auto put = [&](int j, int i, float v) {
        const int col = n0 + i;
        if (col >= p.n) return;
        if (p.bias != nullptr) v += load_f32(p.bias, p.bias_dtype, col);
        store_out(p.y, p.y_dtype, (int64_t) (row0 + j) * p.ldy + col, v);
    };
    const bool epi = half < L::kHalves;
    if (S == 1) {
        if (epi) {
#pragma unroll
            for (int j = 0; j < L::kCols; ++j)
                if (j0 + j < rows) put(j0 + j, lg * 32 + lane, acc[j]);
        }
        __syncthreads();
    } else {
        __syncthreads();                                   // every stage has been read: the ring is free
        float* part = reinterpret_cast<float*>(ring);       // [rows][128]
        if (epi) {
#pragma unroll
            for (int j = 0; j < L::kCols; ++j)
                if (j0 + j < rows) part[(j0 + j) * 128 + lg * 32 + lane] = acc[j];
        }
        cluster_reduce<true>(part, rows, S, rank, tid, kFrThreads, put);
    }
    if (warp == kFrMmaWarp) {
        tc_fence_after();
        tmem_free(tmem, L::kTmemCols);
    }
}

// ------------------------------------------------------------------ many rows
constexpr int kFgEpiWarps = 8;       // warp w: TMEM lanes 32 (w % 4), column half w / 4
constexpr int kFgProducerWarp = 8;
constexpr int kFgMmaWarp = 9;
constexpr int kFgThreads = 384;      // warps 10, 11 fill the third warpgroup
constexpr int kFgTmemCols = 512;

struct FgParams {
    CUtensorMap xmap;            // e4m3 x [rows][k], box [128 k, 128 rows]
    CUtensorMap wmap;            // W [n][k], box [128 k, NW / 2]
    CUtensorMap ymap;            // y [rows][n], box [128 bytes, 32 rows] (yvec)
    const float* xs;             // xs[row * xsr + group * xsg]
    const float* ws;             // [ceil(n / 128)][groups]
    const void* bias;
    void* y;
    int64_t ldy, xsr, xsg;
    int y_dtype, bias_dtype, yvec, early;
    int rows, n, groups, ntiles, tiles;
};

template <int NW>
struct FgLayout {
    // Groups of 128 columns in a step.  Two with the narrow tile: a step's barriers
    // and its commit cost the issuing warp about as much as four MMAs of 256 x 128
    // (512 x 4096 x 4096: 15.2 us with one).
    static constexpr int kKS = NW == 256 ? 1 : 2;
    static constexpr int kA = 128 * 128, kB = NW / 2 * 128, kGroup = kA + kB, kStage = kKS * kGroup;
    static constexpr int kStages = NW == 256 ? 5 : 3;
    static constexpr int kBufs = kFgTmemCols / (NW * kKS);
    static constexpr int kCols = NW / 2;                   // columns of a thread
    static constexpr int kOut = 32 * 256;                  // 256 bytes of a warp's rows on their way out
    static constexpr int kSmem = 1024 + kStages * kStage + kFgEpiWarps * kOut + 512;
};

// Byte offset of 16-byte piece c (< 16) of row r in a warp's output buffer: two
// tiles of 32 rows x 128 bytes, each with the 128-byte swizzle.
__device__ __forceinline__ int fg_out(int r, int c) { return (c >> 3) * 4096 + r * 128 + (((c ^ r) & 7) << 4); }

template <int NW>
struct FgHead {
    uint64_t full[FgLayout<NW>::kStages];      // in the pair's first CTA: both CTAs' bytes
    uint64_t done[FgLayout<NW>::kStages];      // the stage's MMAs: it may be refilled, and its sums be read
    uint64_t tempty[FgLayout<NW>::kBufs];      // in the pair's first CTA: both CTAs' epilogues
    uint32_t tmem;
};

template <int NW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFgThreads, 1) fp8_gemm_kernel(const __grid_constant__ FgParams p) {
    using L = FgLayout<NW>;
    extern __shared__ uint8_t fg_raw[];
    uint8_t* ring = fg_raw + ((1024u - (smem_u32(fg_raw) & 1023u)) & 1023u);
    uint8_t* stage_out = ring + L::kStages * L::kStage;
    FgHead<NW>& H = *reinterpret_cast<FgHead<NW>*>(stage_out + kFgEpiWarps * L::kOut);
    static_assert(sizeof(FgHead<NW>) <= 512, "head must fit its slot");
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const int pair = (int) blockIdx.x >> 1, pairs = (int) gridDim.x >> 1;
    const int steps = (p.groups + L::kKS - 1) / L::kKS;                       // of a tile
    const int total = ((p.tiles - pair + pairs - 1) / pairs) * steps;         // of this pair
    auto groups_of = [&](int step) { return min(L::kKS, p.groups - step * L::kKS); };
    uint32_t* status = &g_fp8_status;

    if (tid == 0) {
        for (int s = 0; s < L::kStages; ++s) { mbar_init(&H.full[s], 1); mbar_init(&H.done[s], 1); }
        for (int b = 0; b < L::kBufs; ++b) mbar_init(&H.tempty[b], 2 * kFgEpiWarps);
        fence_barrier_init();
    }
    if (warp == kFgMmaWarp) tmem_alloc_pair(&H.tmem, kFgTmemCols);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, H.tmem, 0);

    if (warp == kFgProducerWarp) {
        regs_down();
        if (lane == 0) {
            int it = 0, ahead = 0;
            auto weights = [&](int st, int nt, int step) {
                const int n = groups_of(step);
                if (rank == 0) mbar_arrive_expect_tx(&H.full[st], 2 * n * L::kGroup);
                for (int q = 0; q < n; ++q)
                    tma_load_2d_pair(ring + st * L::kStage + q * L::kGroup + L::kA, &p.wmap, (step * L::kKS + q) * 128,
                                     nt * NW + (int) rank * (NW / 2), mapa_u32(smem_u32(&H.full[st]), 0));
            };
            if (p.early) {
                // weights ahead of the quantiser's end: this kernel started behind its wait for all before
                const int nt = pair % p.ntiles;
                for (; ahead < min(L::kStages, steps); ++ahead) weights(ahead, nt, ahead);
            }
            pdl_wait();
            pdl_launch_dependents();
            fence_proxy_async_global();
            bool ok = true;
            for (int t = pair; t < p.tiles && ok; t += pairs) {
                const int nt = t % p.ntiles, row = t / p.ntiles * 256 + (int) rank * 128;
                for (int step = 0; step < steps; ++step, ++it) {
                    const int st = it % L::kStages;
                    if (it >= L::kStages) {
                        ok = mbar_poll(&H.done[st], ((it / L::kStages) + 1u) & 1u, status);
                        if (!ok) break;
                    }
                    if (it >= ahead) weights(st, nt, step);
                    for (int q = 0; q < groups_of(step); ++q)
                        tma_load_2d_pair(ring + st * L::kStage + q * L::kGroup, &p.xmap, (step * L::kKS + q) * 128, row,
                                         mapa_u32(smem_u32(&H.full[st]), 0));
                }
            }
            // no copy may still be in flight when the CTA retires: the pair's last MMAs have read every stage
            for (int i = max(0, total - L::kStages); i < total && ok; ++i)
                ok = mbar_poll(&H.done[i % L::kStages], (i / L::kStages) & 1u, status);
        } else {
            pdl_wait();
        }
    } else if (warp == kFgMmaWarp) {
        regs_down();
        pdl_wait();
        if (rank == 0) {
            const uint32_t id = idesc_f16(256, NW);
            const uint64_t desc0 = sdesc_sw128(smem_u32(ring));
            for (int it = 0, step = 0; it < total; ++it, step = step + 1 == steps ? 0 : step + 1) {
                const int st = it % L::kStages, b = it % L::kBufs;
                if (!mbar_poll2_lanes(&H.full[st], (it / L::kStages) & 1u, &H.tempty[b], ((it / L::kBufs) + 1u) & 1u, status)) break;
                tc_fence_after();
                const uint64_t ad = desc0 + (uint64_t) (st * (L::kStage >> 4)), bd = ad + (L::kA >> 4);
                const int n = groups_of(step);
                if (elect_lane()) {
#pragma unroll
                    for (int g = 0; g < L::kKS; ++g) {
                        if (g >= n) break;
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            tc_mma_f8_pair(tmem + (b * L::kKS + g) * NW, ad + g * (L::kGroup >> 4) + 2 * q, bd + g * (L::kGroup >> 4) + 2 * q, id, q);
                    }
                    tc_commit_pair(&H.done[st]);
                }
            }
        }
    } else if (warp > kFgMmaWarp) {
        regs_down();
    } else {
        // scale and add: thread = row of x, registers = its half of the weight rows
        regs_up();
        pdl_wait();
        const int half = warp >> 2, lg = warp & 3;
        const uint32_t tcol = tmem + ((uint32_t) (lg * 32) << 16) + (uint32_t) (half * L::kCols);
        const uint32_t tempty0 = mapa_u32(smem_u32(&H.tempty[0]), 0);
        int it = 0;
        bool ok = true;
        for (int t = pair; t < p.tiles && ok; t += pairs) {
            const int nt = t % p.ntiles;
            const int row = t / p.ntiles * 256 + (int) rank * 128 + lg * 32 + lane;
            const int col0 = nt * NW + half * L::kCols;
            const bool live = row < p.rows, wlive = col0 < p.n;
            const float* xs = p.xs + (live ? row : 0) * p.xsr;
            const float* ws = p.ws + (int64_t) (wlive ? col0 / 128 : 0) * p.groups;
            float acc[L::kCols];
#pragma unroll
            for (int j = 0; j < L::kCols; ++j) acc[j] = 0.f;
            // scales two steps ahead: a step is shorter than a load from L2
            struct Scales { float x[L::kKS], w[L::kKS]; };
            auto scales = [&](int step) {
                Scales v;
#pragma unroll
                for (int g = 0; g < L::kKS; ++g) {
                    const int kb = step * L::kKS + g;
                    const bool on = live && wlive && kb < p.groups;
                    v.x[g] = on ? __ldcg(xs + kb * p.xsg) : 0.f;
                    v.w[g] = on ? __ldg(ws + kb) : 0.f;
                }
                return v;
            };
            Scales s0 = scales(0), s1 = scales(1);
            for (int step = 0; step < steps; ++step, ++it) {
                const int b = it % L::kBufs, n = groups_of(step);
                float f[L::kKS];
#pragma unroll
                for (int g = 0; g < L::kKS; ++g) f[g] = s0.x[g] * s0.w[g];
                s0 = s1;
                s1 = scales(step + 2);
                ok = mbar_poll_lanes(&H.done[it % L::kStages], (it / L::kStages) & 1u, status);
                if (!ok) break;
                tc_fence_after();
                // the next 32 columns are on their way while these are scaled
                constexpr int NC = L::kCols / 32;
                uint32_t v[2][32];
                auto col_of = [&](int i) { return tcol + (uint32_t) ((b * L::kKS + i / NC) * NW + i % NC * 32); };
                tc_ld32_issue(col_of(0), v[0]);
#pragma unroll
                for (int i = 0; i < NC * L::kKS; ++i) {
                    const int c = i % NC;
                    if (i / NC >= n) break;
                    tc_ld_wait(v[i & 1]);
                    if (i + 1 < NC * n) {
                        tc_ld32_issue(col_of(i + 1), v[(i + 1) & 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * (uint32_t) b);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(__uint_as_float(v[i & 1][j]), f[i / NC], acc[c * 32 + j]);
                }
            }
            if (!ok) break;
            // Out through shared memory, 256 bytes of each row at a time, by TMA
            // stores that run on while the next tile is accumulated: written
            // straight from the registers (a row a lane) a tile took 8000 clocks,
            // by the warps from shared memory 5500.
            const int es = p.y_dtype == 2 ? 4 : 2;
            uint8_t* buf = stage_out + warp * L::kOut;
            const int wrow = t / p.ntiles * 256 + (int) rank * 128 + lg * 32;
            if (p.bias != nullptr) {
                // a column a lane, handed round
                float bv[L::kCols / 32];
#pragma unroll
                for (int c = 0; c < L::kCols / 32; ++c)
                    bv[c] = col0 + c * 32 + lane < p.n ? load_f32(p.bias, p.bias_dtype, col0 + c * 32 + lane) : 0.f;
#pragma unroll
                for (int j = 0; j < L::kCols; ++j) acc[j] += __shfl_sync(0xffffffffu, bv[j / 32], j % 32);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // 16-bit types: all kCols at once in pass 0; fp32: 64 in each pass
                const int cols = es == 4 ? 64 : L::kCols;
                if (h * cols >= L::kCols) break;
                if (lane == 0) bulk_wait_read();                                  // the buffer's last stores
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    uint4 w;
                    if (es == 4) {
                        if (h * 64 + c * 4 + 3 >= L::kCols) break;
                        w = make_uint4(__float_as_uint(acc[h * 64 + c * 4]), __float_as_uint(acc[h * 64 + c * 4 + 1]),
                                       __float_as_uint(acc[h * 64 + c * 4 + 2]), __float_as_uint(acc[h * 64 + c * 4 + 3]));
                    } else {
                        if (c * 8 + 7 >= L::kCols || h > 0) break;
                        uint32_t q[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float lo = acc[c * 8 + 2 * j], hi = acc[c * 8 + 2 * j + 1];
                            if (p.y_dtype == 0) {
                                const __half2 v = __floats2half2_rn(lo, hi);
                                q[j] = *reinterpret_cast<const uint32_t*>(&v);
                            } else {
                                const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
                                q[j] = *reinterpret_cast<const uint32_t*>(&v);
                            }
                        }
                        w = make_uint4(q[0], q[1], q[2], q[3]);
                    }
                    *reinterpret_cast<uint4*>(buf + fg_out(lane, c)) = w;
                }
                fence_proxy_async_smem();
                __syncwarp();
                const int c0 = col0 + h * cols, left = min(cols, p.n - c0);       // columns of this pass
                const int rows = min(32, p.rows - wrow);
                if (left <= 0 || rows <= 0) continue;
                if (p.yvec) {
                    const int wide = 128 / es;                                    // columns of a box
                    if (lane == 0) {
                        for (int c = 0; c < left; c += wide) tma_store_2d(&p.ymap, buf + c / wide * 4096, c0 + c, wrow);
                        bulk_commit();
                    }
                } else {
                    uint8_t* y = static_cast<uint8_t*>(p.y) + ((int64_t) wrow * p.ldy + c0) * es;
                    for (int r = 0; r < rows; ++r)
                        for (int j = lane; j < left; j += 32) {
                            if (es == 4) reinterpret_cast<uint32_t*>(y + (int64_t) r * p.ldy * 4)[j] = *reinterpret_cast<const uint32_t*>(buf + fg_out(r, j >> 2) + (j & 3) * 4);
                            else reinterpret_cast<uint16_t*>(y + (int64_t) r * p.ldy * 2)[j] = *reinterpret_cast<const uint16_t*>(buf + fg_out(r, j >> 3) + (j & 7) * 2);
                        }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) bulk_wait();                        // stores are complete when the CTA retires
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                    // the pair's memory and barriers stay until both are done
    if (warp == kFgMmaWarp) {
        tc_fence_after();
        tmem_free_pair(tmem, kFgTmemCols);
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

// y [rows][n] of pitch ldy elements; box 128 bytes x 32 rows, 128-byte swizzle.
int fp8_out_map(CUtensorMap* map, void* y, int64_t rows, int64_t n, int64_t ldy, int dtype) {
    auto encode = fp8_encoder();
    EXL3_REQUIRE(encode != nullptr, EXL3_ERR_CUDA, "exl3_fp8_linear: cuTensorMapEncodeTiled is not available");
    const int es = dtype == 2 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t) n, (cuuint64_t) rows};
    const cuuint64_t strides[1] = {(cuuint64_t) (ldy * es)};
    const cuuint32_t box[2] = {(cuuint32_t) (128 / es), 32u};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = encode(map, dtype == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              2, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    EXL3_REQUIRE(r == CUDA_SUCCESS, EXL3_ERR_CUDA, "exl3_fp8_linear: output tensor map failed (%d)", (int) r);
    return EXL3_OK;
}

namespace {

// CTAs that split k: the largest power of two (a portable cluster) that keeps
// the grid within what is resident at once and leaves every CTA two groups.
int fs_cluster(int64_t tiles, int groups, int resident) {
    int s = 1;
    while (s < kFsMaxCluster && tiles * s * 2 <= resident && groups >= s * 4) s *= 2;
    return s;
}

// Launches one of the kernels whose clusters split k: `nt` rows a tile, `stage`
// bytes a stage, `head` bytes beside the ring, `ctas` that share an SM.
int fs_launch(void (*kern)(FsParams), std::once_flag (&once)[64], FsParams& p, int nt, int stage, int head, int ctas, cudaStream_t stream) {
    const int64_t tiles = ((int64_t) p.n + 127) / 128, rtiles = ((int64_t) p.rows + nt - 1) / nt;
    p.cluster = fs_cluster(tiles * rtiles, p.groups, 148 * ctas);
    const int steps = (p.groups + p.cluster - 1) / p.cluster, budget = (ctas == 2 ? 112 : 200) * 1024;
    int stages = (budget - 1024 - head) / stage;
    if (stages > kFsMaxStages) stages = kFsMaxStages;
    const int least = (nt * 512 + stage - 1) / stage;      // the partial sums' room
    if (stages > steps) stages = steps < least ? least : steps;
    if (stages < 4) stages = 4;                            // not fewer than TMEM buffers
    p.stages = stages;
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    cudaError_t attr = cudaSuccess;
    std::call_once(once[dev & 63], [&] { attr = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024); });
    EXL3_CUDA(attr);
    EXL3_REQUIRE(tiles * p.cluster <= INT32_MAX && rtiles <= 65535, EXL3_ERR_UNSUPPORTED, "exl3_fp8_linear: matrix too large");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (tiles * p.cluster), (unsigned) rtiles);
    cfg.blockDim = dim3(kFsThreads);
    cfg.dynamicSmemBytes = (size_t) (1024 + head + stages * stage);
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
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
    return EXL3_OK;
}

template <int NT>
int fr_launch(FsParams& p, cudaStream_t stream) {
    static std::once_flag once[64];
    static_assert(kFrThreads == kFsThreads, "one launch shape");
    return fs_launch(fp8_rows_kernel<NT>, once, p, NT, FrLayout<NT>::kStage, (int) sizeof(FrHead<NT>), FrLayout<NT>::kCtas, stream);
}

template <int NW>
int fg_launch(FgParams& p, int sms, cudaStream_t stream) {
    using L = FgLayout<NW>;
    static std::once_flag once[64];
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    cudaError_t attr = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr = cudaFuncSetAttribute(fp8_gemm_kernel<NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    });
    EXL3_CUDA(attr);
    const int64_t ntiles = ((int64_t) p.n + NW - 1) / NW, tiles = ntiles * (((int64_t) p.rows + 255) / 256);
    EXL3_REQUIRE(tiles * p.groups <= INT32_MAX, EXL3_ERR_UNSUPPORTED, "exl3_fp8_linear: matrix too large");
    p.ntiles = (int) ntiles;
    p.tiles = (int) tiles;
    const int pairs = (int) (tiles < sms / 2 ? tiles : sms / 2);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (2 * pairs));
    cfg.blockDim = dim3(kFgThreads);
    cfg.dynamicSmemBytes = (size_t) L::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<NW>, p));
    return EXL3_OK;
}

// Rows up to which the weights are the M operand and k is split: below, the
// 256-row tiles of the pair kernel are too few to fill the GPU.
constexpr int kFsInlineRows = 8;     // x quantised inside the kernel (16 rows x 4096 x 4096: 11.6 us so, 9.6 by a launch before)
constexpr int kFsMaxRows = 128;

int64_t fp8_ldq(int64_t k) { return (k + 15) / 16 * 16; }

}  // namespace

int fp8_quantize_launch(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq,
                        float* scale, int64_t sr, int64_t sg, int block_rows, bool pow2, cudaStream_t s);
int fp8_moe_status(int clear, uint32_t* status, cudaStream_t s);

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
    EXL3_REQUIRE(aligned_to(x, dtype_bytes(x_dtype)) && aligned_to(y, dtype_bytes(y_dtype)) && aligned_to(x_scale, 4) &&
                     aligned_to(w_scale, 4) && aligned_to(bias, dtype_bytes(bias_dtype)),
                 EXL3_ERR_ARG, "exl3_fp8_linear: x, y, bias and the scales must be aligned to their elements");
    auto s = static_cast<cudaStream_t>(stream);
    const int groups = (int) ((k + 127) / 128);
    const int es = x_dtype == 2 ? 4 : x_dtype == 3 ? 1 : 2;
    int rc;
    FsParams p{};
    p.x = x; p.ldx = ldx; p.xs = x_scale; p.xsr = groups; p.xsg = 1; p.ws = w_scale; p.bias = bias; p.y = y; p.ldy = ldy;
    p.x_dtype = x_dtype; p.y_dtype = y_dtype; p.bias_dtype = bias_dtype; p.pow2 = pow2 != 0;
    p.rows = (int) rows; p.n = (int) n; p.k = (int) k; p.groups = groups;
    p.xvec = k % 16 == 0 && ldx * es % 16 == 0 && aligned16(x);
    if (rows <= kFsMaxRows && (rc = fp8_map(&p.wmap, w, n, k, ldw, 128, "exl3_fp8_linear")) != EXL3_OK) return rc;
    if (rows <= kFsInlineRows) {
        static std::once_flag once[64];
        return fs_launch(fp8_stream_kernel, once, p, FsLayout::NT, FsLayout::kStage, (int) sizeof(FsHead), 2, s);
    }

    // e4m3 rows that TMA can load: the caller's, or a copy / the quantised rows in the scratch
    const void* xq = x;
    int64_t ldq = ldx;
    const float* xs = x_scale;
    int64_t xsr = groups, xsg = 1;           // here one group's scales lie together: a warp's rows read them in one piece
    int early = 0;
    if (x_dtype != EXL3_DTYPE_E4M3 || !aligned16(x) || ldx % 16 != 0) {
        const int64_t need = exl3_fp8_linear_scratch_bytes(rows, k, n, x_dtype);
        EXL3_REQUIRE(scratch && aligned16(scratch) && scratch_bytes >= need, EXL3_ERR_ARG,
                     "exl3_fp8_linear: scratch must be 16-byte aligned and hold %lld bytes", (long long) need);
        ldq = fp8_ldq(k);
        xq = scratch;
        if (x_dtype == EXL3_DTYPE_E4M3) {
            EXL3_CUDA(cudaMemcpy2DAsync(scratch, (size_t) ldq, x, (size_t) ldx, (size_t) k, (size_t) rows, cudaMemcpyDeviceToDevice, s));
        } else {
            float* sc = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + align_up(rows * ldq, 256));
            if ((rc = fp8_quantize_launch(x, x_dtype, rows, k, ldx, scratch, ldq, sc, 1, rows, 1, pow2 != 0, s)) != EXL3_OK) return rc;
            xs = sc;
            xsr = 1;
            xsg = rows;
            early = 1;
        }
    }
    if (rows <= kFsMaxRows) {
        const int nt = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
        if ((rc = fp8_map(&p.xmap, xq, rows, k, ldq, nt, "exl3_fp8_linear")) != EXL3_OK) return rc;
        p.xs = xs; p.xsr = xsr; p.xsg = xsg;
        p.early = early;
        return nt == 16 ? fr_launch<16>(p, s) : nt == 32 ? fr_launch<32>(p, s) : nt == 64 ? fr_launch<64>(p, s) : fr_launch<128>(p, s);
    }
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    DeviceInfo di;
    if ((rc = device_info(dev, &di)) != EXL3_OK) return rc;
    // Weight rows of a tile: 256 unless tiles of 128 fill the pairs of SMs enough
    // better to pay for loading x twice as often.
    const int64_t pairs = di.sms / 2, mt = (rows + 255) / 256;
    const int64_t c256 = (mt * ((n + 255) / 256) + pairs - 1) / pairs * 20, c128 = (mt * ((n + 127) / 128) + pairs - 1) / pairs * 13;
    const int nw = c128 < c256 ? 128 : 256;
    FgParams g{};
    if ((rc = fp8_map(&g.xmap, xq, rows, k, ldq, 128, "exl3_fp8_linear")) != EXL3_OK) return rc;
    if ((rc = fp8_map(&g.wmap, w, n, k, ldw, nw / 2, "exl3_fp8_linear")) != EXL3_OK) return rc;
    g.xs = xs; g.xsr = xsr; g.xsg = xsg; g.ws = w_scale; g.bias = bias; g.y = y; g.ldy = ldy;
    g.y_dtype = y_dtype; g.bias_dtype = bias_dtype; g.early = early;
    const int ys = y_dtype == 2 ? 4 : 2;
    g.yvec = aligned16(y) && ldy * ys % 16 == 0;
    if (g.yvec && (rc = fp8_out_map(&g.ymap, y, rows, n, ldy, y_dtype)) != EXL3_OK) return rc;
    g.rows = (int) rows; g.n = (int) n; g.groups = groups;
    return nw == 128 ? fg_launch<128>(g, di.sms, s) : fg_launch<256>(g, di.sms, s);
}

extern "C" int64_t exl3_fp8_linear_scratch_bytes(int64_t rows, int64_t k, int64_t n, int x_dtype) {
    using namespace exl3;
    if (rows < 0 || k < 1 || n < 1 || x_dtype < 0 || x_dtype > 3) return -1;
    if (rows <= kFsInlineRows) return 0;
    return align_up(rows * fp8_ldq(k), 256) + (x_dtype == EXL3_DTYPE_E4M3 ? 0 : rows * ((k + 127) / 128) * 4);
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
    uint32_t moe = 0u;
    const int rc = fp8_moe_status(clear, &moe, s);
    *status |= moe;
    return rc;
}
