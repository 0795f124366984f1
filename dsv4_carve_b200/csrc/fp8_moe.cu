// fp8_moe.cu -- routed-expert MoE layer for a few tokens over e4m3 experts with
// one fp32 scale for each 128 x 128 block of a weight, in two kernels.
//   G = x . Wgate_e^T, U = x . Wup_e^T      (x quantised by row and 128 columns)
//   a = silu(min(G, L)) * clamp(U, -L, L)   (fp32; quantised the same way)
//   out[t] = sum over the valid slots of weight * (a . Wdown_e^T)   (fp32, one cast)
// Bound: the routed experts' weights, 3 * H * I bytes each, read once.  So both
// kernels do nothing but stream weight blocks: a 128 x 128 block is one TMA box
// and the M operand of four tcgen05.mma (K = 32 e4m3 each), the tokens of the
// expert are N, and each block's sums are read back from TMEM, scaled by the
// two scales and added to fp32 registers while the next block is multiplied.
//
// Work is cut evenly, not by experts: the layer's blocks in one fixed order
// (kernel 1: expert, 128 columns of I, block of H; kernel 2: 128 columns of H,
// expert, block of I) are split into as many equal ranges as there are CTAs, so
// every SM streams the same number of bytes.  A CTA's first and last output
// tile may be shared with its neighbours: each leaves its partial sums in the
// scratch and counts its blocks, and the one that completes the count adds the
// parts in CTA order, so results do not depend on timing.  No CTA ever waits for
// another one.  Kernel 2 starts while kernel 1 runs (programmatic launch): it
// builds the same route plan and fills its shared-memory ring with weights, then
// waits for kernel 1 to complete before it touches what kernel 1 wrote.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "fp8.cuh"
#include "host.hpp"

namespace exl3 {

int fp8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, const char* what);

constexpr int kFmMaxRows = 64;
constexpr int kFmMaxSlots = 256;             // m * topk
constexpr int kFmMaxTopk = 16;
constexpr int kFmMaxInter = 8192;
constexpr int kFmMaxHidden = 16384;
constexpr int kFmMaxCtas = 160;
constexpr int kFmThreads = 320;              // warps 0-3 epilogue, 4-7 x, 8 producer, 9 MMA
constexpr int kFmProducerWarp = 8;
constexpr int kFmMmaWarp = 9;
constexpr int kFmMaxStages = 8;
constexpr int kFmMaxBufs = 4;
// Control region (uint32 words): [2] status; counters of kernel 1's output
// tiles (expert group, 128 columns of I) and of kernel 2's (128 columns of H).
constexpr int kFmCntA = 16;
constexpr int kFmCntB = kFmCntA + kFmMaxSlots * (kFmMaxInter / 128);
constexpr int kFmCtrlWords = kFmCntB + kFmMaxHidden / 128;
static_assert(4 * kFmCtrlWords <= EXL3_FP8_MOE_CTRL_BYTES, "control region too small");

struct FmParams {
    CUtensorMap w13;             // [E * 2 I][H], box 128 x 128
    CUtensorMap w2;              // [E * H][I], box 128 x 128
    CUtensorMap amap;            // down input [slots][I], box 128 x NT
    const void* x;
    void* out;
    const float* w13s;           // [E][2 I / 128][H / 128]
    const float* w2s;            // [E][H / 128][I / 128]
    uint8_t* aq;                 // [slots][I] e4m3
    float* as;                   // [slots][I / 128]
    float* part;                 // partial sums of the CTAs' first and last tiles
    uint32_t* ctrl;
    RouteIn route;
    float limit;
    int x_dtype, out_dtype, pow2, xvec;
    int m, topk, E, H, I, stages;
};

// Pairs are the valid (token, slot)s ordered by (expert, slot); a group is up
// to NT pairs of one expert.
struct FmPlan {
    alignas(16) int id[kFmMaxSlots];
    short slot[kFmMaxSlots];          // pair -> slot
    short pexp[kFmMaxSlots];          // pair -> expert
    short gstart[kFmMaxSlots + 2];    // group -> first pair; [G] = pairs
    uint8_t first[kFmMaxSlots];       // pair begins a group
    int wsum[8];
    int G;
};

template <int NT, int PH>
struct FmLayout {
    static constexpr int kMats = PH == 0 ? 2 : 1;                    // gate and up, or down
    static constexpr int kW = kMats * (int) kFp8WTile;
    static constexpr int kStage = kW + NT * 128;
    static constexpr int kBufs = NT <= 16 ? 4 : PH == 0 ? 2 : NT <= 32 ? 4 : 2;
    static constexpr int kTmemCols = NT * kMats * kBufs;             // 64 .. 256
};

template <int NT>
struct FmHead {
    FmPlan plan;
    uint64_t full[kFmMaxStages];
    uint64_t empty[kFmMaxStages];
    uint64_t tfull[kFmMaxBufs];
    uint64_t tempty[kFmMaxBufs];
    alignas(16) float fac[kFmMaxStages][NT];
    float wsc[kFmMaxStages][2];
    uint32_t wmax[4][NT];
    uint32_t tmem;
    uint32_t last;
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Every thread of the CTA calls this; ends with a barrier.
__device__ void fm_plan(FmPlan& P, const FmParams& p, int nt, int tid) {
    const int n = p.m * p.topk;
    int id = INT32_MAX;
    if (tid < kFmMaxSlots) {
        if (tid < n) {
            const int e = route_local_id(p.route, tid, p.E);
            if (e >= 0) id = e;
        }
        P.id[tid] = id;
        P.first[tid] = 0;
    }
    const int pairs = __syncthreads_count(id != INT32_MAX);
    if (id != INT32_MAX) {
        int before = 0, rank = 0;
        for (int s = 0; s < n; s += 4) {
            const int4 o = *reinterpret_cast<const int4*>(&P.id[s]);
            const int v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const bool same = v[q] == id && s + q < tid;
                rank += same;
                before += same || v[q] < id;
            }
        }
        P.slot[before] = (short) tid;
        P.pexp[before] = (short) id;
        P.first[before] = rank % nt == 0;
    }
    __syncthreads();
    const bool f = tid < kFmMaxSlots && P.first[tid] != 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, f);
    if (tid < kFmMaxSlots && (tid & 31) == 0) P.wsum[tid >> 5] = __popc(mask);
    __syncthreads();
    if (tid < kFmMaxSlots) {
        int g = __popc(mask & ((1u << (tid & 31)) - 1u)), total = 0;
        for (int w = 0; w < 8; ++w) {
            g += w < (tid >> 5) ? P.wsum[w] : 0;
            total += P.wsum[w];
        }
        if (f) P.gstart[g] = (short) tid;
        if (tid == 0) { P.G = total; P.gstart[total] = (short) pairs; }
    }
    __syncthreads();
}

// Equal ranges: CTA c of C has blocks [start(c), start(c + 1)) of `total`.
__device__ __forceinline__ int fm_start(int c, int C, int total) { return (int) ((int64_t) c * total / C); }
__device__ __forceinline__ int fm_owner(int t, int C, int total) { return (int) (((int64_t) (t + 1) * C - 1) / total); }

// The block a CTA is at, and the step to the next one.
template <int PH>
struct FmAt {
    int tile, g, kb;          // PH 0: tile = group * NBI + column block; PH 1: tile = column block of H
    int G, NB, KB;            // groups, column blocks of I (PH 0), k blocks
    __device__ __forceinline__ FmAt(int t, int G_, int NB_, int KB_) : G(G_), NB(NB_), KB(KB_) {
        kb = t % KB;
        const int u = t / KB;
        if (PH == 0) { tile = u; g = u / NB; } else { g = u % G; tile = u / G; }
    }
    __device__ __forceinline__ void next() {
        if (++kb < KB) return;
        kb = 0;
        if (PH == 0) { ++tile; g = tile / NB; } else if (++g == G) { g = 0; ++tile; }
    }
};

template <int NT, int PH>
__global__ void __launch_bounds__(kFmThreads, 1) fp8_moe_kernel(const __grid_constant__ FmParams p) {
    using L = FmLayout<NT, PH>;
    constexpr int kMats = L::kMats;
    extern __shared__ uint8_t fm_raw[];
    uint8_t* ring = fm_raw + ((1024u - (smem_u32(fm_raw) & 1023u)) & 1023u);
    FmHead<NT>& S = *reinterpret_cast<FmHead<NT>*>(ring + p.stages * L::kStage);
    float* oacc = reinterpret_cast<float*>(ring + p.stages * L::kStage + sizeof(FmHead<NT>));    // PH 1: [m][128]
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const int C = (int) gridDim.x, cta = (int) blockIdx.x;
    const int NBI = p.I / 128, NBH = p.H / 128, KB = PH == 0 ? NBH : NBI;
    uint32_t* status = p.ctrl + 2;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&S.full[s], PH == 0 ? 1 + 4 : 1 + 1);
            mbar_init(&S.empty[s], 1 + 4);
        }
        for (int b = 0; b < L::kBufs; ++b) { mbar_init(&S.tfull[b], 1); mbar_init(&S.tempty[b], 4); }
        fence_barrier_init();
    }
    if (warp == kFmMmaWarp) tmem_alloc(&S.tmem, L::kTmemCols);
    if (PH == 0) {
        // Kernel 1 lets kernel 2 start only behind its own wait, so what came
        // before the layer (the routes among it) is complete for kernel 2 too.
        pdl_wait();
        pdl_launch_dependents();
    }
    tc_fence_before();
    fm_plan(S.plan, p, NT, tid);
    tc_fence_after();
    const FmPlan& P = S.plan;
    const uint32_t tmem = S.tmem;
    const int G = P.G;
    const int per_tile = PH == 0 ? KB : G * KB;                       // blocks of one output tile
    const int total = PH == 0 ? G * NBI * KB : NBH * per_tile;
    const int beg = fm_start(cta, C, total), end = fm_start(cta + 1, C, total), nsteps = end - beg;
    const int sm = p.stages;

    if (warp == kFmProducerWarp) {
        if (lane == 0 && nsteps > 0) {
            const CUtensorMap* wm = PH == 0 ? &p.w13 : &p.w2;
            auto weights = [&](const FmAt<PH>& a, int st) {
                const int e = P.pexp[P.gstart[a.g]];
                mbar_arrive_expect_tx(&S.full[st], (uint32_t) (PH == 0 ? L::kW : L::kStage));
                uint8_t* dst = ring + st * L::kStage;
                if (PH == 0) {
                    const int row = e * 2 * p.I + (a.tile % NBI) * 128;
                    tma_load_2d(dst, wm, a.kb * 128, row, &S.full[st]);
                    tma_load_2d(dst + kFp8WTile, wm, a.kb * 128, row + p.I, &S.full[st]);
                } else {
                    tma_load_2d(dst, wm, a.kb * 128, e * p.H + a.tile * 128, &S.full[st]);
                }
            };
            auto inputs = [&](const FmAt<PH>& a, int st) {
                tma_load_2d(ring + st * L::kStage + L::kW, &p.amap, a.kb * 128, P.gstart[a.g], &S.full[st]);
            };
            FmAt<PH> a(beg, G, NBI, KB);
            int issued = 0;
            if (PH == 1) {
                // the weights do not depend on kernel 1: a ring of them ahead of the wait
                FmAt<PH> a0 = a;
                for (; issued < min(sm, nsteps); ++issued) { weights(a, issued); a.next(); }
                pdl_wait();
                fence_proxy_async_global();
                for (int s = 0; s < issued; ++s) { inputs(a0, s); a0.next(); }
            }
            for (int s = issued; s < nsteps; ++s, a.next()) {
                const int st = s % sm;
                if (!mbar_wait(&S.empty[st], ((s / sm) + 1u) & 1u, status)) break;
                weights(a, st);
                if (PH == 1) inputs(a, st);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - sm); i < issued; ++i)
                if (!mbar_wait(&S.full[i % sm], (i / sm) & 1u, status)) break;
        } else if (PH == 1) {
            pdl_wait();
        }
    } else if (warp == kFmMmaWarp) {
        const uint64_t desc0 = sdesc_sw128(smem_u32(ring));
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        for (int s = 0; s < nsteps; ++s, a.next()) {
            const int st = s % sm, b = s % L::kBufs;
            const int n = P.gstart[a.g + 1] - P.gstart[a.g];
            const uint32_t id = __shfl_sync(0xffffffffu, idesc_f16(128, (n + 15) & ~15), 0);
            if (!mbar_wait_lanes(&S.full[st], (s / sm) & 1u, status)) break;
            if (!mbar_wait_lanes(&S.tempty[b], ((s / L::kBufs) + 1u) & 1u, status)) break;
            tc_fence_after();
            const uint64_t wd = desc0 + (uint64_t) (st * (L::kStage >> 4)), xd = wd + (L::kW >> 4);
            if (elect_lane()) {
#pragma unroll
                for (int mat = 0; mat < kMats; ++mat)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        tc_mma_f8(tmem + (b * kMats + mat) * NT, wd + mat * (kFp8WTile >> 4) + 2 * q, xd + 2 * q, id, q);
                tc_commit(&S.empty[st]);
                tc_commit(&S.tfull[b]);
            }
        }
    } else if (warp >= 4) {
        const int xw = warp - 4;
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        if (PH == 0) {
            // quantise the group's rows of x, one warp a row, 4 elements a lane
            if (cta == 0)
                for (int i = tid - 128; i < NBH; i += 128) p.ctrl[kFmCntB + i] = 0u;   // kernel 2's counters
            const int k4 = lane * 4;
            auto fetch = [&](const FmAt<PH>& at, int r) {
                const int tok = P.slot[P.gstart[at.g] + r] / p.topk;
                const int64_t i = (int64_t) tok * p.H + at.kb * 128 + k4;
                return p.xvec ? load_raw4(p.x, p.x_dtype, i) : load_raw4_tail(p.x, p.x_dtype, i, 4);
            };
            uint4 next = make_uint4(0u, 0u, 0u, 0u);
            if (nsteps > 0 && (xw & 3) < P.gstart[a.g + 1] - P.gstart[a.g]) next = fetch(a, xw & 3);
            for (int s = 0; s < nsteps; ++s) {
                const int st = s % sm, n = P.gstart[a.g + 1] - P.gstart[a.g];
                FmAt<PH> b = a;
                b.next();
                // rows go round the warps, so that few rows keep all of them busy
                const int r0 = (xw + s) & 3, r1 = (xw + s + 1) & 3;
                uint4 raw = next;
                if (s + 1 < nsteps && r1 < P.gstart[b.g + 1] - P.gstart[b.g]) next = fetch(b, r1);
                bool ok = true;
                if (r0 < n) {
                    for (int r = r0; r < n; r += 4) {
                        float v[4];
                        unpack4(raw, p.x_dtype, v);
                        if (r + 4 < n) raw = fetch(a, r + 4);
                        const float sx = fp8_scale(__reduce_max_sync(0xffffffffu, abs_bits4(v)), p.pow2);
                        const uint32_t q = fp8_quant4(v, sx, __frcp_rn(sx), p.pow2);
                        if (r == r0) ok = mbar_wait_lanes(&S.empty[st], ((s / sm) + 1u) & 1u, status);
                        if (!ok) break;
                        *reinterpret_cast<uint32_t*>(ring + st * L::kStage + L::kW + sw128_byte(r, k4)) = q;
                        if (lane == 0) S.fac[st][r] = sx;
                    }
                } else {
                    ok = mbar_wait_lanes(&S.empty[st], ((s / sm) + 1u) & 1u, status);
                }
                if (!ok) break;
                if (r0 == 0 && lane < 2) {
                    const int e = P.pexp[P.gstart[a.g]];
                    S.wsc[st][lane] = __ldg(p.w13s + ((int64_t) e * 2 * NBI + lane * NBI + a.tile % NBI) * NBH + a.kb);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.full[st]);
                a = b;
            }
        } else {
            // scales of the down input, the weight block and the route, one warp a block
            pdl_wait();
            for (int i = cta * 128 + tid - 128; i < G * NBI; i += C * 128) p.ctrl[kFmCntA + i] = 0u;   // kernel 1's
            for (int q = 0; q < xw && q < nsteps; ++q) a.next();
            for (int s = xw; s < nsteps; s += 4) {
                const int st = s % sm, p0 = P.gstart[a.g], n = P.gstart[a.g + 1] - p0, e = P.pexp[p0];
                const float ws = __ldg(p.w2s + ((int64_t) e * NBH + a.tile) * NBI + a.kb);
                float f[(NT + 31) / 32];
#pragma unroll
                for (int h = 0; h < (NT + 31) / 32; ++h) {
                    const int j = h * 32 + lane;
                    f[h] = j < n ? __ldcg(p.as + (int64_t) (p0 + j) * NBI + a.kb) * ws * route_weight(p.route, P.slot[p0 + j]) : 0.f;
                }
                if (!mbar_wait_lanes(&S.empty[st], ((s / sm) + 1u) & 1u, status)) break;
#pragma unroll
                for (int h = 0; h < (NT + 31) / 32; ++h)
                    if (h * 32 + lane < NT) S.fac[st][h * 32 + lane] = f[h];
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.full[st]);
                for (int q = 0; q < 4; ++q) a.next();
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        float acc[kMats][NT];
        auto clear = [&] {
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[mat][j] = 0.f;
        };
        // Counts this CTA's blocks of an output tile; true in the CTA that completes it.
        auto completes = [&](int counter, int blocks) {
            epi_sync();
            if (tid == 0) S.last = atom_add_acq_rel_gpu(&p.ctrl[counter], (uint32_t) blocks) + blocks == (uint32_t) per_tile;
            epi_sync();
            return S.last != 0u;
        };
        // a tile's part: slot 1 where the tile began before this CTA's range did not
        const int rows_pt = PH == 0 ? kMats * NT : p.m;               // rows of 128 in a part
        auto part_of = [&](int c, int first) { return p.part + ((int64_t) c * 2 + (fm_start(c, C, total) >= first ? 0 : 1)) * rows_pt * 128; };
        if (PH == 1) {
            pdl_wait();
            if (total == 0)
                for (int64_t i = (int64_t) cta * 128 + tid; i < (int64_t) p.m * p.H; i += (int64_t) C * 128)
                    store_out(p.out, p.out_dtype, i, 0.f);
            for (int t = 0; t < p.m; ++t) oacc[t * 128 + tid] = 0.f;
        }
        clear();
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        int seg = 0;                                                  // blocks of the current tile so far
        for (int s = 0; s < nsteps; ++s) {
            const int st = s % sm, b = s % L::kBufs;
            const int p0 = P.gstart[a.g], n = P.gstart[a.g + 1] - p0;
            if (!mbar_wait_lanes(&S.tfull[b], (s / L::kBufs) & 1u, status)) break;
            tc_fence_after();
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
                const float ws = PH == 0 ? S.wsc[st][mat] : 1.f;
#pragma unroll
                for (int c = 0; c < NT / 16; ++c) {
                    if (c * 16 >= n) break;
                    float v[16];
                    tc_ld16(tmem + ((uint32_t) (warp * 32) << 16) + (uint32_t) ((b * kMats + mat) * NT + c * 16), v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float f = PH == 0 ? S.fac[st][c * 16 + j] * ws : S.fac[st][c * 16 + j];
                        acc[mat][c * 16 + j] = fmaf(v[j], f, acc[mat][c * 16 + j]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&S.tempty[b]);
                mbar_arrive(&S.empty[st]);
            }
            ++seg;
            const bool tile_end = (PH == 0 ? a.kb + 1 == KB : (a.kb + 1 == KB && a.g + 1 == G)) || s + 1 == nsteps;
            if (PH == 1 && (a.kb + 1 == KB || s + 1 == nsteps)) {
                // the group's columns go to their tokens
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    if (j < n) oacc[(P.slot[p0 + j] / p.topk) * 128 + tid] += acc[0][j];
                clear();
            }
            if (tile_end) {
                const int first = a.tile * per_tile;                  // the tile's first block
                bool whole = seg == per_tile, finish = whole;
                if (!whole) {
                    float* dst = part_of(cta, first);
                    if (PH == 0) {
#pragma unroll
                        for (int mat = 0; mat < kMats; ++mat)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
                                if (j < n) dst[(mat * NT + j) * 128 + tid] = acc[mat][j];
                    } else {
                        for (int t = 0; t < p.m; ++t) dst[t * 128 + tid] = oacc[t * 128 + tid];
                    }
                    finish = completes((PH == 0 ? kFmCntA : kFmCntB) + a.tile, seg);
                    if (finish) {
                        const int c0 = fm_owner(first, C, total), c1 = fm_owner(first + per_tile - 1, C, total);
                        if (PH == 0) clear();
                        else for (int t = 0; t < p.m; ++t) oacc[t * 128 + tid] = 0.f;
                        for (int c = c0; c <= c1; ++c) {
                            if (fm_start(c, C, total) == fm_start(c + 1, C, total)) continue;
                            const float* src = part_of(c, first);
                            if (PH == 0) {
#pragma unroll
                                for (int mat = 0; mat < kMats; ++mat)
#pragma unroll
                                    for (int j = 0; j < NT; ++j)
                                        if (j < n) acc[mat][j] += __ldcg(src + (mat * NT + j) * 128 + tid);
                            } else {
                                for (int t = 0; t < p.m; ++t) oacc[t * 128 + tid] += __ldcg(src + t * 128 + tid);
                            }
                        }
                    }
                }
                if (finish && PH == 0) {
                    // SwiGLU, then one scale for each token's 128 columns; NaN passes through
                    const int ib = a.tile % NBI;
                    const float lim = p.limit;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if (j >= n) break;
                        float g = acc[0][j], u = acc[kMats - 1][j];
                        g = g > lim ? lim : g;
                        u = u > lim ? lim : u < -lim ? -lim : u;
                        acc[0][j] = g / (1.f + expf(-g)) * u;
                        const uint32_t mx = __reduce_max_sync(0xffffffffu, abs_bits(acc[0][j]));
                        if (lane == 0) S.wmax[warp][j] = mx;
                    }
                    epi_sync();
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if (j >= n) break;
                        const uint32_t mx = max(max(S.wmax[0][j], S.wmax[1][j]), max(S.wmax[2][j], S.wmax[3][j]));
                        const float sa = fp8_scale(mx, p.pow2);
                        p.aq[(int64_t) (p0 + j) * p.I + ib * 128 + tid] =
                            (uint8_t) e4m3x2(fp8_quotient(acc[0][j], sa, __frcp_rn(sa), p.pow2), 0.f);
                        if (tid == 0) p.as[(int64_t) (p0 + j) * NBI + ib] = sa;
                    }
                    epi_sync();                                       // wmax is free for the next tile
                }
                if (finish && PH == 1)
                    for (int t = 0; t < p.m; ++t)
                        store_out(p.out, p.out_dtype, (int64_t) t * p.H + a.tile * 128 + tid, oacc[t * 128 + tid]);
                if (PH == 0) clear();
                else for (int t = 0; t < p.m; ++t) oacc[t * 128 + tid] = 0.f;
                seg = 0;
            }
            a.next();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kFmMmaWarp) {
        tc_fence_after();
        tmem_free(tmem, L::kTmemCols);
    }
}

// ------------------------------------------------------------------ host side
namespace {

struct FmGeom {
    int nt;
    int64_t off_aq, off_as, off_part, bytes;
};

FmGeom fm_geom(int64_t m, int64_t topk, int64_t H, int64_t I) {
    FmGeom g{};
    (void) H;
    g.nt = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    const int64_t slots = m * topk;
    g.off_aq = EXL3_FP8_MOE_CTRL_BYTES;
    g.off_as = g.off_aq + align_up(slots * I, 256);
    g.off_part = g.off_as + align_up(slots * (I / 128) * 4, 256);
    const int64_t part_rows = 2 * g.nt > m ? 2 * g.nt : m;
    g.bytes = g.off_part + (int64_t) kFmMaxCtas * 2 * part_rows * 128 * 4;
    return g;
}

template <int NT, int PH>
int fm_launch(FmParams p, int sms, cudaStream_t stream) {
    using L = FmLayout<NT, PH>;
    // Up to 32 rows the two kernels share an SM while kernel 2 waits (shared
    // memory 120 + 104 KB); above that their registers leave room for one.
    constexpr int kBudget = (NT > 32 ? 200 : PH == 0 ? 120 : 104) * 1024;
    const int extra = 1024 + (int) sizeof(FmHead<NT>) + (PH == 1 ? p.m * 512 : 0);
    int stages = (kBudget - extra) / L::kStage;
    if (stages > kFmMaxStages) stages = kFmMaxStages;
    p.stages = stages;
    const int smem = extra + stages * L::kStage;
    static std::once_flag once[64];
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    cudaError_t attr = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr = cudaFuncSetAttribute(fp8_moe_kernel<NT, PH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget);
    });
    EXL3_CUDA(attr);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (sms < kFmMaxCtas ? sms : kFmMaxCtas));
    cfg.blockDim = dim3(kFmThreads);
    cfg.dynamicSmemBytes = (size_t) smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, fp8_moe_kernel<NT, PH>, p));
    return EXL3_OK;
}

template <int NT>
int fm_run(const FmParams& p, int sms, cudaStream_t s) {
    const int rc = fm_launch<NT, 0>(p, sms, s);
    return rc != EXL3_OK ? rc : fm_launch<NT, 1>(p, sms, s);
}

}  // namespace
}  // namespace exl3

extern "C" int64_t exl3_fp8_moe_max_rows(void) { return exl3::kFmMaxRows; }

extern "C" int64_t exl3_fp8_moe_scratch_bytes(int64_t m, int64_t topk, int64_t hidden, int64_t inter) {
    using namespace exl3;
    if (m < 1 || m > kFmMaxRows || topk < 1 || topk > kFmMaxTopk || m * topk > kFmMaxSlots || hidden < 128 || hidden % 128 ||
        hidden > kFmMaxHidden || inter < 128 || inter % 128 || inter > kFmMaxInter)
        return -1;
    return fm_geom(m, topk, hidden, inter).bytes;
}

extern "C" int exl3_fp8_moe_decode(const void* x, int x_dtype, void* out, int out_dtype, int64_t m, int64_t hidden,
                                   int64_t inter, const void* gate_up, const float* gate_up_scale, const void* down,
                                   const float* down_scale, int64_t n_experts, const exl3_moe_route* route, int64_t topk,
                                   float swiglu_limit, int pow2, void* scratch, int64_t scratch_bytes, void* stream) {
    using namespace exl3;
    EXL3_REQUIRE(x && out && gate_up && gate_up_scale && down && down_scale && route && route->ids && route->weights && scratch,
                 EXL3_ERR_ARG, "exl3_fp8_moe_decode: null pointer");
    EXL3_REQUIRE(m >= 1 && m <= kFmMaxRows, EXL3_ERR_ARG, "exl3_fp8_moe_decode: row count must be 1..%d", kFmMaxRows);
    EXL3_REQUIRE(topk >= 1 && topk <= kFmMaxTopk && m * topk <= kFmMaxSlots, EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: topk must be 1..16 and rows * topk at most %d", kFmMaxSlots);
    EXL3_REQUIRE(hidden >= 128 && hidden % 128 == 0 && hidden <= kFmMaxHidden, EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: hidden must be a multiple of 128 up to %d", kFmMaxHidden);
    EXL3_REQUIRE(inter >= 128 && inter % 128 == 0 && inter <= kFmMaxInter, EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: intermediate must be a multiple of 128 up to %d", kFmMaxInter);
    EXL3_REQUIRE(n_experts >= 1 && n_experts <= 32767 && n_experts * 2 * inter <= INT32_MAX && n_experts * hidden <= INT32_MAX,
                 EXL3_ERR_ARG, "exl3_fp8_moe_decode: expert count out of range");
    EXL3_REQUIRE(x_dtype >= 0 && x_dtype <= 2 && out_dtype >= 0 && out_dtype <= 2 && route->weights_dtype >= 0 &&
                     route->weights_dtype <= 2 && (route->ids_dtype == 0 || route->ids_dtype == 1),
                 EXL3_ERR_ARG, "exl3_fp8_moe_decode: dtypes must be fp16, bf16 or fp32, ids int32 or int64");
    EXL3_REQUIRE(route->expert_map == nullptr || route->n_global >= 1, EXL3_ERR_ARG, "exl3_fp8_moe_decode: empty expert map");
    EXL3_REQUIRE(swiglu_limit > 0.f, EXL3_ERR_ARG, "exl3_fp8_moe_decode: the SwiGLU limit must be positive");
    EXL3_REQUIRE(aligned16(gate_up) && aligned16(down) && aligned16(scratch), EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: weights and scratch must be 16-byte aligned");
    const FmGeom g = fm_geom(m, topk, hidden, inter);
    EXL3_REQUIRE(scratch_bytes >= g.bytes, EXL3_ERR_ARG, "exl3_fp8_moe_decode: scratch too small (%lld < %lld bytes)",
                 (long long) scratch_bytes, (long long) g.bytes);
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    DeviceInfo di;
    int rc = device_info(dev, &di);
    if (rc != EXL3_OK) return rc;
    uint8_t* sb = static_cast<uint8_t*>(scratch);
    FmParams p{};
    if ((rc = fp8_map(&p.w13, gate_up, n_experts * 2 * inter, hidden, hidden, 128, "exl3_fp8_moe_decode")) != EXL3_OK) return rc;
    if ((rc = fp8_map(&p.w2, down, n_experts * hidden, inter, inter, 128, "exl3_fp8_moe_decode")) != EXL3_OK) return rc;
    if ((rc = fp8_map(&p.amap, sb + g.off_aq, m * topk, inter, inter, g.nt, "exl3_fp8_moe_decode")) != EXL3_OK) return rc;
    p.x = x; p.out = out; p.w13s = gate_up_scale; p.w2s = down_scale;
    p.aq = sb + g.off_aq;
    p.as = reinterpret_cast<float*>(sb + g.off_as);
    p.part = reinterpret_cast<float*>(sb + g.off_part);
    p.ctrl = reinterpret_cast<uint32_t*>(sb);
    p.route = RouteIn{route->ids, route->weights, route->expert_map, route->n_global, route->ids_dtype, route->weights_dtype};
    p.limit = swiglu_limit;
    p.x_dtype = x_dtype; p.out_dtype = out_dtype; p.pow2 = pow2 != 0;
    p.xvec = reinterpret_cast<uintptr_t>(x) % (x_dtype == 2 ? 16 : 8) == 0;
    p.m = (int) m; p.topk = (int) topk; p.E = (int) n_experts; p.H = (int) hidden; p.I = (int) inter;
    auto s = static_cast<cudaStream_t>(stream);
    if (g.nt == 16) return fm_run<16>(p, di.sms, s);
    if (g.nt == 32) return fm_run<32>(p, di.sms, s);
    return fm_run<64>(p, di.sms, s);
}
