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
int fp8_quantize_launch(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq,
                        float* scale, int64_t sr, int64_t sg, int block_rows, bool pow2, cudaStream_t s);

constexpr int kFmMaxRows = 64;
constexpr int kFmMaxSlots = 256;             // m * topk
constexpr int kFmMaxTopk = 16;
constexpr int kFmMaxInter = 8192;
constexpr int kFmMaxHidden = 16384;
constexpr int kFmMaxCtas = 160;
// Warps 0-3 epilogue, 4 producer, 5 MMA, 6-7 x.  Two warps on each of an SM's
// four register files: CTAs of both kernels fit side by side (kernel 2 waits
// there, its ring filled), which three would not.
constexpr int kFmThreads = 256;
constexpr int kFmProducerWarp = 4;
constexpr int kFmMmaWarp = 5;
constexpr int kFmXWarp = 6;
constexpr int kFmXWarps = 2;
// Rows up to which kernel 1 quantises the rows of x that it multiplies itself;
// above, a launch of the quantiser does it once for all CTAs.
constexpr int kFmInlineRows = 16;
constexpr int kFmMaxSlotsW = 12;             // weight blocks in the ring
constexpr int kFmMaxBufs = 4;                // steps whose sums and inputs are held
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
    CUtensorMap xmap;            // more than kFmInlineRows rows: x in e4m3 [m][H], box 128 x NT
    const void* x;
    void* out;
    const float* w13s;           // [E][2 I / 128][H / 128]
    const float* w2s;            // [E][H / 128][I / 128]
    const float* xs;             // its scales [H / 128][m]
    uint8_t* aq;                 // [slots][I] e4m3
    float* as;                   // [slots][I / 128]
    float* part;                 // partial sums of the CTAs' first and last tiles
    uint32_t* ctrl;
    RouteIn route;
    float limit;
    int x_dtype, out_dtype, pow2, xvec;
    int m, topk, E, H, I, slots;
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

// Shared memory of a CTA: a ring of weight blocks (16 KB each, so that few bytes
// wait while many are in flight; with the NT input rows of the block where TMA
// brings them), kernel 1's own quantised rows of x of kBufs steps, the head,
// kernel 2's output rows.  A step is one block of k: kernel 1 multiplies the gate
// and the up block, each into TMEM columns of its own, kernel 2 the down block.
// D's columns are the group's pairs, or all tokens where kernel 1's x comes
// quantised (NT > 16): columns of other tokens are never used.
template <int NT, int PH>
struct FmLayout {
    static constexpr bool kInline = PH == 0 && NT <= kFmInlineRows;
    static constexpr int kMats = PH == 0 ? 2 : 1;
    static constexpr int kBufs = NT <= 16 ? 4 : PH == 0 ? 2 : NT <= 32 ? 4 : 2;
    static constexpr int kTmemCols = NT * kMats * kBufs;             // 64 .. 256
    static constexpr int kX = NT * 128;
    static constexpr int kSlot = (int) kFp8WTile + (kInline ? 0 : kX);
    static constexpr int kXRing = kInline ? kBufs * kX : 0;
};

template <int NT>
struct FmHead {
    FmPlan plan;
    uint64_t wfull[kFmMaxSlotsW];        // a weight block has arrived
    uint64_t wdone[kFmMaxSlotsW];        // it has been multiplied
    uint64_t xfull[kFmMaxBufs];          // a step's input rows (kernel 1) and factors are there
    uint64_t tfull[kFmMaxBufs];          // a step's sums are in TMEM; its input rows have been read
    uint64_t tempty[kFmMaxBufs];         // they have been read
    // Factors of a step's columns.  Twice kBufs deep: x's warps write step s once
    // step s - kBufs is in TMEM, i.e. the epilogue is done with s - 2 kBufs.
    alignas(16) float fac[2 * kFmMaxBufs][NT];
    float wsc[2 * kFmMaxBufs][2];
    alignas(16) uint32_t wmax[4][NT];
    short tokpair[NT];                   // a token's first pair in the group
    uint32_t tmem;
    uint32_t last;
};

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Every thread of the CTA calls this; ends with a barrier.
__device__ void fm_plan(FmPlan& P, const FmParams& p, int nt, int tid) {
    const int n = p.m * p.topk;
    static_assert(kFmThreads == kFmMaxSlots, "every slot has its own thread");
    int id = INT32_MAX;
    if (tid < n) {
        const int e = route_local_id(p.route, tid, p.E);
        if (e >= 0) id = e;
    }
    P.id[tid] = id;
    P.first[tid] = 0;
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
    const bool f = P.first[tid] != 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, f);
    if ((tid & 31) == 0) P.wsum[tid >> 5] = __popc(mask);
    __syncthreads();
    {
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

// Equal ranges: CTA c of C has steps [start(c), start(c + 1)) of `total`, at most
// 256 groups x 64 x 128 blocks, so the products stay below 2^32.
static_assert((int64_t) kFmMaxSlots * (kFmMaxInter / 128) * (kFmMaxHidden / 128) * kFmMaxCtas < (int64_t) 1 << 32, "");
__device__ __forceinline__ int fm_start(int c, int C, int total) { return (int) ((uint32_t) c * (uint32_t) total / (uint32_t) C); }
__device__ __forceinline__ int fm_owner(int t, int C, int total) { return (int) (((uint32_t) (t + 1) * (uint32_t) C - 1u) / (uint32_t) total); }

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
    constexpr int kMats = L::kMats, kBufs = L::kBufs, kFacs = 2 * L::kBufs;
    constexpr bool kInline = L::kInline, kTokens = PH == 0 && !kInline;   // kTokens: D's columns are all tokens
    constexpr int kCh = NT < 32 ? 4 : 8;                              // columns handled together at a tile's end
    extern __shared__ uint8_t fm_raw[];
    uint8_t* ring = fm_raw + ((1024u - (smem_u32(fm_raw) & 1023u)) & 1023u);
    uint8_t* xring = ring + p.slots * L::kSlot;
    FmHead<NT>& S = *reinterpret_cast<FmHead<NT>*>(xring + L::kXRing);
    float* oacc = reinterpret_cast<float*>(xring + L::kXRing + sizeof(FmHead<NT>));    // PH 1: [m][128]
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const int C = (int) gridDim.x, cta = (int) blockIdx.x;
    const int NBI = p.I / 128, NBH = p.H / 128, KB = PH == 0 ? NBH : NBI;
    const int W = p.slots;
    uint32_t* status = p.ctrl + 2;

    if (tid == 0) {
        tmap_prefetch(PH == 0 ? &p.w13 : &p.w2);
        for (int s = 0; s < W; ++s) { mbar_init(&S.wfull[s], 1); mbar_init(&S.wdone[s], 1); }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&S.xfull[b], kInline ? kFmXWarps : 1);
            mbar_init(&S.tfull[b], 1);
            mbar_init(&S.tempty[b], 4);
        }
        fence_barrier_init();
    }
    if (warp == kFmMmaWarp) tmem_alloc(&S.tmem, L::kTmemCols);
    if (PH == 0) {
        // Kernel 2 may start once what came before the layer (the routes among
        // it) is complete: behind this kernel's own wait, or at once where the
        // quantiser, an ordinary launch, ran in between.  Then only x is waited
        // for, by those who read it.
        if (kInline) pdl_wait();
        pdl_launch_dependents();
    }
    tc_fence_before();
    fm_plan(S.plan, p, NT, tid);
    tc_fence_after();
    const FmPlan& P = S.plan;
    const uint32_t tmem = __shfl_sync(0xffffffffu, S.tmem, 0);
    const int G = P.G;
    const int per_tile = PH == 0 ? KB : G * KB;                       // steps of one output tile
    const int total = PH == 0 ? G * NBI * KB : NBH * per_tile;
    const int beg = fm_start(cta, C, total), end = fm_start(cta + 1, C, total), nsteps = end - beg;

    if (warp == kFmProducerWarp) {
        if (lane == 0 && nsteps > 0) {
            const int nblk = nsteps * kMats;
            auto weights = [&](const FmAt<PH>& a, int mat, int slot) {
                const int e = P.pexp[P.gstart[a.g]];
                mbar_arrive_expect_tx(&S.wfull[slot], (uint32_t) L::kSlot);
                const int row = PH == 0 ? e * 2 * p.I + mat * p.I + (a.tile % NBI) * 128 : e * p.H + a.tile * 128;
                tma_load_2d(ring + slot * L::kSlot, PH == 0 ? &p.w13 : &p.w2, a.kb * 128, row, &S.wfull[slot]);
            };
            auto inputs = [&](const FmAt<PH>& a, int slot) {
                if (PH == 0) tma_load_2d(ring + slot * L::kSlot + kFp8WTile, &p.xmap, a.kb * 128, 0, &S.wfull[slot]);
                else tma_load_2d(ring + slot * L::kSlot + kFp8WTile, &p.amap, a.kb * 128, P.gstart[a.g], &S.wfull[slot]);
            };
            FmAt<PH> a(beg, G, NBI, KB);
            auto mat_of = [](int t) { return PH == 0 ? t & 1 : 0; };
            auto next = [&](FmAt<PH>& at, int t) { if (PH == 1 || (t & 1)) at.next(); };
            int t = 0;
            if (!kInline) {
                // a ring of weights ahead of the wait: no kernel that may still run writes them
                FmAt<PH> a0 = a;
                for (; t < min(W, nblk); ++t) { weights(a, mat_of(t), t); next(a, t); }
                pdl_wait();
                fence_proxy_async_global();
                for (int i = 0; i < t; ++i) { inputs(a0, i); next(a0, i); }
            }
            int issued = t;
            for (; t < nblk; ++t) {
                const int slot = t % W;
                if (t >= W && !mbar_wait(&S.wdone[slot], ((t / W) + 1u) & 1u, status)) break;
                weights(a, mat_of(t), slot);
                if (!kInline) inputs(a, slot);
                next(a, t);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - W); i < issued; ++i)
                if (!mbar_wait(&S.wfull[i % W], (i / W) & 1u, status)) break;
        } else if (!kInline) {
            pdl_wait();
        }
    } else if (warp == kFmMmaWarp) {
        const uint64_t wdesc0 = sdesc_sw128(smem_u32(ring)), xdesc0 = sdesc_sw128(smem_u32(xring));
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        int slot = 0;
        uint32_t wpar = 0;
        bool ok = true;
        for (int s = 0; s < nsteps && ok; ++s, a.next()) {
            const int b = s % kBufs;
            const int n = kTokens ? p.m : P.gstart[a.g + 1] - P.gstart[a.g];
            const uint32_t id = __shfl_sync(0xffffffffu, idesc_f16(128, (n + 15) & ~15), 0);
            ok = mbar_poll2_lanes(&S.xfull[b], (s / kBufs) & 1u, &S.tempty[b], ((s / kBufs) + 1u) & 1u, status);
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
                ok = ok && mbar_poll_lanes(&S.wfull[slot], wpar, status);
                if (!ok) break;
                tc_fence_after();
                const uint64_t wd = wdesc0 + (uint64_t) (slot * (L::kSlot >> 4));
                const uint64_t xd = kInline ? xdesc0 + (uint64_t) (b * (L::kX >> 4)) : wd + (kFp8WTile >> 4);
                if (elect_lane()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) tc_mma_f8(tmem + (b * kMats + mat) * NT, wd + 2 * q, xd + 2 * q, id, q);
                    tc_commit(&S.wdone[slot]);
                    if (mat + 1 == kMats) tc_commit(&S.tfull[b]);
                }
                if (++slot == W) { slot = 0; wpar ^= 1u; }
            }
        }
    } else if (warp >= kFmXWarp) {
        const int xw = warp - kFmXWarp, xt = tid - kFmXWarp * 32;
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        if (PH == 0 && cta == 0)
            for (int i = xt; i < NBH; i += 32 * kFmXWarps) p.ctrl[kFmCntB + i] = 0u;   // kernel 2's counters
        if (kInline) {
            // Quantise the group's rows of x, four a warp; which four goes round
            // with the steps, so that few rows keep both warps busy.
            XRows next[2];                                    // the next rows of this warp, fetched ahead
            FmAt<PH> f = a;
            int fs = 0, fq = xw;
            auto fetch = [&](XRows& to) {
                while (fs < nsteps && fq * 4 >= P.gstart[f.g + 1] - P.gstart[f.g]) {
                    ++fs;
                    f.next();
                    fq = (xw + fs) % kFmXWarps;
                }
                if (fs >= nsteps) return;
                const int p0 = P.gstart[f.g] + fq * 4, cnt = min(4, P.gstart[f.g + 1] - p0), lr = XRows::row(cnt, lane);
                const int tok = P.slot[p0 + min(lr, cnt - 1)] / p.topk;
                to.load(cnt, p.x, p.x_dtype, (int64_t) tok * p.H + f.kb * 128 + XRows::col(cnt, lane), lr < cnt ? 16 : 0, p.xvec);
                fq += kFmXWarps;
            };
            fetch(next[0]);
            fetch(next[1]);
            for (int s = 0; s < nsteps; ++s, a.next()) {
                const int b = s % kBufs, n = P.gstart[a.g + 1] - P.gstart[a.g], q0 = (xw + s) % kFmXWarps;
                uint8_t* tile = xring + b * L::kX;
                float* fac = S.fac[s % kFacs];
                float ws = 0.f;
                if (q0 == 0 && lane < 2)
                    ws = __ldg(p.w13s + ((int64_t) P.pexp[P.gstart[a.g]] * 2 * NBI + lane * NBI + a.tile % NBI) * NBH + a.kb);
                bool free = false;
                for (int q = q0; q * 4 < n; q += kFmXWarps) {
                    const XRows cur = next[0];
                    next[0] = next[1];
                    fetch(next[1]);
                    const int cnt = min(4, n - q * 4), lr = XRows::row(cnt, lane);
                    float sx;
                    const uint4 v = cur.quantize(cnt, p.x_dtype, p.pow2, sx);
                    if (!free && !(free = mbar_wait_lanes(&S.tfull[b], ((s / kBufs) + 1u) & 1u, status))) break;
                    if (lr < cnt) XRows::store(cnt, tile, q * 4 + lr, lane, v);
                    if (lr < cnt && (cnt == 1 ? lane == 0 : (lane & 7) == 0)) fac[q * 4 + lr] = sx;
                }
                if (!free && !mbar_wait_lanes(&S.tfull[b], ((s / kBufs) + 1u) & 1u, status)) break;
                if (q0 == 0 && lane < 2) S.wsc[s % kFacs][lane] = ws;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.xfull[b]);
            }
        } else {
            // The factors of a step's columns, one warp a step: x's scales and the two
            // blocks' (kernel 1), or the down input's, the block's and the route's.
            pdl_wait();
            if (PH == 1) {
                for (int i = cta * 32 * kFmXWarps + xt; i < G * NBI; i += C * 32 * kFmXWarps) p.ctrl[kFmCntA + i] = 0u;   // kernel 1's
            }
            for (int q = 0; q < xw && q < nsteps; ++q) a.next();
            for (int s = xw; s < nsteps; s += kFmXWarps) {
                const int b = s % kBufs, p0 = P.gstart[a.g], n = PH == 0 ? p.m : P.gstart[a.g + 1] - p0, e = P.pexp[p0];
                float ws = 0.f;
                if (PH == 1) ws = __ldg(p.w2s + ((int64_t) e * NBH + a.tile) * NBI + a.kb);
                else if (lane < 2) ws = __ldg(p.w13s + ((int64_t) e * 2 * NBI + lane * NBI + a.tile % NBI) * NBH + a.kb);
                float f[(NT + 31) / 32];
#pragma unroll
                for (int h = 0; h < (NT + 31) / 32; ++h) {
                    const int j = h * 32 + lane;
                    f[h] = 0.f;
                    if (j < n) f[h] = PH == 0 ? __ldcg(p.xs + (int64_t) a.kb * p.m + j)
                                              : __ldcg(p.as + (int64_t) (p0 + j) * NBI + a.kb) * ws * route_weight(p.route, P.slot[p0 + j]);
                }
                if (!mbar_wait_lanes(&S.tfull[b], ((s / kBufs) + 1u) & 1u, status)) break;
#pragma unroll
                for (int h = 0; h < (NT + 31) / 32; ++h)
                    if (h * 32 + lane < NT) S.fac[s % kFacs][h * 32 + lane] = f[h];
                if (PH == 0 && lane < 2) S.wsc[s % kFacs][lane] = ws;
                __syncwarp();
                if (lane == 0) mbar_arrive(&S.xfull[b]);
                for (int q = 0; q < kFmXWarps; ++q) a.next();
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
        // Counts this CTA's steps of an output tile; true in the CTA that completes it.
        auto completes = [&](int counter, int steps) {
            epi_sync();
            if (tid == 0) S.last = atom_add_acq_rel_gpu(&p.ctrl[counter], (uint32_t) steps) + steps == (uint32_t) per_tile;
            epi_sync();
            return S.last != 0u;
        };
        // a tile's part: slot 1 where the CTA's range began before the tile did
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
        int seg = 0;                                                  // steps of the current tile so far
        for (int s = 0; s < nsteps; ++s) {
            const int b = s % kBufs;
            const int p0 = P.gstart[a.g], pairs = P.gstart[a.g + 1] - p0, n = kTokens ? p.m : pairs;   // n: D's columns
            if (!mbar_wait_lanes(&S.tfull[b], (s / kBufs) & 1u, status)) break;
            tc_fence_after();
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
                const float ws = PH == 0 ? S.wsc[s % kFacs][mat] : 1.f;
                const float4* f4 = reinterpret_cast<const float4*>(S.fac[s % kFacs]);
#pragma unroll
                for (int c = 0; c < NT / 16; ++c) {
                    if (c * 16 >= n) break;
                    float v[16];
                    tc_ld16(tmem + ((uint32_t) (warp * 32) << 16) + (uint32_t) ((b * kMats + mat) * NT + c * 16), v);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 f = f4[c * 4 + q];
                        float* o = &acc[mat][c * 16 + q * 4];
                        o[0] = fmaf(v[q * 4 + 0], f.x * ws, o[0]);
                        o[1] = fmaf(v[q * 4 + 1], f.y * ws, o[1]);
                        o[2] = fmaf(v[q * 4 + 2], f.z * ws, o[2]);
                        o[3] = fmaf(v[q * 4 + 3], f.w * ws, o[3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.tempty[b]);
            ++seg;
            const bool tile_end = (PH == 0 ? a.kb + 1 == KB : (a.kb + 1 == KB && a.g + 1 == G)) || s + 1 == nsteps;
            if (PH == 1 && (a.kb + 1 == KB || s + 1 == nsteps)) {
                // the group's columns go to their tokens
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (j >= n) break;
                    oacc[(P.slot[p0 + j] / p.topk) * 128 + tid] += acc[0][j];
                }
                clear();
            }
            if (tile_end) {
                const int first = a.tile * per_tile;                  // the tile's first step
                bool finish = seg == per_tile;
                // the columns that the group has, a bit each
                uint64_t have = n < 64 ? (1ull << n) - 1ull : ~0ull;
                if (kTokens) {
                    have = 0;
                    for (int j = 0; j < pairs; ++j) have |= 1ull << (P.slot[p0 + j] / p.topk);
                }
                auto chunk = [&](int c) { return (have >> (c * kCh) & ((1ull << kCh) - 1ull)) != 0; };
                if (!finish) {
                    float* dst = part_of(cta, first);
                    if (PH == 0) {
#pragma unroll
                        for (int c = 0; c < NT / kCh; ++c) {
                            if (!chunk(c)) continue;
#pragma unroll
                            for (int j = c * kCh; j < (c + 1) * kCh; ++j)
#pragma unroll
                                for (int mat = 0; mat < kMats; ++mat) __stcg(dst + (mat * NT + j) * 128 + tid, acc[mat][j]);
                        }
                    } else {
                        for (int t = 0; t < p.m; ++t) __stcg(dst + t * 128 + tid, oacc[t * 128 + tid]);
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
                                for (int h = 0; h < NT / kCh; ++h) {
                                    if (!chunk(h)) continue;
                                    float v[kMats][kCh];              // all of them on their way together
#pragma unroll
                                    for (int j = 0; j < kCh; ++j)
#pragma unroll
                                        for (int mat = 0; mat < kMats; ++mat) v[mat][j] = __ldcg(src + (mat * NT + h * kCh + j) * 128 + tid);
#pragma unroll
                                    for (int j = 0; j < kCh; ++j)
#pragma unroll
                                        for (int mat = 0; mat < kMats; ++mat) acc[mat][h * kCh + j] += v[mat][j];
                                }
                            } else {
                                for (int t = 0; t < p.m; t += 4) {
                                    float v[4];
#pragma unroll
                                    for (int q = 0; q < 4; ++q) v[q] = t + q < p.m ? __ldcg(src + (t + q) * 128 + tid) : 0.f;
#pragma unroll
                                    for (int q = 0; q < 4; ++q)
                                        if (t + q < p.m) oacc[(t + q) * 128 + tid] += v[q];
                                }
                            }
                        }
                    }
                }
                if (finish && PH == 0) {
                    // SwiGLU, then one scale for each token's 128 columns; NaN passes
                    // through.  kCh columns at a time: columns behind the group's last
                    // are computed with them and never stored.
                    const int ib = a.tile % NBI;
                    const float lim = p.limit;
                    if (kTokens)
                        for (int j = tid; j < pairs; j += 128) {
                            const int t = P.slot[p0 + j] / p.topk;
                            if (j == 0 || P.slot[p0 + j - 1] / p.topk != t) S.tokpair[t] = (short) (p0 + j);
                        }
#pragma unroll
                    for (int c = 0; c < NT / kCh; ++c) {
                        if (!chunk(c)) continue;
#pragma unroll
                        for (int j = c * kCh; j < (c + 1) * kCh; ++j) {
                            float g = acc[0][j], u = acc[kMats - 1][j];
                            g = g > lim ? lim : g;
                            u = u > lim ? lim : u < -lim ? -lim : u;
                            acc[0][j] = g / (1.f + expf(-g)) * u;
                            const uint32_t mx = __reduce_max_sync(0xffffffffu, abs_bits(acc[0][j]));
                            if (lane == 0) S.wmax[warp][j] = mx;
                        }
                    }
                    epi_sync();
#pragma unroll
                    for (int c = 0; c < NT / kCh; ++c) {
                        if (!chunk(c)) continue;
#pragma unroll
                        for (int j = c * kCh; j < (c + 1) * kCh; ++j) {
                            const uint32_t mx = max(max(S.wmax[0][j], S.wmax[1][j]), max(S.wmax[2][j], S.wmax[3][j]));
                            const float sa = fp8_scale(mx, p.pow2);
                            const uint32_t q = e4m3x2(fp8_quotient(acc[0][j], sa, __frcp_rn(sa), p.pow2), 0.f);
                            if (have >> j & 1ull) {
                                // an expert listed twice for a token has two pairs next to each other
                                int pr = kTokens ? S.tokpair[j] : p0 + j;
                                do {
                                    p.aq[(int64_t) pr * p.I + ib * 128 + tid] = (uint8_t) q;
                                    if (tid == 0) p.as[(int64_t) pr * NBI + ib] = sa;
                                } while (kTokens && ++pr < p0 + pairs && P.slot[pr] / p.topk == j);
                            }
                        }
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
    int64_t off_aq, off_as, off_xq, off_xs, off_part, bytes;
};

FmGeom fm_geom(int64_t m, int64_t topk, int64_t H, int64_t I) {
    FmGeom g{};
    const bool xq = m > kFmInlineRows;
    g.nt = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    const int64_t slots = m * topk;
    g.off_aq = EXL3_FP8_MOE_CTRL_BYTES;
    g.off_as = g.off_aq + align_up(slots * I, 256);
    g.off_xq = g.off_as + align_up(slots * (I / 128) * 4, 256);
    g.off_xs = g.off_xq + (xq ? align_up(m * H, 256) : 0);
    g.off_part = g.off_xs + (xq ? align_up(m * (H / 128) * 4, 256) : 0);
    const int64_t part_rows = 2 * g.nt > m ? 2 * g.nt : m;
    g.bytes = g.off_part + (int64_t) kFmMaxCtas * 2 * part_rows * 128 * 4;
    return g;
}

template <int NT, int PH>
int fm_launch(FmParams p, int sms, cudaStream_t stream) {
    using L = FmLayout<NT, PH>;
    // The two kernels share an SM while kernel 2 waits: 120 + 104 KB of its memory.
    constexpr int kBudget = (PH == 0 ? 120 : 104) * 1024;
    const int extra = 1024 + (int) sizeof(FmHead<NT>) + L::kXRing + (PH == 1 ? p.m * 512 : 0);
    static_assert(sizeof(FmHead<64>) + 64 * 512 + 1024 + 2 * FmLayout<64, 1>::kSlot <= 104 * 1024, "room for two blocks");
    int slots = (kBudget - extra) / L::kSlot;
    if (slots > kFmMaxSlotsW) slots = kFmMaxSlotsW;
    p.slots = slots;
    const int smem = extra + slots * L::kSlot;
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
    p.xs = reinterpret_cast<const float*>(sb + g.off_xs);
    p.as = reinterpret_cast<float*>(sb + g.off_as);
    p.part = reinterpret_cast<float*>(sb + g.off_part);
    p.ctrl = reinterpret_cast<uint32_t*>(sb);
    p.route = RouteIn{route->ids, route->weights, route->expert_map, route->n_global, route->ids_dtype, route->weights_dtype};
    p.limit = swiglu_limit;
    p.x_dtype = x_dtype; p.out_dtype = out_dtype; p.pow2 = pow2 != 0;
    p.xvec = aligned16(x);
    p.m = (int) m; p.topk = (int) topk; p.E = (int) n_experts; p.H = (int) hidden; p.I = (int) inter;
    auto s = static_cast<cudaStream_t>(stream);
    if (m > kFmInlineRows) {
        if ((rc = fp8_map(&p.xmap, sb + g.off_xq, m, hidden, hidden, g.nt, "exl3_fp8_moe_decode")) != EXL3_OK) return rc;
        if ((rc = fp8_quantize_launch(x, x_dtype, m, hidden, hidden, sb + g.off_xq, hidden, reinterpret_cast<float*>(sb + g.off_xs),
                                      1, m, 1, pow2 != 0, s)) != EXL3_OK)
            return rc;
    }
    if (g.nt == 16) return fm_run<16>(p, di.sms, s);
    if (g.nt == 32) return fm_run<32>(p, di.sms, s);
    return fm_run<64>(p, di.sms, s);
}
