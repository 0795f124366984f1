// fp8_moe.cu -- routed-expert MoE layer for a few tokens over e4m3 experts with
// one fp32 scale for each 128 x 128 block of a weight, in two kernels.
//   G = x . Wgate_e^T, U = x . Wup_e^T      (x in e4m3, scales by row and 128 columns)
//   a = silu(min(G, L)) * clamp(U, -L, L)   (fp32; quantised the same way)
//   out[t] = sum over the valid slots of weight * (a . Wdown_e^T)   (fp32, one cast)
// An x in 16 or 32 bits is quantised by kernel 1, once in every CTA while its first
// weights are on their way, up to four rows; above that by the quantiser's kernel
// before it.  (Quantising it inside kernel 1 for every output tile anew cost one
// warp about 2000 clocks a row and block: four tokens took 232 us.)
//
// Bound: the routed experts' weights, 3 * H * I bytes each, read once.  So both
// kernels do nothing but stream weight blocks: a 128 x 128 block is one TMA box
// and the M operand of four tcgen05.mma (K = 32 e4m3 each), the tokens are N, and
// each block's sums are read back from TMEM, scaled by the two scales and added
// to fp32 registers while the next block is multiplied.
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
// waits for kernel 1 to complete before it touches what kernel 1 wrote.  4096
// columns, top-8 of 256, calls in a CUDA graph: 1 token of I = 256 20.8 us, 4 of 2048
// 132.7 us (758 MB, 87 % of the copy rate; called one by one 137-148 us), 32 of 512
// with Zipf routes 110-113 us (400 MB; 105-126, as the routes and the GPU are).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "fp8.cuh"
#include "host.hpp"

namespace exl3 {

int fp8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, const char* what);
int fp8_quantize_launch(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq,
                        float* scale, int64_t sr, int64_t sg, int block_rows, bool pow2, cudaStream_t s);

// Status bits of this file's kernels on this device, whatever scratch they ran with
// (exl3_fp8_status): a captured call's scratch belongs to its graph and its control
// words are cleared with every replay.
__device__ uint32_t g_fp8_moe_status = 0u;

constexpr int kFmMaxRows = 64;
constexpr int kFmMaxSlots = 256;             // m * topk
constexpr int kFmMaxTopk = 16;
constexpr int kFmMaxInter = 8192;
constexpr int kFmMaxHidden = 16384;
constexpr int kFmMaxCtas = 160;
// Warps 0-3 epilogue, 4 producer, 5 MMA, 6 factors, 7 finisher.  Two warps on each of
// an SM's four register files: CTAs of both kernels fit side by side (kernel 2
// waits there, its ring filled), which three would not.
constexpr int kFmThreads = 256;
constexpr int kFmProducerWarp = 4;
constexpr int kFmMmaWarp = 5;
constexpr int kFmFacWarp = 6;
// Rows and width of an x that kernel 1 quantises itself, once a CTA and into its
// own shared memory (a launch less: 1 token of 4096 takes 20.4 us for 21.4, 4 tokens
// 130.5 for 133.1); above, the quantiser's launch comes first.  Four rows are what
// a warp quantises at once.  A wider x takes too much of the ring: with 8 experts of
// 2048 a token takes 33.3 us for 34.7 at 2048 columns, 49.7 for 51.1 at 4096, but
// 60.5 for 59.5 at 5120 and 72.2 for 67.4 at 6144.
constexpr int kFmInlineRows = 4;
constexpr int kFmInlineHidden = 4096;
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
    CUtensorMap xmap;            // x in e4m3 [m][H], box 128 x NT
    void* out;
    const float* w13s;           // [E][2 I / 128][H / 128]
    const float* w2s;            // [E][H / 128][I / 128]
    const void* x;               // an x that kernel 1 quantises: fp16 / bf16 / fp32 [m][H]
    int x_dtype, xvec;
    const float* xs;             // scales of an e4m3 x: xs[token * xsr + block * xsg]
    int64_t xsr, xsg;
    uint8_t* aq;                 // [slots][I] e4m3
    float* as;                   // [slots][I / 128]
    float* part;                 // partial sums of the CTAs' first and last tiles
    uint32_t* ctrl;
    RouteIn route;
    float limit;
    int out_dtype, pow2;
    int early;                   // all before the quantiser's launch is complete when kernel 1 starts
    int m, topk, E, H, I, slots;
};

// Pairs are the valid (token, slot)s ordered by (expert, slot); a group is up
// to NT pairs of one expert.
struct FmPlan {
    alignas(16) int id[kFmMaxSlots];
    short slot[kFmMaxSlots];          // pair -> slot
    short tok[kFmMaxSlots];           // pair -> token
    short pexp[kFmMaxSlots];          // pair -> expert
    short gstart[kFmMaxSlots + 2];    // group -> first pair; [G] = pairs
    uint8_t first[kFmMaxSlots];       // pair begins a group
    int wsum[8];
    int G;
};

// Shared memory of a CTA: a ring of weight blocks with the NT input rows of the
// block (16 + 2 .. 8 KB, so that few bytes wait while many are in flight), the
// head, kernel 2's output rows.  A step is one block of k: kernel 1 multiplies
// the gate and the up block, each into TMEM columns of its own, kernel 2 the down
// block.  D's columns are all tokens in kernel 1 -- those that are not the
// expert's are never used -- and the group's pairs in kernel 2.  INL (rows that a
// warp quantises at once, 1 or 4): kernel 1's x lies beside the ring, 8 rows x 128
// bytes a block of k and then its scales; the tensor core reads 16 rows, the second
// half being the next block's, whose columns are never used.
template <int NT, int PH, int INL = 0>
struct FmLayout {
    static_assert(!INL || (NT == 16 && PH == 0), "");
    static constexpr int kMats = PH == 0 ? 2 : 1;
    static constexpr int kBufs = NT <= 16 ? 4 : PH == 0 ? 2 : NT <= 32 ? 4 : 2;
    static constexpr int kTmemCols = NT * kMats * kBufs;             // 64 .. 256
    static constexpr int kSlot = (int) kFp8WTile + (INL ? 0 : NT * 128);
};

template <int NT>
struct FmHead {
    FmPlan plan;
    uint64_t wfull[kFmMaxSlotsW];        // a weight block has arrived
    uint64_t wdone[kFmMaxSlotsW];        // it has been multiplied
    uint64_t ffull[kFmMaxBufs];          // a step's factors are there
    uint64_t tfull[kFmMaxBufs];          // a step's sums are in TMEM
    uint64_t tempty[kFmMaxBufs];         // they have been read
    // Factors of a step's columns.  Twice kBufs deep: step s's are written once
    // step s - kBufs is in TMEM, i.e. the epilogue is done with s - 2 kBufs.
    alignas(16) float fac[2 * kFmMaxBufs][NT];
    float wsc[2 * kFmMaxBufs][2];
    alignas(16) uint32_t wmax[4][NT];
    short tokpair[NT];                   // a token's first pair in the group
    uint32_t tmem;
    uint32_t last;
    uint32_t fail;                       // status bits of this CTA's waits
};

// The head's bytes, so that what follows it starts on a swizzle atom.
template <int NT>
__host__ __device__ constexpr int fm_head_bytes() { return ((int) sizeof(FmHead<NT>) + 1023) / 1024 * 1024; }

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The epilogue hands a part that it has stored to the finisher and goes on.
__device__ __forceinline__ void part_ready() { asm volatile("bar.arrive 2, 160;" ::: "memory"); }
__device__ __forceinline__ void part_wait() { asm volatile("bar.sync 2, 160;" ::: "memory"); }

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
        P.tok[before] = (short) (tid / p.topk);
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

// A step's factors on their way: column h * 32 + lane, and a block's scale.
template <int NT>
struct FmFac {
    float f[(NT + 31) / 32];
    float ws;
};

// A CTA's part of a tile that it shares: slot 1 where its range began before the tile did.
__device__ __forceinline__ float* fm_part(float* part, int rows_pt, int c, int first, int C, int total) {
    return part + ((int64_t) c * 2 + (fm_start(c, C, total) >= first ? 0 : 1)) * rows_pt * 128;
}

// Sums of rows of the parts of CTAs c0 .. c1, in their order; four values a lane,
// the loads of four CTAs in flight.
template <int NR>
__device__ __forceinline__ void fm_sum(float4 (&out)[NR], const int (&row)[NR], int n, float* part, int rows_pt, int c0, int c1,
                                       int first, int C, int total, int lane) {
#pragma unroll
    for (int h = 0; h < NR; ++h) out[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0; c <= c1; c += 4) {
        float4 v[4][NR];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool on = c + q <= c1 && fm_start(c + q, C, total) != fm_start(c + q + 1, C, total);
            const float4* src = reinterpret_cast<const float4*>(fm_part(part, rows_pt, min(c + q, c1), first, C, total));
#pragma unroll
            for (int h = 0; h < NR; ++h)
                v[q][h] = on && h < n ? __ldcg(src + row[h] * 32 + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int h = 0; h < NR; ++h) {
                out[h].x += v[q][h].x; out[h].y += v[q][h].y; out[h].z += v[q][h].z; out[h].w += v[q][h].w;
            }
    }
}

// silu(min(g, L)) * clamp(u, -L, L); NaN passes through
__device__ __forceinline__ float fm_swiglu(float g, float u, float lim) {
    g = g > lim ? lim : g;
    u = u > lim ? lim : u < -lim ? -lim : u;
    return g / (1.f + expf(-g)) * u;
}

template <int NT, int PH, int INL>
__global__ void __launch_bounds__(kFmThreads, NT <= 32 ? 2 : 1) fp8_moe_kernel(const __grid_constant__ FmParams p) {
    using L = FmLayout<NT, PH, INL>;
    constexpr int kMats = L::kMats, kBufs = L::kBufs, kFacs = 2 * L::kBufs;
    // The CTA's last tile, where the CTA completes its count: the epilogue's warps
    // finish it at once, but all warps once all have come to an end where it can have
    // many rows (32 tokens 114.4 us for 120.2, 4 tokens 130.9 for 130.3, one 21.1 for 20.7).
    constexpr bool kAllFinish = NT > 16;
    constexpr int kCh = NT < 32 ? 4 : 8;                              // columns handled together at a tile's end
    extern __shared__ uint8_t fm_raw[];
    uint8_t* ring = fm_raw + ((1024u - (smem_u32(fm_raw) & 1023u)) & 1023u);
    FmHead<NT>& S = *reinterpret_cast<FmHead<NT>*>(ring + p.slots * L::kSlot);
    float* oacc = reinterpret_cast<float*>(ring + p.slots * L::kSlot + sizeof(FmHead<NT>));    // PH 1: [m][128]
    uint8_t* xres = ring + p.slots * L::kSlot + fm_head_bytes<NT>();                           // INL: [KB + 1][1024]
    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const int C = (int) gridDim.x, cta = (int) blockIdx.x;
    const int NBI = p.I / 128, NBH = p.H / 128, KB = PH == 0 ? NBH : NBI;
    const int W = p.slots;
    float* xsc = reinterpret_cast<float*>(xres + (KB + 1) * 1024);                             // INL: [KB][8]
    uint32_t* status = &S.fail;

    if (tid == 0) {
        tmap_prefetch(PH == 0 ? &p.w13 : &p.w2);
        for (int s = 0; s < W; ++s) { mbar_init(&S.wfull[s], 1); mbar_init(&S.wdone[s], 1); }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&S.ffull[b], 1);
            mbar_init(&S.tfull[b], 1);
            mbar_init(&S.tempty[b], 4);
        }
        S.last = 0u;
        S.fail = 0u;
        fence_barrier_init();
    }
    if (warp == kFmMmaWarp) tmem_alloc(&S.tmem, L::kTmemCols);
    if (PH == 0) {
        // Kernel 2 may start once what came before the layer (the routes among
        // it) is complete: at once where the quantiser, which waits for that before it
        // lets this kernel start, ran in between -- only x is waited for then, by
        // those who read it -- otherwise behind this kernel's own wait.
        if (!p.early) pdl_wait();
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
    // Parts: what a CTA has of a tile that it shares; slot 1 where its range began before the tile did.
    const int rows_pt = PH == 0 ? kMats * NT : p.m;                   // rows of 128 in a part
    auto token = [&](int pair) { return (int) P.tok[pair]; };

    // A shared tile whose count this CTA completed: the parts are added in CTA
    // order and the tile is finished, by warp w of n.
    auto finish_shared = [&](int tile, int w, int nw) {
        const int first = tile * per_tile;
        const int c0 = fm_owner(first, C, total), c1 = fm_owner(first + per_tile - 1, C, total);
        float4 o[2 * kMats];
        int row[2 * kMats];
        if (PH == 0) {
            const int g = tile / NBI, ib = tile % NBI, p0 = P.gstart[g], pe = P.gstart[g + 1];
            for (int pr = p0 + 2 * w; pr < pe; pr += 2 * nw) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = token(min(pr + h, pe - 1));
                    row[h * kMats] = col;
                    row[h * kMats + kMats - 1] = (kMats - 1) * NT + col;
                }
                fm_sum<2 * kMats>(o, row, pr + 1 < pe ? 2 * kMats : kMats, p.part, rows_pt, c0, c1, first, C, total, lane);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (pr + h >= pe) break;
                    const float4 g4 = o[h * kMats], u4 = o[h * kMats + kMats - 1];
                    float v[4] = {fm_swiglu(g4.x, u4.x, p.limit), fm_swiglu(g4.y, u4.y, p.limit),
                                  fm_swiglu(g4.z, u4.z, p.limit), fm_swiglu(g4.w, u4.w, p.limit)};
                    const uint32_t mx = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
                    const float sa = fp8_scale(__reduce_max_sync(0xffffffffu, mx), p.pow2);
                    *reinterpret_cast<uint32_t*>(p.aq + (int64_t) (pr + h) * p.I + ib * 128 + lane * 4) =
                        fp8_pack4(v[0], v[1], v[2], v[3], sa, p.pow2 != 0);
                    if (lane == 0) p.as[(int64_t) (pr + h) * NBI + ib] = sa;
                }
            }
        } else {
            for (int t = 2 * w; t < p.m; t += 2 * nw) {
                row[0] = t;
                row[1] = t + 1;
                fm_sum<2 * kMats>(o, row, min(2, p.m - t), p.part, rows_pt, c0, c1, first, C, total, lane);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (t + h >= p.m) break;
                    const int64_t at = (int64_t) (t + h) * p.H + tile * 128 + lane * 4;
                    store_out(p.out, p.out_dtype, at, o[h].x);
                    store_out(p.out, p.out_dtype, at + 1, o[h].y);
                    store_out(p.out, p.out_dtype, at + 2, o[h].z);
                    store_out(p.out, p.out_dtype, at + 3, o[h].w);
                }
            }
        }
    };

    if (INL && warp != kFmProducerWarp) {
        // x's blocks of this CTA's range, while the first weights are on their way
        const int w = warp < kFmProducerWarp ? warp : warp - 1, lr = XRows::row(INL, lane);
#pragma unroll 1
        for (int i = w; i < min(nsteps, KB); i += 7) {
            const int kb = (beg + i) % KB;
            XRows r;
            r.load(INL, p.x, p.x_dtype, (int64_t) lr * p.H + kb * 128 + XRows::col(INL, lane), lr < p.m ? 16 : 0, p.xvec != 0);
            float sx;
            const uint4 q = r.quantize(INL, p.x_dtype, p.pow2 != 0, sx);
            if (lr < p.m) {
                XRows::store(INL, xres + kb * 1024, lr, lane, q);
                if (INL == 1 ? lane == 0 : (lane & 7) == 0) xsc[kb * 8 + lr] = sx;
            }
        }
        fence_proxy_async_smem();
        asm volatile("bar.sync 3, 224;" ::: "memory");
    }

    if (warp == kFmProducerWarp) {
        if (lane == 0 && nsteps > 0) {
            const int nblk = nsteps * kMats;
            auto weights = [&](const FmAt<PH>& a, int mat, int slot) {
                const int e = P.pexp[P.gstart[a.g]];
                mbar_arrive_expect_tx(&S.wfull[slot], (uint32_t) L::kSlot);
                const int row = PH == 0 ? e * 2 * p.I + mat * p.I + (a.tile % NBI) * 128 : e * p.H + a.tile * 128;
                tma_load_2d_once(ring + slot * L::kSlot, PH == 0 ? &p.w13 : &p.w2, a.kb * 128, row, &S.wfull[slot]);
            };
            auto inputs = [&](const FmAt<PH>& a, int slot) {
                if (PH == 0) tma_load_2d(ring + slot * L::kSlot + kFp8WTile, &p.xmap, a.kb * 128, 0, &S.wfull[slot]);
                else tma_load_2d(ring + slot * L::kSlot + kFp8WTile, &p.amap, a.kb * 128, P.gstart[a.g], &S.wfull[slot]);
            };
            FmAt<PH> a(beg, G, NBI, KB);
            auto mat_of = [](int t) { return PH == 0 ? t & 1 : 0; };
            auto next = [&](FmAt<PH>& at, int t) { if (PH == 1 || (t & 1)) at.next(); };
            // a ring of weights ahead of the wait: no kernel that may still run writes them
            FmAt<PH> a0 = a;
            int t = 0;
            for (; t < min(W, nblk); ++t) { weights(a, mat_of(t), t); next(a, t); }
            if (!INL) {
                pdl_wait();
                fence_proxy_async_global();
                for (int i = 0; i < t; ++i) { inputs(a0, i); next(a0, i); }
            }
            int issued = t;
            for (; t < nblk; ++t) {
                const int slot = t % W;
                if (t >= W && !mbar_wait(&S.wdone[slot], ((t / W) + 1u) & 1u, status)) break;
                weights(a, mat_of(t), slot);
                if (!INL) inputs(a, slot);
                next(a, t);
                ++issued;
            }
            // no copy may still be in flight when the CTA retires
            for (int i = max(0, issued - W); i < issued; ++i)
                if (!mbar_wait(&S.wfull[i % W], (i / W) & 1u, status)) break;
        } else {
            pdl_wait();
        }
    } else if (warp == kFmMmaWarp) {
        pdl_wait();                                                   // the bounded waits begin behind it
        const uint64_t wdesc0 = sdesc_sw128(smem_u32(ring)), xdesc0 = sdesc_sw128(smem_u32(xres));
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        int slot = 0;
        uint32_t wpar = 0;
        bool ok = true;
        for (int s = 0; s < nsteps && ok; ++s, a.next()) {
            const int b = s % kBufs;
            const int n = PH == 0 ? p.m : P.gstart[a.g + 1] - P.gstart[a.g];
            const uint32_t id = __shfl_sync(0xffffffffu, idesc_f16(128, (n + 15) & ~15), 0);
            ok = mbar_poll2_lanes(&S.ffull[b], (s / kBufs) & 1u, &S.tempty[b], ((s / kBufs) + 1u) & 1u, status);
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
                ok = ok && mbar_poll_lanes(&S.wfull[slot], wpar, status);
                if (!ok) break;
                tc_fence_after();
                const uint64_t wd = wdesc0 + (uint64_t) (slot * (L::kSlot >> 4));
                const uint64_t xd = INL ? xdesc0 + (uint64_t) (a.kb * 64) : wd + (kFp8WTile >> 4);
                if (elect_lane()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) tc_mma_f8(tmem + (b * kMats + mat) * NT, wd + 2 * q, xd + 2 * q, id, q);
                    tc_commit(&S.wdone[slot]);
                    if (mat + 1 == kMats) tc_commit(&S.tfull[b]);
                }
                if (++slot == W) { slot = 0; wpar ^= 1u; }
            }
        }
    } else if (warp == kFmFacWarp) {
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        if (PH == 0 && cta == 0)
            for (int i = lane; i < NBH; i += 32) p.ctrl[kFmCntB + i] = 0u;   // kernel 2's counters
        // The factors of a step's columns: x's scales and the two blocks' (kernel 1),
        // or the down input's, the block's and the route's.  Loaded two steps ahead.
        pdl_wait();
        if (PH == 1)
            for (int i = cta * 32 + lane; i < G * NBI; i += C * 32) p.ctrl[kFmCntA + i] = 0u;   // kernel 1's
        FmAt<PH> at = a;
        auto load = [&](int s) {
            FmFac<NT> v;
            v.ws = 0.f;
#pragma unroll
            for (int h = 0; h < (NT + 31) / 32; ++h) v.f[h] = 0.f;
            if (s >= nsteps) return v;
            const int p0 = P.gstart[at.g], n = PH == 0 ? p.m : P.gstart[at.g + 1] - p0, e = P.pexp[p0];
            if (PH == 1) v.ws = __ldg(p.w2s + ((int64_t) e * NBH + at.tile) * NBI + at.kb);
            else if (lane < 2) v.ws = __ldg(p.w13s + ((int64_t) e * 2 * NBI + lane * NBI + at.tile % NBI) * NBH + at.kb);
#pragma unroll
            for (int h = 0; h < (NT + 31) / 32; ++h) {
                const int j = h * 32 + lane;
                if (j < n) v.f[h] = INL ? xsc[at.kb * 8 + j] : PH == 0 ? __ldcg(p.xs + j * p.xsr + at.kb * p.xsg) : __ldcg(p.as + (int64_t) (p0 + j) * NBI + at.kb);
            }
            at.next();
            return v;
        };
        FmFac<NT> v0 = load(0), v1 = load(1);
        for (int s = 0; s < nsteps; ++s, a.next()) {
            const int b = s % kBufs, p0 = P.gstart[a.g], n = P.gstart[a.g + 1] - p0;
            const FmFac<NT> v = v0;
            v0 = v1;
            v1 = load(s + 2);
            if (!mbar_wait_lanes(&S.tfull[b], ((s / kBufs) + 1u) & 1u, status)) break;
#pragma unroll
            for (int h = 0; h < (NT + 31) / 32; ++h) {
                const int j = h * 32 + lane;
                float f = v.f[h];
                if (PH == 1) f = j < n ? f * v.ws * route_weight(p.route, P.slot[p0 + j]) : 0.f;
                if (j < NT) S.fac[s % kFacs][j] = f;
            }
            if (PH == 0 && lane < 2) S.wsc[s % kFacs][lane] = v.ws;
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.ffull[b]);
        }
    } else if (warp > kFmFacWarp) {
        // -------------------------------------------------------------- finisher
        // The first tile of the CTA's range, where the CTA shares it and goes on
        // behind it: a chain of trips to L2, during which the epilogue takes the
        // next steps (6 us for one token when the epilogue did it itself, with the
        // CTA's weights waiting).
        if (PH == 1) pdl_wait();
        if (nsteps > 0) {
            const int first = beg / per_tile * per_tile, steps = min(end, first + per_tile) - beg;
            if (steps != per_tile && beg + steps < end) {
                part_wait();
                uint32_t done = 0u;
                if (lane == 0) done = atom_add_acq_rel_gpu(&p.ctrl[(PH == 0 ? kFmCntA : kFmCntB) + first / per_tile], (uint32_t) steps) + (uint32_t) steps;
                done = __shfl_sync(0xffffffffu, done, 0);
                __syncwarp();                                         // a shuffle orders no memory: lane 0's acquire before all lanes' loads
                if (done == (uint32_t) per_tile) finish_shared(first / per_tile, 0, 1);
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
        pdl_wait();
        if (PH == 1) {
            if (total == 0)
                for (int64_t i = (int64_t) cta * 128 + tid; i < (int64_t) p.m * p.H; i += (int64_t) C * 128)
                    store_out(p.out, p.out_dtype, i, 0.f);
            for (int t = 0; t < p.m; ++t) oacc[t * 128 + tid] = 0.f;
        }
        clear();
        FmAt<PH> a(beg, max(G, 1), NBI, KB);
        int seg = 0;                                                  // steps of the current tile so far
        // The four warps meet at barriers of a fixed count at tile ends, and each has
        // a verdict of its own on every wait.  So a warp whose wait gave up walks on
        // through its steps and meets them all, without waiting, reading TMEM or
        // arriving any more; what it leaves is in bounds, and the status marks it.
        bool ok = true;
        for (int s = 0; s < nsteps; ++s) {
            const int b = s % kBufs;
            const int p0 = P.gstart[a.g], pairs = P.gstart[a.g + 1] - p0, n = PH == 0 ? p.m : pairs;   // n: D's columns
            ok = ok && mbar_wait_lanes(&S.tfull[b], (s / kBufs) & 1u, status);
            tc_fence_after();
#pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
                const float ws = PH == 0 ? S.wsc[s % kFacs][mat] : 1.f;
                const float4* f4 = reinterpret_cast<const float4*>(S.fac[s % kFacs]);
#pragma unroll
                for (int c = 0; c < NT / 16; ++c) {
                    if (c * 16 >= n || !ok) break;
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
            if (ok && lane == 0) mbar_arrive(&S.tempty[b]);
            ++seg;
            const bool tile_end = (PH == 0 ? a.kb + 1 == KB : (a.kb + 1 == KB && a.g + 1 == G)) || s + 1 == nsteps;
            if (PH == 1 && (a.kb + 1 == KB || s + 1 == nsteps)) {
                // the group's columns go to their tokens
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (j >= n) break;
                    oacc[token(p0 + j) * 128 + tid] += acc[0][j];
                }
                clear();
            }
            if (tile_end) {
                const bool whole = seg == per_tile;
                // kernel 1: the columns whose tokens the group has, a bit each
                uint64_t have = 0;
                if (PH == 0)
                    for (int j = 0; j < pairs; ++j) have |= 1ull << token(p0 + j);
                auto chunk = [&](int c) { return (have >> (c * kCh) & ((1ull << kCh) - 1ull)) != 0; };
                if (!whole) {
                    float* dst = fm_part(p.part, rows_pt, cta, a.tile * per_tile, C, total);
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
                    if (s + 1 < nsteps) {
                        part_ready();
                    } else {
                        epi_sync();
                        if (tid == 0)
                            S.last = atom_add_acq_rel_gpu(&p.ctrl[(PH == 0 ? kFmCntA : kFmCntB) + a.tile], (uint32_t) seg) + (uint32_t) seg == (uint32_t) per_tile;
                        if (!kAllFinish) {
                            epi_sync();
                            if (S.last) finish_shared(a.tile, warp, 4);
                        }
                    }
                }
                if (whole && PH == 0) {
                    // SwiGLU, then one scale for each token's 128 columns; NaN passes
                    // through.  kCh columns at a time: columns behind the group's last
                    // are computed with them and never stored.
                    const int ib = a.tile % NBI;
                    for (int j = tid; j < pairs; j += 128) {
                            const int t = token(p0 + j);
                            if (j == 0 || token(p0 + j - 1) != t) S.tokpair[t] = (short) (p0 + j);
                        }
#pragma unroll
                    for (int c = 0; c < NT / kCh; ++c) {
                        if (!chunk(c)) continue;
#pragma unroll
                        for (int j = c * kCh; j < (c + 1) * kCh; ++j) {
                            acc[0][j] = fm_swiglu(acc[0][j], acc[kMats - 1][j], p.limit);
                            const uint32_t mx = __reduce_max_sync(0xffffffffu, abs_bits(acc[0][j]));
                            if (lane == 0) S.wmax[warp][j] = mx;
                        }
                    }
                    epi_sync();
                    // a lane has a column's scale and its reciprocal: every thread dividing
                    // for itself, 32 tokens took 125.6 us, so 120.1
                    float sl[(NT + 31) / 32], il[(NT + 31) / 32];
#pragma unroll
                    for (int h = 0; h < (NT + 31) / 32; ++h) {
                        const int j = min(h * 32 + lane, NT - 1);
                        sl[h] = fp8_scale(max(max(S.wmax[0][j], S.wmax[1][j]), max(S.wmax[2][j], S.wmax[3][j])), p.pow2);
                        il[h] = __frcp_rn(sl[h]);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if (!(have >> j & 1ull)) continue;
                        const float sa = __shfl_sync(0xffffffffu, sl[j >> 5], j & 31), inv = __shfl_sync(0xffffffffu, il[j >> 5], j & 31);
                        const uint32_t q = fp8_pack1(acc[0][j], sa, inv, p.pow2 != 0);
                        // an expert listed twice for a token has two pairs next to each other
                        int pr = S.tokpair[j];
                        do {
                            p.aq[(int64_t) pr * p.I + ib * 128 + tid] = (uint8_t) q;
                            if (tid == 0) p.as[(int64_t) pr * NBI + ib] = sa;
                        } while (++pr < p0 + pairs && token(pr) == j);
                    }
                    epi_sync();                                       // wmax is free for the next tile
                }
                if (whole && PH == 1)
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
    if (tid == 0 && S.fail != 0u) {
        set_error(p.ctrl + 2, S.fail);
        set_error(&g_fp8_moe_status, S.fail);
    }
    if (kAllFinish && S.last) finish_shared((end - 1) / per_tile, warp, kFmThreads / 32);
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
    g.nt = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    const int64_t slots = m * topk;
    g.off_aq = EXL3_FP8_MOE_CTRL_BYTES;
    g.off_as = g.off_aq + align_up(slots * I, 256);
    g.off_xq = g.off_as + align_up(slots * (I / 128) * 4, 256);
    g.off_xs = g.off_xq + align_up(m * H, 256);
    g.off_part = g.off_xs + align_up(m * (H / 128) * 4, 256);
    const int64_t part_rows = 2 * g.nt > m ? 2 * g.nt : m;
    g.bytes = g.off_part + (int64_t) kFmMaxCtas * 2 * part_rows * 128 * 4;
    return g;
}

template <int NT, int PH, int INL>
int fm_launch(FmParams p, int sms, cudaStream_t stream) {
    using L = FmLayout<NT, PH, INL>;
    // The two kernels share an SM while kernel 2 waits: 120 + 104 KB of its memory.
    constexpr int kBudget = (PH == 0 ? 120 : 104) * 1024;
    static_assert(sizeof(FmHead<64>) + 64 * 512 + 1024 + 2 * FmLayout<64, 1>::kSlot <= 104 * 1024, "room for two blocks");
    const int extra = INL ? 1024 + fm_head_bytes<NT>() + (p.H / 128 + 1) * 1024 + p.H / 128 * 32
                          : 1024 + (int) sizeof(FmHead<NT>) + (PH == 1 ? p.m * 512 : 0);
    int slots = (kBudget - extra) / L::kSlot;
    if (slots > kFmMaxSlotsW) slots = kFmMaxSlotsW;
    p.slots = slots;
    const int smem = extra + slots * L::kSlot;
    static std::once_flag once[64];
    int dev = 0;
    EXL3_CUDA(cudaGetDevice(&dev));
    cudaError_t attr = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr = cudaFuncSetAttribute(fp8_moe_kernel<NT, PH, INL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget);
        if (attr == cudaSuccess)   // all of it, or the SM's split made for one CTA keeps the other kernel's out
            attr = cudaFuncSetAttribute(fp8_moe_kernel<NT, PH, INL>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
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
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, fp8_moe_kernel<NT, PH, INL>, p));
    return EXL3_OK;
}

template <int NT, int INL = 0>
int fm_run(const FmParams& p, int sms, cudaStream_t s) {
    const int rc = fm_launch<NT, 0, INL>(p, sms, s);
    return rc != EXL3_OK ? rc : fm_launch<NT, 1, 0>(p, sms, s);
}

}  // namespace

// Reads the word into `status` (host memory) and clears it on request; synchronizes.
int fp8_moe_status(int clear, uint32_t* status, cudaStream_t s) {
    EXL3_CUDA(cudaMemcpyFromSymbolAsync(status, g_fp8_moe_status, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, s));
    EXL3_CUDA(cudaStreamSynchronize(s));
    if (clear) {
        const uint32_t zero = 0u;
        EXL3_CUDA(cudaMemcpyToSymbolAsync(g_fp8_moe_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s));
        EXL3_CUDA(cudaStreamSynchronize(s));
    }
    return EXL3_OK;
}

}  // namespace exl3

extern "C" int64_t exl3_fp8_moe_max_rows(void) { return exl3::kFmMaxRows; }

extern "C" int64_t exl3_fp8_moe_scratch_bytes(int64_t m, int64_t topk, int64_t hidden, int64_t inter) {
    using namespace exl3;
    if (m < 1 || m > kFmMaxRows || topk < 1 || topk > kFmMaxTopk || m * topk > kFmMaxSlots || hidden < 128 || hidden % 128 ||
        hidden > kFmMaxHidden || inter < 128 || inter % 128 || inter > kFmMaxInter)
        return -1;
    return fm_geom(m, topk, hidden, inter).bytes;
}

extern "C" int exl3_fp8_moe_decode(const void* x, int x_dtype, const float* x_scale, void* out, int out_dtype, int64_t m, int64_t hidden,
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
    EXL3_REQUIRE(x_dtype >= 0 && x_dtype <= 3 && out_dtype >= 0 && out_dtype <= 2 && route->weights_dtype >= 0 &&
                     route->weights_dtype <= 2 && (route->ids_dtype == 0 || route->ids_dtype == 1),
                 EXL3_ERR_ARG, "exl3_fp8_moe_decode: dtypes must be fp16, bf16 or fp32 (x: e4m3 too), ids int32 or int64");
    EXL3_REQUIRE((x_dtype == EXL3_DTYPE_E4M3) == (x_scale != nullptr) && (x_scale == nullptr || aligned16(x)), EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: x_scale goes with an e4m3 x, 16-byte aligned, and only with one");
    EXL3_REQUIRE(route->expert_map == nullptr || route->n_global >= 1, EXL3_ERR_ARG, "exl3_fp8_moe_decode: empty expert map");
    EXL3_REQUIRE(swiglu_limit > 0.f, EXL3_ERR_ARG, "exl3_fp8_moe_decode: the SwiGLU limit must be positive");
    EXL3_REQUIRE(aligned16(gate_up) && aligned16(down) && aligned16(scratch), EXL3_ERR_ARG,
                 "exl3_fp8_moe_decode: weights and scratch must be 16-byte aligned");
    EXL3_REQUIRE(aligned_to(x, dtype_bytes(x_dtype)) && aligned_to(out, dtype_bytes(out_dtype)) && aligned_to(x_scale, 4) &&
                     aligned_to(gate_up_scale, 4) && aligned_to(down_scale, 4) && aligned_to(route->ids, route->ids_dtype ? 8 : 4) &&
                     aligned_to(route->weights, dtype_bytes(route->weights_dtype)) && aligned_to(route->expert_map, 8),
                 EXL3_ERR_ARG, "exl3_fp8_moe_decode: x, out, scales, ids, routing weights and map must be aligned to their elements");
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
    p.out = out; p.w13s = gate_up_scale; p.w2s = down_scale;
    p.aq = sb + g.off_aq;
    p.as = reinterpret_cast<float*>(sb + g.off_as);
    p.part = reinterpret_cast<float*>(sb + g.off_part);
    p.ctrl = reinterpret_cast<uint32_t*>(sb);
    p.route = RouteIn{route->ids, route->weights, route->expert_map, route->n_global, route->ids_dtype, route->weights_dtype};
    p.limit = swiglu_limit;
    p.out_dtype = out_dtype; p.pow2 = pow2 != 0;
    p.m = (int) m; p.topk = (int) topk; p.E = (int) n_experts; p.H = (int) hidden; p.I = (int) inter;
    auto s = static_cast<cudaStream_t>(stream);
    const void* xq = x;
    p.xs = x_scale; p.xsr = hidden / 128; p.xsg = 1;
    if (x_dtype != EXL3_DTYPE_E4M3 && m <= kFmInlineRows && hidden <= kFmInlineHidden) {
        p.x = x;
        p.x_dtype = x_dtype;
        p.xvec = aligned16(x);
        return m == 1 ? fm_run<16, 1>(p, di.sms, s) : fm_run<16, kFmInlineRows>(p, di.sms, s);
    }
    if (x_dtype != EXL3_DTYPE_E4M3) {
        float* xs = reinterpret_cast<float*>(sb + g.off_xs);
        xq = sb + g.off_xq;
        if ((rc = fp8_quantize_launch(x, x_dtype, m, hidden, hidden, sb + g.off_xq, hidden, xs, 1, m, 1, pow2 != 0, s)) != EXL3_OK) return rc;
        p.xs = xs; p.xsr = 1; p.xsg = m;
        p.early = 1;
    }
    if ((rc = fp8_map(&p.xmap, xq, m, hidden, hidden, g.nt, "exl3_fp8_moe_decode")) != EXL3_OK) return rc;
    if (g.nt == 16) return fm_run<16>(p, di.sms, s);
    if (g.nt == 32) return fm_run<32>(p, di.sms, s);
    return fm_run<64>(p, di.sms, s);
}
