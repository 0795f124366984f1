// fp8.cuh -- device helpers shared by the e4m3 operators: the group scale, the
// correctly rounded e4m3 quotient, activation loads, the fp8 tensor-core
// instruction and cluster (distributed shared memory) accesses.
#pragma once

#include "tcgen05.cuh"

namespace exl3 {

constexpr int kFp8Block = 128;          // columns (and weight rows) that share one scale
constexpr float kE4M3Max = 448.0f;
constexpr int kDtE4M3 = 3;              // EXL3_DTYPE_E4M3
constexpr uint32_t kFp8WTile = 128 * 128;   // one weight block, bytes

// ---------------------------------------------------------------- quantising
// Scale of a group from the bits of its largest magnitude (non-negative
// floats order like their bits; a NaN orders above infinity, so it is kept):
// max(amax / 448, 2^-126), or the smallest power of two not below that.  The
// power of two is found on the rounded quotient: amax <= 448 * 2^e if and only
// if RN(amax / 448) <= 2^e, because 2^e is an fp32 number and the next amax
// above 448 * 2^e already rounds above it.
__device__ __forceinline__ float fp8_scale(uint32_t amax_bits, bool pow2) {
    float s = __fdiv_rn(__uint_as_float(amax_bits), kE4M3Max);
    if (s < 0x1p-126f) s = 0x1p-126f;
    if (pow2 && s < INFINITY) {
        const uint32_t b = __float_as_uint(s);
        s = __uint_as_float((b + 0x7FFFFFu) & 0xFF800000u);
    }
    return s;
}

// x / s to within the e4m3 rounding that follows, i.e. RN_e4m3 of the result
// is RN_e4m3 of the real quotient.  q = x * (1 / s) is off by at most two units
// in its last place (two roundings of 2^-24), which moves the e4m3 rounding
// only next to a midpoint of two e4m3 values.  Those have at most 5 significant
// bits, as the values themselves do, i.e. 19 low bits that are zero.  Where q is
// within two units of such a number v, the remainder r = x - v * s, which one FMA
// has exactly, says on which side of v the real quotient v + r / s lies; v + 64 r
// / s keeps that side, does not round back to v (r is a multiple of 2^-27 of v *
// s at least, so 64 r / s is a unit in the last place) and is still 2^-15 of v at
// most, far from the next boundary.  A tie (r = 0) stays v, for the conversion to
// round to even.  Both FMAs are taken with the sign turned (v * s - x, times
// -64 / s), so that -0 stays -0: (-0) * s + 0 is +0, times a negative number -0,
// plus v = -0 is -0.  All of it is arithmetic without a branch: 16-bit inputs meet
// midpoints often, because amax divides many of their multiples by 448, and a
// branch for each value, predicated or voted, was slower (8192 x 4096: 28 us).
__device__ __forceinline__ float fp8_quotient_fast(float x, float s, float inv) {
    const float q = x * inv;
    const uint32_t b = __float_as_uint(q);
    const float v = __uint_as_float((b + 0x40000u) & 0xFFF80000u);
    const float side = __fmaf_rn(__fmaf_rn(v, s, -x), -64.f * inv, v);
    return ((b + 2u) & 0x7FFFFu) <= 4u ? side : q;
}

// The same for any scale: a remainder clear of the subnormal numbers for tiny
// ones, and nothing multiplied by an infinite one.
static __device__ __noinline__ void fp8_quotients_any(float* x, int n, float s, float inv) {
    const float up = s < 0x1p-60f ? 0x1p64f : 1.f;
    for (int i = 0; i < n; ++i) {
        const float q = x[i] * inv;
        const uint32_t b = __float_as_uint(q), v = (b + 0x40000u) & 0xFFF80000u;
        float o = q;
        if (((b + 2u) & 0x7FFFFu) <= 4u && s < INFINITY) {
            const float r = __fmaf_rn(-__uint_as_float(v), s * up, x[i] * up);
            o = __uint_as_float(r == 0.f || q == 0.f ? v : (r > 0.f) == (q > 0.f) ? v + 1u : v - 1u);
        }
        x[i] = o;
    }
}

__device__ __forceinline__ bool fp8_easy(float s) { return s >= 0x1p-60f && s < 0x1p100f; }

// N quotients by one scale, with one branch for all of them.
template <int N>
__device__ __forceinline__ void fp8_quotients(float (&v)[N], float s, float inv, bool pow2) {
    if (pow2 || s == 0x1p-126f) {                  // exact; the latter: rows of zeros, and lanes without a row
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= inv;
    } else if (fp8_easy(s)) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fp8_quotient_fast(v[i], s, inv);
    } else {
        float t[N];                                // its address keeps `v` itself in registers
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = v[i];
        fp8_quotients_any(t, N, s, inv);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i];
    }
}

// Two fp32 -> two e4m3 bytes (nearest, ties to even, finite values saturate),
// `lo` in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four values by one scale -> e4m3 bytes; one copy of the code, for places that
// run it a few times only.
static __device__ __noinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float s, bool pow2) {
    float v[4] = {a, b, c, d};
    fp8_quotients(v, s, __frcp_rn(s), pow2);
    return e4m3x2(v[0], v[1]) | (e4m3x2(v[2], v[3]) << 16);
}

static __device__ __noinline__ uint32_t fp8_pack1(float a, float s, float inv, bool pow2) {
    float v[1] = {a};
    fp8_quotients(v, s, inv, pow2);
    return e4m3x2(v[0], 0.f) & 0xFFu;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// ---------------------------------------------------------------- loads
__device__ __forceinline__ float load_f32(const void* x, int dtype, int64_t i) {
    if (dtype == 0) return __half2float(reinterpret_cast<const __half*>(x)[i]);
    if (dtype == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[i]);
    return reinterpret_cast<const float*>(x)[i];
}

// Four values from element i on, as they lie in memory (a 16-bit type in the
// first two words, e4m3 in the first), read one by one; those at or past `left`
// are zero.
__device__ __forceinline__ uint4 load_raw4_tail(const void* x, int dtype, int64_t i, int left) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (q >= left) continue;
        if (dtype == 2) w[q] = reinterpret_cast<const uint32_t*>(x)[i + q];
        else if (dtype == kDtE4M3) w[0] |= (uint32_t) reinterpret_cast<const uint8_t*>(x)[i + q] << (8 * q);
        else w[q >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(x)[i + q] << (16 * (q & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void unpack4(const uint4& raw, int dtype, float (&v)[4]) {
    if (dtype == 2) {
        v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
        v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
    } else if (dtype == 1) {
        v[0] = __uint_as_float(raw.x << 16); v[1] = __uint_as_float(raw.x & 0xFFFF0000u);
        v[2] = __uint_as_float(raw.y << 16); v[3] = __uint_as_float(raw.y & 0xFFFF0000u);
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
}

// A TMA load of bytes that are read once: first to leave L2, so that code, scales
// and what CTAs share stay.  A whole MoE layer of 4 tokens (758 MB) takes 129.0 us
// with it and 137.3 without, of 32 tokens (400 MB) 127.5 and 129.7; one token's
// 25 MB, which L2 would keep from call to call, 20.8 and 20.4.
__device__ __forceinline__ void tma_load_2d_once(void* dst, const void* tmap, int c0, int c1, uint64_t* bar) {
    uint64_t pol;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
        :: "r"(smem_u32(dst)), "l"(tmap), "r"(c0), "r"(c1), "r"(smem_u32(bar)), "l"(pol) : "memory");
}

// A warp's share of quantising rows of x into a stage: four rows, eight lanes
// and 16 elements a lane each -- one chain of latencies for four rows -- or a
// lone row over all 32 lanes, where the shorter chain counts.
struct XRows {
    uint4 r[4];                  // a lane's elements as they lie in memory

    __device__ __forceinline__ static int row(int cnt, int lane) { return cnt == 1 ? 0 : lane >> 3; }
    __device__ __forceinline__ static int col(int cnt, int lane) { return cnt == 1 ? lane * 4 : (lane & 7) * 16; }

    // This lane's elements from element `at` on, those at or past `left` as zero.
    // vec: starts are aligned to 16 bytes (e4m3: four elements) and `left` is a
    // multiple of the lane's elements.
    __device__ __forceinline__ void load(int cnt, const void* x, int dtype, int64_t at, int left, bool vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = make_uint4(0u, 0u, 0u, 0u);
        if (left <= 0) return;
        const uint8_t* src = static_cast<const uint8_t*>(x) + at * (dtype == 2 ? 4 : dtype == kDtE4M3 ? 1 : 2);
        if (!vec) {
            const int n = cnt == 1 ? 1 : 4;
            uint4 t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = i < n ? load_raw4_tail(x, dtype, at + 4 * i, left - 4 * i) : make_uint4(0u, 0u, 0u, 0u);
            if (dtype == 2) {
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = t[i];
            } else if (dtype == kDtE4M3) {
                r[0] = make_uint4(t[0].x, t[1].x, t[2].x, t[3].x);
            } else {
                r[0] = make_uint4(t[0].x, t[0].y, t[1].x, t[1].y);
                r[1] = make_uint4(t[2].x, t[2].y, t[3].x, t[3].y);
            }
        } else if (cnt == 1) {
            if (dtype == 2) r[0] = *reinterpret_cast<const uint4*>(src);
            else if (dtype == kDtE4M3) r[0].x = *reinterpret_cast<const uint32_t*>(src);
            else {
                const uint2 h = *reinterpret_cast<const uint2*>(src);
                r[0].x = h.x; r[0].y = h.y;
            }
        } else {
            const uint4* v = reinterpret_cast<const uint4*>(src);
            r[0] = v[0];
            if (dtype != kDtE4M3) r[1] = v[1];
            if (dtype == 2) { r[2] = v[2]; r[3] = v[3]; }
        }
    }

    // The lane's elements in e4m3 (cnt == 1: the first word); `s`: their row's scale.
    __device__ __forceinline__ uint4 quantize(int cnt, int dtype, bool pow2, float& s) const {
        float v[16];
        if (dtype == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[4 * i] = __uint_as_float(r[i].x); v[4 * i + 1] = __uint_as_float(r[i].y);
                v[4 * i + 2] = __uint_as_float(r[i].z); v[4 * i + 3] = __uint_as_float(r[i].w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float t[4];
                unpack4(r[i], dtype, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[8 * i + j] = t[j];
                unpack4(make_uint4(r[i].z, r[i].w, 0u, 0u), dtype, t);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[8 * i + 4 + j] = t[j];
            }
        }
        uint32_t m = 0u;
        uint32_t q[4] = {0u, 0u, 0u, 0u};
        if (cnt == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max(m, abs_bits(v[i]));
            m = __reduce_max_sync(0xffffffffu, m);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, abs_bits(v[i]));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        }
        s = fp8_scale(m, pow2);
        const float inv = __frcp_rn(s);
        if (cnt == 1) {
            float t[4] = {v[0], v[1], v[2], v[3]};
            fp8_quotients(t, s, inv, pow2);
            q[0] = e4m3x2(t[0], t[1]) | (e4m3x2(t[2], t[3]) << 16);
            return make_uint4(q[0], 0u, 0u, 0u);
        }
        fp8_quotients(v, s, inv, pow2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = e4m3x2(v[4 * i], v[4 * i + 1]) | (e4m3x2(v[4 * i + 2], v[4 * i + 3]) << 16);
        }
        return make_uint4(q[0], q[1], q[2], q[3]);
    }

    // Into a K-major tile of 128-byte rows with the 128-byte swizzle, this lane's row being `row`.
    __device__ __forceinline__ static void store(int cnt, uint8_t* tile, int row, int lane, const uint4& q) {
        if (cnt == 1) *reinterpret_cast<uint32_t*>(tile + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = q.x;
        else *reinterpret_cast<uint4*>(tile + row * 128 + (((lane & 7) ^ (row & 7)) << 4)) = q;
    }
};

// ---------------------------------------------------------------- waits
// mbar_wait (2 s, then the ring-timeout bit) for pipelines whose steps take a
// fraction of a microsecond: the clock is read once in 256 polls only, because
// a read of %globaltimer takes about as long as such a step.
static __device__ __noinline__ bool poll_expired(uint64_t& t0) {
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    return t - t0 > kWaitLimitNs;
}

__device__ __forceinline__ bool mbar_poll(uint64_t* bar, uint32_t parity, uint32_t* status) {
    uint64_t t0 = 0;
    for (uint32_t i = 0; i < kSpinCap; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 255u && poll_expired(t0)) break;
    }
    set_error(status, ERR_RING_TIMEOUT);
    return false;
}

// Polled by every lane of a warp, with one verdict for the warp.
__device__ __forceinline__ bool mbar_poll_lanes(uint64_t* bar, uint32_t parity, uint32_t* status) {
    return __all_sync(0xffffffffu, mbar_poll(bar, parity, status));
}

// Two phases at once: both looks are in flight together, so that a loop whose
// barriers have completed pays for one of them.
__device__ __forceinline__ bool mbar_poll2_lanes(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint32_t* status) {
    const bool ra = mbar_try_wait(a, pa), rb = mbar_try_wait(b, pb);
    if (__all_sync(0xffffffffu, ra && rb)) return true;
    return mbar_poll_lanes(a, pa, status) && mbar_poll_lanes(b, pb, status);
}

// ---------------------------------------------------------------- tensor core
// The MMA loop runs in all lanes of its warp and one elected lane issues: the
// descriptors then stay in uniform registers.  Issued from inside `if (lane ==
// 0)`, four MMAs and two commits took 870 clocks, more than the MMAs
// themselves (256 x 256 x 32 each: 128 clocks).
__device__ __forceinline__ bool elect_lane() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}

// Warp index as the compiler sees it: the same in all lanes.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int) (threadIdx.x >> 5), 0); }

// D[128 x N] (+)= A . B^T of 8-bit operands, K = 32 per instruction, fp32
// accumulation; the instruction descriptor has the layout of kind::f16 with
// e4m3 as format 0.
__device__ __forceinline__ void tc_mma_f8(uint32_t dtmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(dtmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc) : "memory");
}

// The same over a pair of CTAs: each holds its half of A's rows (128 of 256)
// and its half of B's rows, and gets its rows of D.
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t dtmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(dtmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc) : "memory");
}

// Arrives on the barrier at this offset in both CTAs of the pair once the
// pair's MMAs issued so far have completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(smem_u32(bar)), "h"((uint16_t) 3) : "memory");
}

// TMA load into this CTA's shared memory whose bytes are counted on a barrier
// of either CTA of the pair (`bar`: an address of the cluster's window).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
        :: "r"(smem_u32(dst)), "l"(tmap), "r"(c0), "r"(c1), "r"(bar) : "memory");
}

// 32 lanes x 32-bit, 32 consecutive columns per thread: the load, which owns the
// registers until tc_ld_wait.
__device__ __forceinline__ void tc_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}

// Register split of a launch of 384 threads at 168 registers (64,512): two
// warpgroups raised to 232, one lowered to 40 -- 256 * 232 + 128 * 40 = 64,512.
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 232;"); }
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 40;"); }

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(smem_dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_free_pair(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(taddr), "r"(cols) : "memory");
}

__device__ __forceinline__ void tmap_prefetch(const void* tmap) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(tmap) : "memory");
}

// ---------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Address in the cluster's shared-memory window of `addr` (of this CTA's layout) in CTA `rank`.
__device__ __forceinline__ uint32_t mapa_u32(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}

// Arrival on a barrier of any CTA of the cluster.  It hands over TMEM columns
// that have been read into registers (tcgen05.fence::before_thread_sync comes
// before it) and no memory, so it has CTA scope: a release at cluster scope
// waits for every load in flight and was the largest stall of the pair kernel
// (2048 x 4096 x 4096: 107 us with it).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(addr) : "memory");
}

// fp32 / four fp32 at shared-memory address `addr` (of this CTA's layout) in CTA `rank` of the cluster.
__device__ __forceinline__ float ld_dsmem(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_u32(addr, rank)) : "memory");
    return v;
}

__device__ __forceinline__ float4 ld_dsmem4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_u32(addr, rank)) : "memory");
    return v;
}

// Tile of this CTA's shared memory -> global, asynchronously; what lies outside
// the tensor is not written.
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                 :: "l"(tmap), "r"(c0), "r"(c1), "r"(smem_u32(src)) : "memory");
}

__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// This thread's stores have read their source / are complete.
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Brings one tile into L2 ahead of the load that will use it.
__device__ __forceinline__ void tma_prefetch_2d(const void* tmap, int c0, int c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];"
                 :: "l"(tmap), "r"(c0), "r"(c1) : "memory");
}

}  // namespace exl3
