// fp8_quant.cu -- e4m3 quantiser: one scale for each row and 128 columns
// (activations) or for each 128 x 128 block (weights).
//   s = max(max|x| / 448, 2^-126)   (pow2: the smallest power of two not below it)
//   q = RN_e4m3(x / s)
// Bound: memory, es + 1 bytes for each element (es = 2 or 4) plus the scales.
// Every value is loaded once, kept in registers while its group's maximum is
// taken over the lanes that hold it, and stored as e4m3.  8192 x 4096 bf16 with
// powers of two takes 14 us in a graph (102 MB at the copy rate; 20.6 us with exact
// quotients, bound by instructions), 4000 x 4080 in
// blocks 11.2 us (4.4 TB/s: a block is loaded, reduced and stored in turn).
#include "fp8.cuh"
#include "host.hpp"

namespace exl3 {

// A lane holds VEC = 32 bytes / es elements of one row; 128 / VEC lanes hold a
// group.  (With 16 bytes a lane the scale, its reciprocal and the addresses cost
// as much as the values: 15 instructions a value with power-of-two scales.)
// FAST 2: rows start and end on VEC-element boundaries, so whole vectors are
// inside or outside; 1: the same for half vectors; 0: elements are moved one by one.
template <int DT, int FAST>
struct QuantVec {
    static constexpr int VEC = DT == 2 ? 8 : 16;
    static constexpr int LANES = kFp8Block / VEC;          // 16 (fp32) or 8
    uint32_t w[8];
    __device__ __forceinline__ void load(const void* x, int64_t at, int left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0u;
        if (left <= 0) return;
        if constexpr (FAST != 0) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + at * (DT == 2 ? 4 : 2));
            const uint4 a = __ldcs(src), b = FAST == 2 || left > VEC / 2 ? __ldcs(src + 1) : make_uint4(0u, 0u, 0u, 0u);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        } else {
            constexpr int PER = DT == 2 ? 4 : 2;           // words of four elements
#pragma unroll
            for (int i = 0; i < VEC / 4; ++i) {
                const uint4 t = load_raw4_tail(x, DT, at + 4 * i, left - 4 * i);
                w[PER * i] = t.x;
                w[PER * i + 1] = t.y;
                if constexpr (DT == 2) {
                    w[PER * i + 2] = t.z;
                    w[PER * i + 3] = t.w;
                }
            }
        }
    }
    // Bits of the largest magnitude as fp32, NaN kept; 16-bit types two at a time.
    __device__ __forceinline__ uint32_t amax() const {
        if constexpr (DT == 2) {
            uint32_t m = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            uint32_t a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = w[i] & 0x7FFF7FFFu;
            float2 f;
            if constexpr (DT == 1) {
                auto h = [&](int i) { return *reinterpret_cast<const __nv_bfloat162*>(&a[i]); };
                auto m = [&](int i) { return __hmax2_nan(h(i), h(i + 1)); };
                f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(m(0), m(2)), __hmax2_nan(m(4), m(6))));
            } else {
                auto h = [&](int i) { return *reinterpret_cast<const __half2*>(&a[i]); };
                auto m = [&](int i) { return __hmax2_nan(h(i), h(i + 1)); };
                f = __half22float2(__hmax2_nan(__hmax2_nan(m(0), m(2)), __hmax2_nan(m(4), m(6))));
            }
            return max(abs_bits(f.x), abs_bits(f.y));
        }
    }
    template <bool POW2>
    __device__ __forceinline__ void store(uint8_t* q, int64_t at, int left, float s) const {
        if (left <= 0) return;
        const float inv = __frcp_rn(s);
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) {
            float t[4];
            if constexpr (DT == 2) unpack4(make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]), DT, t);
            else unpack4(make_uint4(w[2 * i], w[2 * i + 1], 0u, 0u), DT, t);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = t[j];
        }
        fp8_quotients(v, s, inv, POW2);
        uint32_t o[VEC / 4];
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
            o[i] = e4m3x2(v[4 * i], v[4 * i + 1]) | (e4m3x2(v[4 * i + 2], v[4 * i + 3]) << 16);
        if constexpr (FAST == 2) {
            if constexpr (DT == 2) *reinterpret_cast<uint2*>(q + at) = make_uint2(o[0], o[1]);
            else *reinterpret_cast<uint4*>(q + at) = make_uint4(o[0], o[1], o[2], o[3]);
        } else if constexpr (FAST == 1) {
            if constexpr (DT == 2) {
                *reinterpret_cast<uint32_t*>(q + at) = o[0];
                if (left > VEC / 2) *reinterpret_cast<uint32_t*>(q + at + 4) = o[1];
            } else {
                *reinterpret_cast<uint2*>(q + at) = make_uint2(o[0], o[1]);
                if (left > VEC / 2) *reinterpret_cast<uint2*>(q + at + 8) = make_uint2(o[2], o[3]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < left) q[at + e] = (uint8_t) (o[e >> 2] >> (8 * (e & 3)));
        }
    }
};

constexpr int kQuantWarps = 4;         // 8192 x 4096, powers of two: 14.5 us with 4 warps a CTA, 17.3 with 8

struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scale;                // scale[row * sr + group * sg]; blocks: [row block][group]
    int64_t ldx, ldq, sr, sg, rows;
    int cols, groups, spans;     // spans: 32-lane pieces of a row
};

// One scale for each row and group of 128 columns.  A warp takes one span of a
// row -- two neighbouring groups (fp32) or four (16-bit) -- in RP consecutive
// rows, all loads first.
template <int DT, bool POW2, int FAST, int RP>
__global__ void __launch_bounds__(kQuantWarps * 32) fp8_quant_rows_kernel(const __grid_constant__ QuantArgs p) {
    using V = QuantVec<DT, FAST>;
    // Whoever starts early behind this kernel finds all that came before it complete.
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const uint32_t item = blockIdx.x * kQuantWarps + (threadIdx.x >> 5);
    const int64_t row0 = (int64_t) (item / (uint32_t) p.spans) * RP;
    const int col = (int) (item % (uint32_t) p.spans) * (32 * V::VEC) + lane * V::VEC, left = p.cols - col;
    if (row0 >= p.rows) return;
    const int n = p.rows - row0 < RP ? (int) (p.rows - row0) : RP;
    V v[RP];
#pragma unroll
    for (int i = 0; i < RP; ++i) v[i].load(p.x, (row0 + i) * p.ldx + col, i < n ? left : 0);
#pragma unroll
    for (int i = 0; i < RP; ++i) {
        uint32_t m = v[i].amax();
#pragma unroll
        for (int o = 1; o < V::LANES; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (i >= n) break;
        const float s = fp8_scale(m, POW2);
        v[i].template store<POW2>(p.q, (row0 + i) * p.ldq + col, left, s);
        if ((lane & (V::LANES - 1)) == 0 && left > 0) p.scale[(row0 + i) * p.sr + col / kFp8Block * p.sg] = s;
    }
}

// One scale for each 128 x 128 block, held in registers: 512 threads of two
// 32-byte pieces (16-bit types) or four (fp32).
template <int DT, bool POW2, int FAST>
__global__ void __launch_bounds__(512) fp8_quant_blocks_kernel(const __grid_constant__ QuantArgs p) {
    using V = QuantVec<DT, FAST>;
    constexpr int RP = 512 / V::LANES;                     // rows in a pass
    constexpr int N = kFp8Block / RP;                      // passes
    __shared__ uint32_t wmax[16];
    pdl_wait();
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t) blockIdx.y * kFp8Block + tid / V::LANES;
    const int col = blockIdx.x * kFp8Block + (tid % V::LANES) * V::VEC, left = p.cols - col;
    V v[N];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i].load(p.x, (row0 + i * RP) * p.ldx + col, row0 + i * RP < p.rows ? left : 0);
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, v[i].amax());
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) wmax[tid >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, wmax[tid & 15]);
    const float s = fp8_scale(m, POW2);
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i].template store<POW2>(p.q, (row0 + i * RP) * p.ldq + col, row0 + i * RP < p.rows ? left : 0, s);
    if (tid == 0) p.scale[(int64_t) blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// Programmatic launch: the grid is set up while the previous kernel ends.
int quant_pdl(void (*kern)(QuantArgs), dim3 grid, int threads, const QuantArgs& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned) threads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    EXL3_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
    return EXL3_OK;
}

template <int DT, bool POW2, int FAST>
int quant_launch(QuantArgs& a, int block_rows, cudaStream_t s) {
    if (block_rows == 1) {
        a.spans = DT == 2 ? (a.groups + 1) / 2 : (a.groups + 3) / 4;
        // Four rows a warp keep 4 KB a warp in flight (8192 rows x 4096: 14.5 us,
        // with one row 18.6); below some 32768 spans the other way round, since the
        // grid is a few waves then (1024 rows: 5.2 us with four, 4.4 with one).
        const int rp = a.rows * a.spans < 32768 ? 1 : 4;
        const int64_t items = (a.rows + rp - 1) / rp * a.spans, grid = (items + kQuantWarps - 1) / kQuantWarps;
        EXL3_REQUIRE(items <= INT32_MAX, EXL3_ERR_UNSUPPORTED, "exl3_fp8_quantize: too many elements for one launch");
        return quant_pdl(rp == 1 ? fp8_quant_rows_kernel<DT, POW2, FAST, 1> : fp8_quant_rows_kernel<DT, POW2, FAST, 4>,
                         dim3((unsigned) grid), kQuantWarps * 32, a, s);
    }
    const int64_t rb = (a.rows + kFp8Block - 1) / kFp8Block;
    EXL3_REQUIRE(rb <= 65535, EXL3_ERR_UNSUPPORTED, "exl3_fp8_quantize: more than 65535 blocks of 128 rows");
    return quant_pdl(fp8_quant_blocks_kernel<DT, POW2, FAST>, dim3((unsigned) a.groups, (unsigned) rb), 512, a, s);
}

template <int DT, bool POW2>
int quant_dispatch(QuantArgs& a, int block_rows, int fast, cudaStream_t s) {
    return fast == 2 ? quant_launch<DT, POW2, 2>(a, block_rows, s) : fast == 1 ? quant_launch<DT, POW2, 1>(a, block_rows, s)
                                                                              : quant_launch<DT, POW2, 0>(a, block_rows, s);
}

// Arguments are checked by the callers.  rows >= 1, cols in 1..2^30.  Rows'
// scales lie at scale[row * sr + group * sg].
int fp8_quantize_launch(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq,
                        float* scale, int64_t sr, int64_t sg, int block_rows, bool pow2, cudaStream_t s) {
    const int half = dtype == 2 ? 4 : 8;                   // elements of 16 bytes
    auto on = [&](int n) { return cols % n == 0 && ldx % half == 0 && ldq % n == 0 && aligned16(x) && reinterpret_cast<uintptr_t>(q) % (uintptr_t) n == 0; };
    const int fast = on(2 * half) ? 2 : on(half) ? 1 : 0;
    QuantArgs a{x, static_cast<uint8_t*>(q), scale, ldx, ldq, sr, sg, rows, (int) cols, (int) ((cols + kFp8Block - 1) / kFp8Block), 0};
    if (dtype == 0) return pow2 ? quant_dispatch<0, true>(a, block_rows, fast, s) : quant_dispatch<0, false>(a, block_rows, fast, s);
    if (dtype == 1) return pow2 ? quant_dispatch<1, true>(a, block_rows, fast, s) : quant_dispatch<1, false>(a, block_rows, fast, s);
    return pow2 ? quant_dispatch<2, true>(a, block_rows, fast, s) : quant_dispatch<2, false>(a, block_rows, fast, s);
}

}  // namespace exl3

extern "C" int exl3_fp8_quantize(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, void* q,
                                 int64_t ldq, float* scale, int block_rows, int pow2, void* stream) {
    using namespace exl3;
    EXL3_REQUIRE(rows >= 0 && cols >= 1 && cols <= INT32_MAX / 2, EXL3_ERR_ARG,
                 "exl3_fp8_quantize: rows must be >= 0 and cols in 1..2^30");
    EXL3_REQUIRE(x_dtype >= 0 && x_dtype <= 2, EXL3_ERR_ARG, "exl3_fp8_quantize: dtype must be fp16, bf16 or fp32");
    EXL3_REQUIRE(block_rows == 1 || block_rows == kFp8Block, EXL3_ERR_ARG, "exl3_fp8_quantize: block_rows must be 1 or 128");
    EXL3_REQUIRE(ldx >= cols && ldq >= cols, EXL3_ERR_ARG, "exl3_fp8_quantize: leading dimensions must be >= cols");
    if (rows == 0) return EXL3_OK;
    EXL3_REQUIRE(x && q && scale, EXL3_ERR_ARG, "exl3_fp8_quantize: null pointer");
    EXL3_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == 2 ? 4 : 2) == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0,
                 EXL3_ERR_ARG, "exl3_fp8_quantize: x and scale must be aligned to their elements");
    return fp8_quantize_launch(x, x_dtype, rows, cols, ldx, q, ldq, scale, (cols + 127) / 128, 1, block_rows, pow2 != 0,
                               static_cast<cudaStream_t>(stream));
}
