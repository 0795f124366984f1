// fp8_quant.cu -- e4m3 quantiser: one scale for each row and 128 columns
// (activations) or for each 128 x 128 block (weights).
//   s = max(max|x| / 448, 2^-126)   (pow2: the smallest power of two not below it)
//   q = RN_e4m3(x / s)
// Bound: memory, es + 1 bytes for each element (es = 2 or 4) plus the scales.
// Every value is loaded once, kept in registers while its group's maximum is
// taken over the lanes that hold it, and stored as e4m3.
#include "fp8.cuh"
#include "host.hpp"

namespace exl3 {

// A lane holds VEC = 16 bytes / es elements of one row; 128 / VEC lanes hold a
// group.  `fast`: rows start and end on VEC-element boundaries, so whole
// vectors are inside or outside; otherwise elements are moved one by one.
template <int DT>
struct QuantVec {
    static constexpr int VEC = DT == 2 ? 4 : 8;
    static constexpr int LANES = kFp8Block / VEC;          // 32 (fp32) or 16
    uint4 raw;
    __device__ __forceinline__ void load(const void* x, int64_t at, int left, bool fast) {
        raw = make_uint4(0u, 0u, 0u, 0u);
        if (left <= 0) return;
        if (fast) {
            raw = DT == 2 ? __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(x) + at))
                          : __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + at));
        } else if (DT == 2) {
            raw = load_raw4_tail(x, DT, at, left);
        } else {
            const uint4 a = load_raw4_tail(x, DT, at, left), b = load_raw4_tail(x, DT, at + 4, left - 4);
            raw = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
    __device__ __forceinline__ void get(int half, float (&v)[4]) const {
        unpack4(DT == 2 ? raw : half ? make_uint4(raw.z, raw.w, 0u, 0u) : raw, DT, v);
    }
    __device__ __forceinline__ uint32_t amax() const {
        float v[4];
        get(0, v);
        uint32_t m = abs_bits4(v);
        if (DT != 2) {
            get(1, v);
            m = max(m, abs_bits4(v));
        }
        return m;
    }
    __device__ __forceinline__ void store(uint8_t* q, int64_t at, int left, bool fast, float s, float inv, bool pow2) const {
        if (left <= 0) return;
        float v[4];
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int h = 0; h < VEC / 4; ++h) {
            get(h, v);
            w[h] = fp8_quant4(v, s, inv, pow2);
        }
        if (fast) {
            if (DT == 2) *reinterpret_cast<uint32_t*>(q + at) = w[0];
            else *reinterpret_cast<uint2*>(q + at) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e < left) q[at + e] = (uint8_t) (w[e >> 2] >> (8 * (e & 3)));
        }
    }
};

constexpr int kQuantWarps = 8;
constexpr int kQuantIlp = 4;        // 16-byte loads in flight for each lane

// One scale for each row and group of 128 columns.  An item is a row's 32-lane
// span: one group (fp32) or two neighbours (16-bit); a warp takes kQuantIlp
// consecutive items, all loads first.
template <int DT>
__global__ void __launch_bounds__(kQuantWarps * 32) fp8_quant_rows_kernel(
    const void* x, int64_t ldx, int64_t rows, int cols, uint8_t* q, int64_t ldq, float* scale, int64_t sr, int64_t sg, bool pow2, bool fast) {
    using V = QuantVec<DT>;
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int groups = (cols + kFp8Block - 1) / kFp8Block;
    constexpr int GP = 32 / V::LANES;                      // groups in an item
    const int per_row = (groups + GP - 1) / GP;
    const int64_t items = rows * per_row;
    const int64_t first = ((int64_t) blockIdx.x * kQuantWarps + (threadIdx.x >> 5)) * kQuantIlp;
    if (first >= items) return;
    V v[kQuantIlp];
    int64_t row[kQuantIlp];
    int col[kQuantIlp];
    row[0] = first / per_row;
    int in_row = (int) (first - row[0] * per_row);
    int64_t r = row[0];
#pragma unroll
    for (int i = 0; i < kQuantIlp; ++i) {
        row[i] = first + i < items ? r : -1;
        col[i] = in_row * GP * kFp8Block + lane * V::VEC;
        v[i].load(x, r * ldx + col[i], row[i] < 0 ? 0 : cols - col[i], fast);
        if (++in_row == per_row) { in_row = 0; ++r; }
    }
#pragma unroll
    for (int i = 0; i < kQuantIlp; ++i) {
        if (row[i] < 0) return;
        uint32_t m = v[i].amax();
#pragma unroll
        for (int o = 1; o < V::LANES; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float s = fp8_scale(m, pow2), inv = __frcp_rn(s);
        v[i].store(q, row[i] * ldq + col[i], cols - col[i], fast, s, inv, pow2);
        if ((lane & (V::LANES - 1)) == 0 && col[i] < cols) scale[row[i] * sr + col[i] / kFp8Block * sg] = s;
    }
}

// One scale for each 128 x 128 block: a CTA of 256 threads holds the block in
// registers (32 of them for 16-bit types, 64 for fp32).
template <int DT>
__global__ void __launch_bounds__(256) fp8_quant_blocks_kernel(
    const void* x, int64_t ldx, int64_t rows, int cols, uint8_t* q, int64_t ldq, float* scale, bool pow2, bool fast) {
    using V = QuantVec<DT>;
    constexpr int RP = 256 / V::LANES;                     // rows in a pass
    constexpr int N = kFp8Block / RP;                      // passes
    __shared__ uint32_t wmax[8];
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t) blockIdx.y * kFp8Block + tid / V::LANES;
    const int col = blockIdx.x * kFp8Block + (tid % V::LANES) * V::VEC;
    V v[N];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t r = row0 + i * RP;
        v[i].load(x, r * ldx + col, r < rows ? cols - col : 0, fast);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, v[i].amax());
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) wmax[tid >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, wmax[w]);
    const float s = fp8_scale(m, pow2), inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int64_t r = row0 + i * RP;
        v[i].store(q, r * ldq + col, r < rows ? cols - col : 0, fast, s, inv, pow2);
    }
    if (tid == 0) scale[(int64_t) blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// Arguments are checked by the callers.  rows >= 1, cols in 1..2^30.  Rows'
// scales lie at scale[row * sr + group * sg].
int fp8_quantize_launch(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx, void* q, int64_t ldq,
                        float* scale, int64_t sr, int64_t sg, int block_rows, bool pow2, cudaStream_t s) {
    const int es = dtype == 2 ? 4 : 2, vec = 16 / es;
    const bool fast = cols % vec == 0 && ldx % vec == 0 && ldq % vec == 0 && aligned16(x) &&
                      (reinterpret_cast<uintptr_t>(q) % (uintptr_t) vec) == 0;
    const int64_t groups = (cols + kFp8Block - 1) / kFp8Block;
    uint8_t* qb = static_cast<uint8_t*>(q);
    if (block_rows == 1) {
        const int64_t per_row = dtype == 2 ? groups : (groups + 1) / 2;
        const int64_t grid = (rows * per_row + kQuantWarps * kQuantIlp - 1) / (kQuantWarps * kQuantIlp);
        EXL3_REQUIRE(grid <= INT32_MAX, EXL3_ERR_UNSUPPORTED, "exl3_fp8_quantize: too many elements for one launch");
        auto kern = dtype == 0 ? fp8_quant_rows_kernel<0> : dtype == 1 ? fp8_quant_rows_kernel<1> : fp8_quant_rows_kernel<2>;
        kern<<<(unsigned) grid, kQuantWarps * 32, 0, s>>>(x, ldx, rows, (int) cols, qb, ldq, scale, sr, sg, pow2, fast);
    } else {
        const int64_t rb = (rows + kFp8Block - 1) / kFp8Block;
        EXL3_REQUIRE(rb <= 65535, EXL3_ERR_UNSUPPORTED, "exl3_fp8_quantize: more than 65535 blocks of 128 rows");
        auto kern = dtype == 0 ? fp8_quant_blocks_kernel<0> : dtype == 1 ? fp8_quant_blocks_kernel<1> : fp8_quant_blocks_kernel<2>;
        kern<<<dim3((unsigned) groups, (unsigned) rb), 256, 0, s>>>(x, ldx, rows, (int) cols, qb, ldq, scale, pow2, fast);
    }
    EXL3_CUDA(cudaGetLastError());
    return EXL3_OK;
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
