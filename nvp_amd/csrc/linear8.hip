// Linear layer on 8-bit floating point with one power-of-two scale per block of 128:
//     y[m][n] = sum_b 2^(sx[m][b] + sw[n / 128][b]) * sum_{k in block b} qx[m][k] qw[n][k]  (+ bias[n])
// q = e4m3(v * 2^-s), s = the smallest power with max|v| <= 448 * 2^s over the block (one row x 128 columns of x, 128 x 128 of w), kept as the
// byte s + 127.  A power of two costs a floating-point operand no precision, makes the quantised value exact to state (no rounding in the
// scale or in v * 2^-s) and is what the matrix instruction multiplies with by itself (v_mfma_scale_f32_*_f8f6f4 takes one exponent byte per
// row and 32 columns): the block scales cost no vector instruction.
//
// Which matrix instruction.  The 8-bit ones add their products to a 32-bit accumulator, but inside each group of 8 products they drop what lies
// more than 13 bits below the largest product's exponent (measured: 2^3 beside 2^16 is kept, 2^2 is not, in one group; across groups nothing is
// lost; normal data: 1.5e-5 of the result's rms, whatever K).  That is an order of magnitude below the rounding of a 16-bit y (bf16 1.7e-3,
// fp16 2e-4 rms), so 16-bit streams take them.  A 32-bit y would show it: fp32 streams widen both operands to bf16 in registers - exact, the
// scale goes into the exponent (v_cvt_scalef32_pk_bf16_fp8) - and use the bf16 instructions, whose sums are fp32 throughout (2e-7), at half the rate.
#include <type_traits>
#include "stream_types.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t kblocks(int64_t k) { return (k + 127) / 128; }
__host__ __device__ inline int64_t kb4(int64_t k) { return (kblocks(k) + 3) / 4 * 4; }       // a row's scale bytes, padded to whole dwords

// exponent byte of a block from the bit pattern of its largest finite |v|: 448 = 1.75 * 2^8
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
    if (amax_bits == 0u) return 127u;
    const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)max(e, 0);
}
// 2^-(byte - 127); bytes of scale_byte() are at most 247, so the result is a normal number
__device__ __forceinline__ float inv_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ unsigned finite_bits(float v) {                                  // |v|, 0 for infinities and NaN
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
// four values -> four e4m3 bytes, round to nearest even; |v * inv| <= 448, so nothing saturates; infinities and NaN become NaN (0x7f)
__device__ __forceinline__ int quant4(const float* v, float inv) {
    int p = 0;
    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, p, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, p, true);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if ((__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u) p = (p & ~(0xff << (8 * e))) | (0x7f << (8 * e));
    return p;
}

// maximum over 16 neighbouring lanes, in every lane: rotations within the row of 16, no LDS
__device__ __forceinline__ unsigned max16(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));    // row_ror:8
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
}
// one row's block of 128, 8 values in each of 16 neighbouring lanes -> 8 bytes per lane and the block's scale byte
__device__ __forceinline__ int2 quant8(const float (&v)[8], unsigned& byte) {
    unsigned top = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    top = max16(top);
    int2 q;
    if (!__any(top >= 0x7f800000u)) {
        byte = scale_byte(top);
        const float inv = inv_scale(byte);
        q.x = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false), true);
        q.y = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false), true);
        return q;
    }
    top = 0u;                                                                                // an infinity or a NaN among the wave's blocks: the careful way
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, finite_bits(v[e]));
    byte = scale_byte(max16(top));
    const float inv = inv_scale(byte);
    q.x = quant4(v, inv);
    q.y = quant4(v + 4, inv);
    return q;
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// one lane's 32 operand bytes of a matrix instruction and their block's scale byte; WIDE: widened to 4 x 8 bf16, scale applied
template <bool WIDE> struct frag;
template <> struct frag<false> {
    v8i q;
    int s;
    __device__ __forceinline__ void set(v8i raw, int byte) { q = raw; s = byte; }
};
template <> struct frag<true> {
    bf16x8 h[4];
    __device__ __forceinline__ void set(v8i raw, int byte) {
        const float f = __uint_as_float((unsigned)(byte & 0xff) << 23);                      // only the exponent field counts: byte 0 is 2^-127
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[p], f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[p], f, true);
            h[p >> 1][4 * (p & 1) + 0] = lo[0];
            h[p >> 1][4 * (p & 1) + 1] = lo[1];
            h[p >> 1][4 * (p & 1) + 2] = hi[0];
            h[p >> 1][4 * (p & 1) + 3] = hi[1];
        }
    }
};
// c += a b^T over 128 (16 x 16 tile) or 64 (32 x 32 tile) values of k.  Which k a register byte stands for is the same in a and b and cancels.
__device__ __forceinline__ f32x4 mma(const frag<false>& a, const frag<false>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.q, b.q, c, 0, 0, 0, a.s, 0, b.s);
}
__device__ __forceinline__ f32x16 mma(const frag<false>& a, const frag<false>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.q, b.q, c, 0, 0, 0, a.s, 0, b.s);
}
__device__ __forceinline__ f32x4 mma(const frag<true>& a, const frag<true>& b, f32x4 c) {
#pragma unroll
    for (int p = 0; p < 4; ++p) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h[p], b.h[p], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x16 mma(const frag<true>& a, const frag<true>& b, f32x16 c) {
#pragma unroll
    for (int p = 0; p < 4; ++p) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h[p], b.h[p], c, 0, 0, 0);
    return c;
}

// two tiles against one operand, their chains interleaved
template <bool W> __device__ __forceinline__ void mma2(const frag<W>& a0, const frag<W>& a1, const frag<W>& b, f32x4& c0, f32x4& c1) {
    if constexpr (W) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            c0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0.h[p], b.h[p], c0, 0, 0, 0);
            c1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1.h[p], b.h[p], c1, 0, 0, 0);
        }
    } else {
        c0 = mma(a0, b, c0);
        c1 = mma(a1, b, c1);
    }
}

// ---- x -> workspace: 16 lanes per block of 128, 8 values each -----------------------------------------------------------------------------
// q: groups of 8 rows, a block's 8 x 128 bytes in one piece ([rows / 8][KB][8][128]: what one load instruction of the tile kernel fetches, 50 bytes per
// clock and CU against 40 for 8 pieces of 128 and 30 for 16 of 64); scales [rows][KB4] (bytes); the launch's last workgroups copy the weights' scales to
// dword-padded rows [NB][KB4].
__host__ __device__ inline int64_t xq_at(int64_t row, int64_t b, int64_t kb) { return ((row >> 3) * kb + b) * 1024 + (row & 7) * 128; }
__host__ __device__ inline int64_t xq_bytes(int64_t rows, int64_t kb) { return (rows + 7) / 8 * kb * 1024; }
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ ex, int64_t rows, int64_t k,
                                                         int64_t x_groups, const uint8_t* __restrict__ ew, uint8_t* __restrict__ ew_pad, int64_t ew_bytes) {
    const int64_t kb = kblocks(k), kb_pad = kb4(k);
    const int lane16 = threadIdx.x & 15;
    if ((int64_t)blockIdx.x >= x_groups) {
        const int64_t i = ((int64_t)blockIdx.x - x_groups) * 256 + threadIdx.x;
        if (i < ew_bytes) {
            const int64_t r = i / kb_pad, b = i - r * kb_pad;
            ew_pad[i] = b < kb ? ew[r * kb + b] : 127;
        }
        return;
    }
    const int64_t g = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);                         // block number: row * KB + b
    if (g >= rows * kb) return;                                                              // whole 16-lane groups leave together
    const int64_t row = g / kb, b = g - row * kb, c0 = b * 128 + lane16 * 8;
    float v[8];
    if (c0 + 8 <= k) {
        nvp_load<T, 8>(x + row * k + c0, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c0 + e < k ? (float)x[row * k + c0 + e] : 0.f;
    }
    unsigned byte;
    const int2 p = quant8(v, byte);
    *reinterpret_cast<int2*>(q + xq_at(row, b, kb) + lane16 * 8) = p;
    if (lane16 == 0) ex[row * kb_pad + b] = (uint8_t)byte;
}

// ---- weights: one workgroup per block of block_rows x 128 (not a hot path: once per set of weights) ----------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void quant_blocks_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint8_t* __restrict__ e, int64_t rows, int64_t k, int block_rows) {
    const int64_t kb = kblocks(k);
    const int64_t rb = (int64_t)blockIdx.x / kb, b = (int64_t)blockIdx.x - rb * kb;
    const int c = threadIdx.x & 127, r0 = threadIdx.x >> 7;
    const int64_t col = b * 128 + c;
    unsigned top = 0u;
    for (int r = r0; r < block_rows; r += 2) {
        const int64_t row = rb * block_rows + r;
        if (row < rows && col < k) top = max(top, finite_bits((float)x[row * k + col]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    __shared__ unsigned red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    const unsigned byte = scale_byte(max(max(red[0], red[1]), max(red[2], red[3])));
    const float inv = inv_scale(byte);
    for (int r = r0; r < block_rows; r += 2) {
        const int64_t row = rb * block_rows + r;
        if (row >= rows) break;
        const float v[4] = {col < k ? (float)x[row * k + col] : 0.f, 0.f, 0.f, 0.f};
        q[row * kb * 128 + col] = (uint8_t)(quant4(v, inv) & 0xff);
    }
    if (threadIdx.x == 0) e[rb * kb + b] = (uint8_t)byte;
}

template <typename T>
__global__ __launch_bounds__(256) void dequant_blocks_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, T* __restrict__ x, int64_t rows, int64_t k, int block_rows) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * k) return;
    const int64_t row = i / k, col = i - row * k, kb = kblocks(k);
    const float v = __builtin_amdgcn_cvt_f32_fp8((int)q[row * kb * 128 + col], 0);
    const unsigned byte = e[row / block_rows * kb + col / 128];
    // 2^(byte - 127) in two factors: byte 0 is 2^-127, below the smallest normal number
    const float s = byte == 255u ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
    x[i] = (T)(v * s);
}

// ---- few rows: every wave walks its share of K with the weights straight from global memory -------------------------------------------------
// One workgroup: 16 MT rows x 16 NT columns; its WAVES waves take every WAVES-th block of 128 and add their tiles up through LDS, so a single row
// times 4096 columns is 256 workgroups x 8 waves that read disjoint weights: bound by the bytes of the weights, which are on their way (kAhead blocks)
// before anything else happens.  FUSED: the workgroup quantises its rows of x into LDS itself - no workspace, no second launch; each workgroup repeats
// that, which pays while there are few workgroups or few rows.  1 x 4096 x 4096 bf16: 5.6 us (16.8 MB, 3 TB/s: one round of loads, whose latency is most of
// it); 32 x 4096 x 4096: 2.2 us for the quantising launch and 10.1: the same round of weight loads, x's rows from L2 behind it (the waves wait 74 % of their life).
// Operand order: lane (i = lane & 15, g = lane >> 4) holds columns 16 g .. 16 g + 15 and 64 + 16 g .. of its row's block, the same for both
// operands: which k a register byte stands for cancels in the sum, and each load instruction covers 64 contiguous bytes of a row.
constexpr int rows_ahead(int mt, int nt) { return mt * nt >= 4 ? 2 : 4; }
template <typename T, int MT, int NT, int WAVES, bool FUSED>
__global__ __launch_bounds__(64 * WAVES) void linear8_rows_kernel(const T* __restrict__ x, const uint8_t* __restrict__ qx, const uint8_t* __restrict__ ex, const uint8_t* __restrict__ qw,
                                                                  const uint8_t* __restrict__ ew, const T* __restrict__ bias, T* __restrict__ y, int64_t rows, int64_t k, int64_t n) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];                           // FUSED: rows of kp + 16 bytes, then their scale bytes; later the partial tiles
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int kAhead = rows_ahead(MT, NT);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int64_t kb = kblocks(k), kp = kb * 128, kbp = kb4(k);
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int mrows = (int)min((int64_t)(16 * MT), rows - m0);
    const uint8_t* wrow[NT];
    const uint8_t* wexp[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int64_t nn = min(n0 + 16 * b + i, n - 1);                                      // rows behind the last one read the last one: their results are not stored
        wrow[b] = qw + nn * kp + 16 * g;
        wexp[b] = ew + nn / 128 * (FUSED ? kb : kbp);
    }
    v8i wr[kAhead][NT];
    int we[kAhead][NT];
    const auto fetch = [&](int64_t b0) {                                                     // (blocks behind the last one read the last one again)
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int64_t bq = min(b0 + WAVES * q, kb - 1);
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const v4i lo = *reinterpret_cast<const v4i*>(wrow[b] + bq * 128), hi = *reinterpret_cast<const v4i*>(wrow[b] + bq * 128 + 64);
                wr[q][b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                we[q][b] = wexp[b][bq];
            }
        }
    };
    fetch(wave);
    const int64_t xs = kp + 16;                                                              // row stride in LDS: 16 rows x 16 bytes fall on different banks
    uint8_t* const xe = lds + mrows * xs;
    if (FUSED) {
        const int l16 = threadIdx.x & 15, tasks = mrows * (int)kb;
        constexpr int kTasks = 2;                                                            // blocks per 16 lanes and round, their loads in front
        for (int t0 = threadIdx.x >> 4; t0 < tasks; t0 += 4 * WAVES * kTasks) {              // 16 lanes per block of 128, 8 values each
            nvp_vec<T, 8> raw[kTasks];
            int at[kTasks];
#pragma unroll
            for (int u = 0; u < kTasks; ++u) {
                const int t = min(t0 + u * 4 * WAVES, tasks - 1), r = t / (int)kb, b = t - r * (int)kb;
                const int c0 = b * 128 + l16 * 8;
                at[u] = r * (int)xs + c0;
                const T* p = x + (m0 + r) * k + c0;
                if (c0 + 8 <= k) {
                    raw[u] = nvp_load_raw<T, 8>(p);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) raw[u].v[e] = c0 + e < k ? p[e] : (T)0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < kTasks; ++u) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (float)raw[u].v[e];
                unsigned byte;
                const int2 q = quant8(v, byte);
                const int t = t0 + u * 4 * WAVES;
                if (t < tasks) {
                    *reinterpret_cast<int2*>(lds + at[u]) = q;
                    if (l16 == 0) xe[t] = (uint8_t)byte;
                }
            }
        }
        __syncthreads();
    }
    f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int64_t b0 = wave; b0 < kb; b0 += WAVES * kAhead) {
        v8i xr[kAhead][MT];
        int xb[kAhead][MT];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int64_t bq = min(b0 + WAVES * q, kb - 1);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                const int64_t r = min(16 * a + i, mrows - 1);
                const uint8_t* p = (FUSED ? lds + r * xs + bq * 128 : qx + xq_at(m0 + r, bq, kb)) + 16 * g;
                const v4i lo = *reinterpret_cast<const v4i*>(p), hi = *reinterpret_cast<const v4i*>(p + 64);
                xr[q][a] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                xb[q][a] = FUSED ? xe[r * kb + bq] : ex[(m0 + r) * kbp + bq];
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            if (b0 + WAVES * q >= kb) break;
            frag<kWide> wf[NT];
#pragma unroll
            for (int b = 0; b < NT; ++b) wf[b].set(wr[q][b], we[q][b]);
#pragma unroll
            for (int a = 0; a < MT; ++a) {
                frag<kWide> xf;
                xf.set(xr[q][a], xb[q][a]);
#pragma unroll
                for (int b = 0; b < NT; ++b) acc[a][b] = mma(xf, wf[b], acc[a][b]);
            }
        }
        if (b0 + WAVES * kAhead < kb) fetch(b0 + WAVES * kAhead);
    }
    // D: row 4 (lane >> 4) + r, column lane & 15
    constexpr int kStride = NT * 16 + 1;
    float* const part = reinterpret_cast<float*>(lds);
    if (FUSED) __syncthreads();                                                              // every wave has read its x
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) part[(wave * MT * 16 + 16 * a + 4 * g + r) * kStride + 16 * b + i] = acc[a][b][r];
    __syncthreads();
    for (int t = threadIdx.x; t < MT * 16 * NT * 16; t += 64 * WAVES) {
        const int r = t / (NT * 16), c = t % (NT * 16);
        if (r >= mrows || n0 + c >= n) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += part[(w * MT * 16 + r) * kStride + c];
        if (bias) s += (float)bias[n0 + c];
        y[(m0 + r) * n + n0 + c] = (T)s;
    }
}

// ---- many rows, few columns: x quantised on the way, weights resident in LDS ---------------------------------------------------------------
// With up to 256 columns the product is bound by the bytes of x and y, and quantising x in a pass of its own would move a quarter more: here a wave
// takes 16 rows at a time, block by block: 16-byte loads (four lanes cover 64 contiguous bytes of a row) one block ahead, the block's maximum by two
// shuffles, and the quantised block is the matrix instruction's operand right away.  The weights (all columns, all of K) stay in LDS, with the bytes of a
// block in the order in which the lanes hold x's columns and the 16-byte pieces of a row swizzled by the row, so that operand reads are free of bank conflicts.
// Weights are the first operand: a lane then holds four consecutive columns of one row of y.
// 1 245 184 x 242 -> 128 columns, fp32: 380 - 394 us (1.84 GB, 4.7 - 4.85 TB/s: the rate of a large copy).
template <int NT> __host__ __device__ constexpr int64_t narrow_lds(int64_t kb) { return 16 * NT * kb * 128 + 2 * kb + 16 * NT * 4; }
template <typename T, int NT>
__global__ __launch_bounds__(256, NT <= 8 ? 3 : 2) void linear8_narrow_kernel(const T* __restrict__ x, const uint8_t* __restrict__ qw, const uint8_t* __restrict__ ew, const T* __restrict__ bias, T* __restrict__ y,
                                                             int64_t rows, int k, int n) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int E = 16 / sizeof(T), J = 32 / E;                                           // columns per load, loads per lane and block
    const int kb = (int)kblocks(k), kp = kb * 128, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    float* const sbias = reinterpret_cast<float*>(lds + 16 * NT * kp);
    uint8_t* const sexp = reinterpret_cast<uint8_t*>(sbias + 16 * NT);
    // Block b is read from column first(b) on: a last block that is not full is moved back to end with the row (k >= 128), and its first columns, which belong
    // to the block before, are dropped from x: every load stays inside its row, at full width.
    const auto first = [&](int b) { return min(b * 128, k - 128); };
    // byte 4 E j + E g + e of a block (column order) -> byte 32 g + E j + e (lane order); its 16-byte piece p of row r lies at place p ^ (r & 7)
    for (int t = threadIdx.x; t < 16 * NT * kp / 4; t += 256) {
        const int r = t / (kp / 4), c = (t - r * (kp / 4)) * 4, b = c >> 7, o = c & 127;
        const int to = 32 * (o % (4 * E) / E) + E * (o / (4 * E)) + o % E;
        unsigned v = 0u;
        if (r < n) __builtin_memcpy(&v, qw + (int64_t)r * kp + first(b) + o, 4);
        *reinterpret_cast<unsigned*>(lds + r * kp + b * 128 + ((to >> 4) ^ (r & 7)) * 16 + (to & 15)) = v;
    }
    for (int t = threadIdx.x; t < 16 * NT; t += 256) sbias[t] = bias && t < n ? (float)bias[t] : 0.f;
    for (int t = threadIdx.x; t < 2 * kb; t += 256) sexp[t] = t < (n + 127) / 128 * kb ? ew[t] : 127;
    __syncthreads();

    const int64_t tiles = (rows + 15) / 16, step = (int64_t)gridDim.x * 4;
    nvp_vec<T, E> raw[J];
    const auto fetch = [&](int64_t tile, int b) {
        const T* p = x + min(tile * 16 + i, rows - 1) * k + first(b) + g * E;               // rows behind the last one read the last one: their results are not stored
#pragma unroll
        for (int j = 0; j < J; ++j) raw[j] = nvp_load_raw<T, E>(p + j * 4 * E);
    };
    int64_t tile = (int64_t)blockIdx.x * 4 + wave;
    if (tile < tiles) fetch(tile, 0);
    for (; tile < tiles; tile += step) {
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int b = 0; b < kb; ++b) {
            float v[32];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) v[j * E + e] = (float)raw[j].v[e];
            if (first(b) < b * 128) {
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) v[j * E + e] = first(b) + (j * 4 + g) * E + e < b * 128 ? 0.f : v[j * E + e];
            }
            {
                const bool here = b + 1 < kb;
                const int64_t then = here ? tile : tile + step;
                if (then < tiles) fetch(then, here ? b + 1 : 0);
            }
            unsigned top = 0u;
#pragma unroll
            for (int e = 0; e < 32; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
            top = max(top, (unsigned)__shfl_xor((int)top, 16));
            top = max(top, (unsigned)__shfl_xor((int)top, 32));
            const bool odd = __any(top >= 0x7f800000u);                                     // an infinity or a NaN somewhere in the 16 rows: the careful way
            if (odd) {
                top = 0u;
#pragma unroll
                for (int e = 0; e < 32; ++e) top = max(top, finite_bits(v[e]));
                top = max(top, (unsigned)__shfl_xor((int)top, 16));
                top = max(top, (unsigned)__shfl_xor((int)top, 32));
            }
            const unsigned byte = scale_byte(top);
            const float inv = inv_scale(byte);
            v8i q;
            if (odd) {
#pragma unroll
                for (int p = 0; p < 8; ++p) q[p] = quant4(&v[4 * p], inv);
            } else {
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * p] * inv, v[4 * p + 1] * inv, 0, false);
                    q[p] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * p + 2] * inv, v[4 * p + 3] * inv, w, true);
                }
            }
            frag<kWide> xf;
            xf.set(q, (int)byte);
            const int s0 = sexp[b], s1 = sexp[kb + b];
            __builtin_amdgcn_sched_barrier(0);                                              // operand reads stay behind the quantisation: its registers are free then
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                frag<kWide> wf[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = 16 * (t + u) + i;
                    const uint8_t* w = lds + r * kp + b * 128;
                    const v4i lo = *reinterpret_cast<const v4i*>(w + ((2 * g) ^ (r & 7)) * 16), hi = *reinterpret_cast<const v4i*>(w + ((2 * g + 1) ^ (r & 7)) * 16);
                    wf[u].set(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), t < 8 ? s0 : s1);
                }
                mma2(wf[0], wf[1], xf, acc[t], acc[t + 1]);
            }
        }
        const int64_t row = tile * 16 + i;
        // D: row (column of y) 4 (lane >> 4) + r, column (row of y) lane & 15
        if (row < rows && n % 4 == 0) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int c = 16 * t + 4 * g;
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = acc[t][e] + sbias[c + e];
                if (c < n) nvp_store<T, 4>(y + row * n + c, f);
            }
        } else if (row < rows) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (16 * t + 4 * g + e < n) y[row * n + 16 * t + 4 * g + e] = (T)(acc[t][e] + sbias[16 * t + 4 * g + e]);
        }
    }
}

// ---- many rows: BM x BN tiles through LDS --------------------------------------------------------------------------------------------------
// A ring of STAGES blocks (128 columns), (BM + BN) x 128 bytes each, filled by direct-to-LDS loads STAGES - 1 blocks ahead; a wave computes
// (BM / WM) x (BN / WN) with 32x32x64 instructions.  One barrier per block, at its start: behind it the block has landed for everyone (every wave waits for
// its own loads, counted: those of later blocks stay in flight) and the stage of the block before has been read, so that its refill is issued at once.
// The scales come through LDS too: a load into registers would be waited for together with all fills before it.
// Measured, with the quantising launch: 8192 x 8192 x 8192 bf16 490 us, 2.24 PFLOP/s (the 256 x 256 tile; the matrix units are busy 57 % of the cycles of a
// clock that their power holds at 1.8 GHz of 2.4: finer interleaving of loads, reads and products, in 4 or 8 waves, was not faster); 256 x 4096 x 4096
// 15.3 us, the tile kernel 13: 256 tiles, so one wave per SIMD, whose 32 blocks take 800 cycles each: 330 of them to fill a stage (16 KB at 50 bytes per clock), 140 of LDS reads,
// 130 of products, one behind the other behind a barrier (counters: the waves wait 45 % of their life, the matrix units are busy 16 % of it, LDS 17 %); splitting a tile's
// blocks over two or four teams of waves was not faster.
// LDS rows are 128 bytes; the 16-byte piece c of row r lies at place c ^ (r >> 1 & 7): of any 16 rows that one 256-byte LDS cycle serves (0 - 15, or
// 0-3, 12-15, 20-23, 24-27) no two share a bank (measured: no conflicts; with c ^ (r & 7) a third of the LDS cycles were conflicts).  The loads swizzle on
// their global side (LDS writes are linear).
template <int AT> __device__ __forceinline__ void glds16(const void* ubase, unsigned lane_off, unsigned lds_byte) {      // to LDS byte lds_byte + AT + 16 lane
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(ubase), "s"(lds_byte), "n"(AT) : "memory", "scc");
}
__device__ __forceinline__ void glds4(const void* ubase, unsigned lane_off, unsigned lds_byte) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(lane_off), "s"(ubase), "s"(lds_byte) : "memory");
}
// every wave's loads but the LATER newest have landed and its LDS reads have returned (that wait by the builtin: the compiler then knows, and waits for them no second time)
template <int LATER> __device__ __forceinline__ void stage_barrier() {
    static_assert(LATER < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

template <int A, int B, typename F> __device__ __forceinline__ void static_for(const F& f) {      // f(A) .. f(B - 1), the argument a constant
    if constexpr (A < B) {
        f(std::integral_constant<int, A>());
        static_for<A + 1, B>(f);
    }
}

template <int BM, int BN, int STAGES> constexpr int tile_lds() { return STAGES * (BM + BN) * 128 + (STAGES > 2 ? 4 : 2) * BM * 4; }
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void linear8_tile_kernel(const uint8_t* __restrict__ qx, const uint8_t* __restrict__ ex, const uint8_t* __restrict__ qw,
                                                                    const uint8_t* __restrict__ ew, const T* __restrict__ bias, T* __restrict__ y, int64_t rows, int64_t k,
                                                                    int64_t n, int tiles_m, int tiles_n) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int kWaves = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int kStage = (BM + BN) * 128, kPlaces = STAGES > 2 ? 4 : 2;
    constexpr int kLoads = (BM + BN) / 8 / kWaves;                                           // one load instruction: 8 rows x 128 bytes
    static_assert(STAGES <= 5 && (BM + BN) % (16 * kWaves) == 0 && BN / WN <= 128 && BM % 64 == 0 && BM / 64 <= kWaves && kLoads % 2 == 0, "tile shape");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, i = lane & 31, hl = lane >> 5;
    const int64_t kb = kblocks(k), kp = kb * 128, kbp = kb4(k);
    const int blocks = (int)kb;

    // workgroups go to the eight XCDs in turn: give each XCD a contiguous run of tiles, walked in groups of 8 tile rows, so that the
    // tiles an XCD works on at one time share operand rows in its own L2
    const int total = tiles_m * tiles_n;
    int id = blockIdx.x;
    {
        const int per = total / 8, more = total % 8, xcd = id % 8, at = id / 8;
        id = xcd * per + min(xcd, more) + at;
    }
    const int gsz = 8 * tiles_n, grp = id / gsz, in = id - grp * gsz, gm = min(8, tiles_m - grp * 8);
    const int tm = __builtin_amdgcn_readfirstlane(grp * 8 + in % gm), tn = __builtin_amdgcn_readfirstlane(in / gm);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;

    // Source rows: row r of a stage is x row m0 + r (r < BM) or weight row n0 + r - BM, in groups of 8; a wave's kLoads groups are all of one kind.  Groups
    // behind the end read the last one; weight rows behind the last one read that row.  (x rows behind the last one are in the workspace, unwritten: what
    // comes of them is not stored.)  Addresses: one scalar that moves with the block, one offset per lane and group that does not.
    static_assert(BM / 8 % kLoads == 0, "a wave loads x or weights");
    const bool isx = wave * kLoads * 8 < BM;
    const uint8_t* const src = isx ? qx + (m0 >> 3) * (kb * 1024) : qw + n0 * kp;
    const int advance = isx ? 1024 : 128;
    const int lr = lane >> 3;
    unsigned off[kLoads];
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
        const int g = wave * kLoads + q;
        const int64_t row = isx ? min((m0 >> 3) + g, (rows - 1) >> 3) - (m0 >> 3) : min(n0 + 8 * g - BM + lr, n - 1) - n0;
        const unsigned piece = 16u * ((lane & 7) ^ (lr >> 1) ^ (4 * (q & 1)));               // (row >> 1) & 7 = 4 (group & 1) + (lr >> 1), kLoads is even
        off[q] = isx ? (unsigned)(row * kb * 1024) + lr * 128u + piece : (unsigned)(row * kp) + piece;      // < BM * kp: the host sees to it that it fits
    }
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;      // STAGES x operands, kPlaces x scales
    const auto fill1 = [&](int b, auto q_) {                                                 // (behind the end the last block is fetched again, into a stage that nobody reads)
        constexpr int q = decltype(q_)::value;
        glds16<q * 1024>(src + (int64_t)min(b, blocks - 1) * advance, off[q], lds0 + (unsigned)b % STAGES * kStage + wave * kLoads * 1024);
    };
    // Scale dwords of four blocks: with block j a wave fetches group (j + 3) / 4 for 64 rows of x, so that the fetches in flight can be counted and a group's first
    // fetch is four blocks old when it is read (the block's own group: 8192 x 8192 x 8192 3 % slower).  Block b reads group b / 4; fetches on their way are for
    // groups up to (b + STAGES + 2) / 4: one behind it with two stages, two with up to five.
    const int srow = wave % (BM / 64) * 64;
    const int64_t sfirst = min(m0 + srow, rows - 1);
    const uint8_t* const sbase = ex + sfirst * kbp;
    const unsigned soff = (unsigned)(min((int64_t)lane, rows - 1 - sfirst) * kbp);
    const auto scales1 = [&](int b) { glds4(sbase + 4 * min((b + 3) >> 2, (blocks - 1) >> 2), soff, lds0 + STAGES * kStage + ((b + 3) >> 2) % kPlaces * (BM * 4) + srow * 4); };
    const uint32_t* const wsrc = reinterpret_cast<const uint32_t*>(ew + min((n0 + wn * (BN / WN)) / 128, (n - 1) / 128) * kbp);      // the wave's columns lie in one weight block row

    f32x16 acc[TM][TN];
#pragma unroll
    for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b) acc[a][b] = nvp_zero16();

    // operands of a half block: 16-byte pieces 4 half + 2 hl and the one behind it, of row i of a 32-row tile
    const int sw = i >> 1 & 7, xrow = (wm * (BM / WM) + i) * 128, wrow = (BM + wn * (BN / WN) + i) * 128;
    const auto operand = [&](int b, int half, int row, int t) {
        const uint8_t* st = lds + (unsigned)b % STAGES * kStage + row + t * 4096;
        return __builtin_shufflevector(*reinterpret_cast<const v4i*>(st + 16 * ((4 * half + 2 * hl) ^ sw)), *reinterpret_cast<const v4i*>(st + 16 * ((4 * half + 2 * hl + 1) ^ sw)), 0, 1, 2, 3, 4, 5,
                                       6, 7);
    };
    const auto scale = [&](int b, int a) { return *reinterpret_cast<const uint32_t*>(lds + STAGES * kStage + (b >> 2) % kPlaces * (BM * 4) + (wm * (BM / WM) + 32 * a + i) * 4); };
    static_for<0, STAGES - 1>([&](auto b) {
        static_for<0, kLoads>([&](auto q) { fill1(b, q); });
        scales1(b);
    });
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
        stage_barrier<(STAGES - 2) * (kLoads + 1)>();
        const int sh = 8 * (b & 3);
        const uint32_t ws = wsrc[b >> 2];
        uint32_t xs[TM];
#pragma unroll
        for (int a = 0; a < TM; ++a) xs[a] = scale(b, a);
        static_for<0, kLoads>([&](auto q) { fill1(b + STAGES - 1, q); });
        scales1(b + STAGES - 1);
        __builtin_amdgcn_sched_barrier(0);                                                   // nothing waits for the scales before all loads are on their way
        static_for<0, 2>([&](auto half_) {
            constexpr int half = decltype(half_)::value;
            frag<kWide> wf[TN];
#pragma unroll
            for (int t = 0; t < TN; ++t) wf[t].set(operand(b, half, wrow, t), (int)(ws >> sh));
            static_for<0, TM>([&](auto a_) {
                constexpr int a = decltype(a_)::value;
                frag<kWide> xf;
                xf.set(operand(b, half, xrow, a), (int)(xs[a] >> sh));
#pragma unroll
                for (int t = 0; t < TN; ++t) acc[a][t] = mma(xf, wf[t], acc[a][t]);
            });
        });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                         // the last fetches, before this LDS can be another workgroup's
#pragma unroll
    for (int t = 0; t < TN; ++t) {
        const int64_t col = n0 + wn * (BN / WN) + 32 * t + i;
        if (col >= n) continue;
        const float bv = bias ? (float)bias[col] : 0.f;
#pragma unroll
        for (int a = 0; a < TM; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t row = m0 + wm * (BM / WM) + 32 * a + nvp_frag_row(r, hl);
                if (row < rows) y[row * n + col] = (T)(acc[a][t][r] + bv);
            }
    }
}

// A launch has fewer than 2^32 threads along x.
constexpr int64_t kMaxThreads = (1ll << 32) - 1, kMaxGroups = kMaxThreads / 256;             // (workgroups of 256)
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
int launch_tile(const uint8_t* qx, const uint8_t* ex, const uint8_t* qw, const uint8_t* ew, const void* bias, void* y, int64_t rows, int64_t k, int64_t n, hipStream_t st) {
    const int64_t tm = (rows + BM - 1) / BM, tn = (n + BN - 1) / BN;
    if (tm * tn * (64 * WM * WN) > kMaxThreads || kblocks(k) * 128 * BM > 0xffffffffll || kblocks(k) * 128 * BN > 0xffffffffll) return NVP_ERR_UNSUPPORTED;      // 32-bit offsets inside a tile
    constexpr size_t lds = tile_lds<BM, BN, STAGES>();
    // (HIP on gfx950 takes more than 64 KiB of dynamic LDS with or without the attribute: a refusal must not fail the call)
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(linear8_tile_kernel<T, BM, BN, WM, WN, STAGES>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (attr != hipSuccess) (void)hipGetLastError();
    hipLaunchKernelGGL((linear8_tile_kernel<T, BM, BN, WM, WN, STAGES>), dim3((unsigned)(tm * tn)), dim3(64 * WM * WN), lds, st, qx, ex, qw, ew, (const T*)bias, (T*)y, rows, k, n, (int)tm, (int)tn);
    NVP_LAUNCH_CHECK();
    return 0;
}

int64_t rows_lds(int64_t rows, int64_t k) { return rows * (kblocks(k) * 129 + 16); }
template <typename T, int MT, int NT, int WAVES, bool FUSED>
int launch_rows(const T* x, const uint8_t* qx, const uint8_t* ex, const uint8_t* qw, const uint8_t* ew, const void* bias, void* y, int64_t rows, int64_t k, int64_t n, hipStream_t st) {
    const int64_t gx = (n + 16 * NT - 1) / (16 * NT), gy = (rows + 16 * MT - 1) / (16 * MT);
    if (gy > 65535 || gx * (64 * WAVES) > kMaxThreads) return NVP_ERR_UNSUPPORTED;
    const int64_t xbytes = FUSED ? rows_lds(rows < 16 * MT ? rows : 16 * MT, k) : 0, pbytes = WAVES * MT * 16 * (NT * 16 + 1) * 4;
    hipLaunchKernelGGL((linear8_rows_kernel<T, MT, NT, WAVES, FUSED>), dim3((unsigned)gx, (unsigned)gy), dim3(64 * WAVES), (size_t)(xbytes > pbytes ? xbytes : pbytes), st, x, qx, ex, qw, ew,
                       (const T*)bias, (T*)y, rows, k, n);
    NVP_LAUNCH_CHECK();
    return 0;
}

// The path for (rows, k, n); both the workspace query and the call go by it.
enum { kFew, kNarrow, kRows, kTiles64, kTiles128, kTiles128x2, kTiles256 };
int narrow_columns(int64_t rows, int64_t k, int64_t n);
int path_of(int64_t rows, int64_t k, int64_t n) {
    // up to 64 blocks of x: two per 16 lanes, one round of loads; beyond that a quantising launch of its own is the shorter way (16 rows x 4096 times 4096
    // columns: 9.3 us with it, 16.4 us without; 1 row: 7.0 us without)
    if (rows <= 16 && rows * kblocks(k) <= 64) return kFew;
    if (narrow_columns(rows, k, n)) return kNarrow;
    // bf16, 4096 x 4096 weights, us with the quantising launch, for the rows kernel / 64 x 64 tiles / 128 x 128 tiles one per CU / two per CU / 256 x 256:
    // 32 rows 12.3 / 13 / 21 / 25 / 48;  64 rows 18 / 13.5 / 21 / 26 / 48;  512 rows - / 26 / 26 / 32 / 54;  1024 rows - / 44 / 30 / 35 / 56;
    // 2048 rows - / 79 / 56 / 46 / 60;  4096 rows - / 146 / 103 / 87 / 76: the smallest tile that still runs in one round of the chip (two
    // workgroups per CU where their LDS allows it), and the largest, which reads the least, for what takes more rounds than that
    if (rows <= 32) return kRows;
    const auto tiles = [&](int64_t b) { return ((rows + b - 1) / b) * ((n + b - 1) / b); };
    if (tiles(64) <= 512) return kTiles64;
    if (tiles(128) <= 256) return kTiles128;
    return tiles(128) <= 512 ? kTiles128x2 : kTiles256;
}
// Columns rounded up to 64, 128 or 256 where the narrow kernel is the faster one, else 0: the weights leave room for two workgroups per CU, there is a whole
// block to read (k >= 128: the kernel moves a row's last block back to end with the row), and the rows are worth the time it takes every workgroup to lay
// the weights out (12 us for 32 KB, 21 us for 64 KB).  bf16, us, tiles / narrow: 242 -> 128 columns (32 KB) 8192 rows 8.1 / 13.0, 32768 rows 16 / 14, 131072 rows
// 52 / 31, 524288 rows 199 / 109;  130 -> 64 (16 KB) 65536 rows 22 / 12;  1000 -> 64 (64 KB) 65536 rows 49 / 64, 131072 rows 121 / 94;  512 -> 128 (64 KB) 131072
// rows 68 / 70, 524288 rows 277 / 198;  228 -> 256 (64 KB) 131072 rows 54 / 71 (fp32 83 / 82), 524288 rows 226 / 174.
int narrow_columns(int64_t rows, int64_t k, int64_t n) {
    const int nt = n <= 64 ? 4 : n <= 128 ? 8 : n <= 256 ? 16 : 0;
    const int64_t bytes = 16 * nt * kblocks(k) * 128;
    return k >= 128 && nt && bytes <= 65536 && rows >= 2 * bytes ? 16 * nt : 0;
}
template <typename T, int NT>
int launch_narrow(const T* x, const uint8_t* qw, const uint8_t* ew, const void* bias, void* y, int64_t rows, int64_t k, int64_t n, hipStream_t st) {
    const int64_t groups = (rows + 63) / 64;
    const size_t bytes = (size_t)narrow_lds<NT>(kblocks(k));
    hipLaunchKernelGGL((linear8_narrow_kernel<T, NT>), dim3((unsigned)(groups < 768 ? groups : 768)), dim3(256), bytes, st, x, qw, ew, (const T*)bias, (T*)y, rows,
                       (int)k, (int)n);
    NVP_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int linear8(const T* x, const uint8_t* qw, const uint8_t* ew, const void* bias, void* y, int64_t rows, int64_t k, int64_t n, uint8_t* ws, hipStream_t st) {
    const int path = path_of(rows, k, n);
    // few columns: twice the waves per workgroup, so that the chip still has enough of them
    if (path == kFew) {
        return n <= 2048 ? launch_rows<T, 1, 1, 16, true>(x, nullptr, nullptr, qw, ew, bias, y, rows, k, n, st) : launch_rows<T, 1, 1, 8, true>(x, nullptr, nullptr, qw, ew, bias, y, rows, k, n, st);
    }
    switch (path == kNarrow ? narrow_columns(rows, k, n) : 0) {
        case 64: return launch_narrow<T, 4>(x, qw, ew, bias, y, rows, k, n, st);
        case 128: return launch_narrow<T, 8>(x, qw, ew, bias, y, rows, k, n, st);
        case 256: return launch_narrow<T, 16>(x, qw, ew, bias, y, rows, k, n, st);
    }
    const int64_t kb = kblocks(k), kbp = kb4(k), nb = (n + 127) / 128;
    uint8_t* const qx = ws;
    uint8_t* const ex = qx + xq_bytes(rows, kb);
    uint8_t* const ewp = ex + rows * kbp;                                                    // rows * kbp is a multiple of 4
    // the weights' scales with the first rows; as many rows a launch as it may have workgroups (a multiple of 8: those share a piece of the workspace)
    const int64_t tail = (nb * kbp + 255) / 256, most = (kMaxGroups - tail) * 16 / kb / 8 * 8;
    if (most < 8) return NVP_ERR_UNSUPPORTED;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t here = rows - r < most ? rows - r : most, groups = (here * kb + 15) / 16;
        hipLaunchKernelGGL((quant_rows_kernel<T>), dim3((unsigned)(groups + (r ? 0 : tail))), dim3(256), 0, st, x + r * k, qx + xq_bytes(r, kb), ex + r * kbp, here, k, groups, ew, ewp,
                           nb * kbp);
        NVP_LAUNCH_CHECK();
    }
    switch (path) {
        case kRows: {
            const bool narrow = (n + 31) / 32 < 256;                                         // 16 columns per workgroup where 32 would leave CUs without one
            if (rows <= 16) return launch_rows<T, 1, 1, 8, false>(x, qx, ex, qw, ewp, bias, y, rows, k, n, st);
            return narrow ? launch_rows<T, 2, 1, 8, false>(x, qx, ex, qw, ewp, bias, y, rows, k, n, st) : launch_rows<T, 2, 2, 8, false>(x, qx, ex, qw, ewp, bias, y, rows, k, n, st);
        }
        case kTiles64: return launch_tile<T, 64, 64, 2, 2, 4>(qx, ex, qw, ewp, bias, y, rows, k, n, st);
        case kTiles128: return launch_tile<T, 128, 128, 4, 2, 4>(qx, ex, qw, ewp, bias, y, rows, k, n, st);
        case kTiles128x2: return launch_tile<T, 128, 128, 2, 2, 2>(qx, ex, qw, ewp, bias, y, rows, k, n, st);
        default: return launch_tile<T, 256, 256, 2, 4, 2>(qx, ex, qw, ewp, bias, y, rows, k, n, st);
    }
}

// as many rows a launch as it may have workgroups: k is at most 2^24, so that is at least 127 blocks of rows, and 255 rows of values
template <typename T> int quant_blocks(const T* x, uint8_t* q, uint8_t* e, int64_t rows, int64_t k, int block_rows, hipStream_t st) {
    const int64_t kb = kblocks(k), most = kMaxGroups / kb * block_rows;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t here = rows - r < most ? rows - r : most, groups = (here + block_rows - 1) / block_rows * kb;
        hipLaunchKernelGGL((quant_blocks_kernel<T>), dim3((unsigned)groups), dim3(256), 0, st, x + r * k, q + r * kb * 128, e + r / block_rows * kb, here, k, block_rows);
        NVP_LAUNCH_CHECK();
    }
    return 0;
}
template <typename T> int dequant_blocks(const uint8_t* q, const uint8_t* e, T* x, int64_t rows, int64_t k, int block_rows, hipStream_t st) {
    const int64_t kb = kblocks(k), most = kMaxGroups * 256 / k / block_rows * block_rows;
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t here = rows - r < most ? rows - r : most, groups = (here * k + 255) / 256;
        hipLaunchKernelGGL((dequant_blocks_kernel<T>), dim3((unsigned)groups), dim3(256), 0, st, q + r * kb * 128, e + r / block_rows * kb, x + r * k, here, k, block_rows);
        NVP_LAUNCH_CHECK();
    }
    return 0;
}

bool sizes_ok(int64_t rows, int64_t k, int64_t n) { return rows >= 0 && n >= 1 && k >= 1 && rows <= (1ll << 31) - 1 && n <= (1ll << 31) - 1 && k <= (1ll << 24); }

}  // namespace

extern "C" int64_t nvp_linear8_workspace_bytes(int64_t rows, int64_t k, int64_t n) {
    if (!sizes_ok(rows, k, n)) return NVP_ERR_BADARG;
    const int path = path_of(rows, k, n);
    if (path == kFew || path == kNarrow) return 0;
    return xq_bytes(rows, kblocks(k)) + rows * kb4(k) + (n + 127) / 128 * kb4(k);
}

extern "C" int nvp_linear8(const void* x, int32_t type, const uint8_t* q, const uint8_t* e, const void* bias, void* y, int64_t rows, int64_t k, int64_t n, void* workspace,
                           int64_t workspace_bytes, void* stream) {
    if (!sizes_ok(rows, k, n) || !nvp_type_size(type)) return NVP_ERR_BADARG;
    if (rows == 0) return 0;
    if (!x || !q || !e || !y || ((uintptr_t)q & 15)) return NVP_ERR_BADARG;
    const int64_t need = nvp_linear8_workspace_bytes(rows, k, n);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return NVP_ERR_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    if (type == NVP_F32) return linear8<float>((const float*)x, q, e, bias, y, rows, k, n, (uint8_t*)workspace, st);
    if (type == NVP_BF16) return linear8<nvp_bf16>((const nvp_bf16*)x, q, e, bias, y, rows, k, n, (uint8_t*)workspace, st);
    return linear8<nvp_f16>((const nvp_f16*)x, q, e, bias, y, rows, k, n, (uint8_t*)workspace, st);
}

extern "C" int nvp_quantize_blocks(const void* x, int32_t type, uint8_t* q, uint8_t* e, int64_t rows, int64_t k, int32_t block_rows, void* stream) {
    if (!sizes_ok(rows, k, 1) || !nvp_type_size(type) || (block_rows != 1 && block_rows != 128)) return NVP_ERR_BADARG;
    if (rows == 0) return 0;
    if (!x || !q || !e) return NVP_ERR_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    if (type == NVP_F32) return quant_blocks<float>((const float*)x, q, e, rows, k, block_rows, st);
    if (type == NVP_BF16) return quant_blocks<nvp_bf16>((const nvp_bf16*)x, q, e, rows, k, block_rows, st);
    return quant_blocks<nvp_f16>((const nvp_f16*)x, q, e, rows, k, block_rows, st);
}

extern "C" int nvp_dequantize_blocks(const uint8_t* q, const uint8_t* e, void* x, int32_t type, int64_t rows, int64_t k, int32_t block_rows, void* stream) {
    if (!sizes_ok(rows, k, 1) || !nvp_type_size(type) || (block_rows != 1 && block_rows != 128)) return NVP_ERR_BADARG;
    if (rows == 0) return 0;
    if (!x || !q || !e) return NVP_ERR_BADARG;
    const hipStream_t st = (hipStream_t)stream;
    if (type == NVP_F32) return dequant_blocks<float>(q, e, (float*)x, rows, k, block_rows, st);
    if (type == NVP_BF16) return dequant_blocks<nvp_bf16>(q, e, (nvp_bf16*)x, rows, k, block_rows, st);
    return dequant_blocks<nvp_f16>(q, e, (nvp_f16*)x, rows, k, block_rows, st);
}
