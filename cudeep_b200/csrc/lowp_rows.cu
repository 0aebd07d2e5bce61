// One-pass kernels around the 8-bit and the grouped products: padding of rows for the TMA unit, quantisation to e4m3
// in blocks and back.  All are bound by HBM: each input is read once and each output written once.
#include "lowp_rows.h"

#include "epilogue_math.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace cudeep_b200 {

namespace {

constexpr int kThreads = 256;

// dst[r, 0..ld) = src[r, 0..cols) followed by zeros; ld is a multiple of 16 bytes, a thread writes 16 of them.
template <typename T>
__global__ void pad_rows_kernel(const T* __restrict__ src, T* __restrict__ dst, long long rows, int cols, int units_row) {
    constexpr int V = 16 / sizeof(T);
    const long long total = rows * units_row;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / units_row;
        const int c0 = int(i - r * units_row) * V;
        const T* s = src + r * cols + c0;
        alignas(16) T v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = c0 + j < cols ? s[j] : T(0);
        reinterpret_cast<uint4*>(dst)[i] = *reinterpret_cast<const uint4*>(v);
    }
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements from a 16-byte aligned (32 for float: two loads) address.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_float(t[j]);
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;      // NaN compares false
}

// Exponent e of the block's scale 2^e: the least with amax <= 448 * 2^e = 1.75 * 2^(e + 8), not below -126 (the scale
// stays a normal number); 0 for a block of zeros.  Read from amax's bits, so it is exact.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    if (bits == 0) return 0;
    const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }      // -126 <= e <= 127

// x / 2^e in e4m3, rounded to nearest even once (the division by a power of two is exact); NaN for what is not finite.
__device__ __forceinline__ uint32_t e4m3(float x, float inv) {
    const float v = x * inv;
    const uint32_t q = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
    return fabsf(x) <= 3.402823466e38f ? q : 0x7fu;
}

// Blocks of 1 x 128.  Sixteen lanes own a block, eight elements each; a warp takes two neighbouring blocks of four
// rows at once (four independent 16-byte loads in flight per lane for 16-bit types), a CTA 32 rows x 256 columns.  The
// scales lie [block][row], so the CTA collects its 32 x 2 scales in shared memory and writes runs of 32.
// VEC: rows start on 16-byte boundaries; otherwise a lane takes every sixteenth element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                 uint8_t* __restrict__ q, float* __restrict__ scales) {
    __shared__ float s_scale[2][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = lane >> 4, l16 = lane & 15;
    const int block = blockIdx.x * 2 + half;
    const int c0 = block * FP8_BLOCK;
    const long long row0 = (long long)blockIdx.y * 32 + warp * 4;
    float v[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = row0 + i;
        const T* src = x + r * cols + c0;
        if (VEC) {
            if (r < rows && c0 + l16 * 8 < cols) {
                load8(src + l16 * 8, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = r < rows && c0 + l16 + 16 * j < cols ? to_float(src[l16 + 16 * j]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(v[i][j]));
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        const int e = scale_exponent(amax);
        const float inv = pow2(-e);
        if (l16 == 0) s_scale[half][warp * 4 + i] = pow2(e);
        const long long r = row0 + i;
        uint8_t* dst = q + r * cols + c0;
        if (r < rows) {
            if (VEC) {
                if (c0 + l16 * 8 < cols) {
                    uint2 out;
                    out.x = e4m3(v[i][0], inv) | e4m3(v[i][1], inv) << 8 | e4m3(v[i][2], inv) << 16 | e4m3(v[i][3], inv) << 24;
                    out.y = e4m3(v[i][4], inv) | e4m3(v[i][5], inv) << 8 | e4m3(v[i][6], inv) << 16 | e4m3(v[i][7], inv) << 24;
                    *reinterpret_cast<uint2*>(dst + l16 * 8) = out;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c0 + l16 + 16 * j < cols) dst[l16 + 16 * j] = uint8_t(e4m3(v[i][j], inv));
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int b = threadIdx.x >> 5;
        const long long r = (long long)blockIdx.y * 32 + lane;
        const int blk = blockIdx.x * 2 + b;
        if (r < rows && (long long)blk * FP8_BLOCK < cols) scales[(long long)blk * rows + r] = s_scale[b][lane];
    }
}

// Blocks of 128 x 128, one CTA each: sixteen lanes hold a row's 128 columns, a thread 8 rows x 8 columns, so the block
// is read once and stays in registers while its maximum is found.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scales) {
    __shared__ float s_max[kThreads / 32];
    const int l16 = threadIdx.x & 15, rr = threadIdx.x >> 4;
    const int c0 = blockIdx.x * FP8_BLOCK;
    const long long row0 = (long long)blockIdx.y * FP8_BLOCK + rr;
    float v[8][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = row0 + 16 * i;
        const T* src = x + r * cols + c0;
        if (VEC) {
            if (r < rows && c0 + l16 * 8 < cols) {
                load8(src + l16 * 8, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = r < rows && c0 + l16 + 16 * j < cols ? to_float(src[l16 + 16 * j]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = fmaxf(amax, finite_abs(v[i][j]));
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, s_max[w]);
    const int e = scale_exponent(amax);
    const float inv = pow2(-e);
    if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = pow2(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = row0 + 16 * i;
        if (r >= rows) break;
        uint8_t* dst = q + r * cols + c0;
        if (VEC) {
            if (c0 + l16 * 8 < cols) {
                uint2 out;
                out.x = e4m3(v[i][0], inv) | e4m3(v[i][1], inv) << 8 | e4m3(v[i][2], inv) << 16 | e4m3(v[i][3], inv) << 24;
                out.y = e4m3(v[i][4], inv) | e4m3(v[i][5], inv) << 8 | e4m3(v[i][6], inv) << 16 | e4m3(v[i][7], inv) << 24;
                *reinterpret_cast<uint2*>(dst + l16 * 8) = out;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c0 + l16 + 16 * j < cols) dst[l16 + 16 * j] = uint8_t(e4m3(v[i][j], inv));
        }
    }
}

__device__ __forceinline__ float e4m3_value(uint8_t q) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

template <typename T>
__global__ void dequantize_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scales, long long rows, int cols,
                                  int block_rows, T* __restrict__ y) {
    const int col_blocks = (cols + FP8_BLOCK - 1) / FP8_BLOCK;
    const long long total = rows * cols;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / cols;
        const int b = int(i - r * cols) / FP8_BLOCK;
        const float s = __ldg(scales + (block_rows == 1 ? b * rows + r : (r / FP8_BLOCK) * col_blocks + b));
        y[i] = from_float<T>(e4m3_value(q[i]) * s);
    }
}

// Slope of the epilogue activations (tanh-form GELU) from CUDA's own expf and tanhf: the pass is bound by HBM, so the
// accurate functions cost nothing.
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == EPI_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (act == EPI_GELU) {
        // Beyond +-30 the slope is 0 or 1 to the last bit, and z * z * z must not overflow.
        z = fminf(fmaxf(z, -30.0f), 30.0f);
        const float c = 0.7978845608028654f;
        const float th = tanhf(c * (z + 0.044715f * z * z * z));
        return 0.5f * (1.0f + th) + 0.5f * z * (1.0f - th * th) * c * (1.0f + 3.0f * 0.044715f * z * z);
    }
    if (act == EPI_NONE) return 1.0f;
    const float s = 1.0f / (1.0f + expf(-z));
    if (act == EPI_SIGMOID) return s * (1.0f - s);
    return s > 0.0f ? s * (1.0f + z * (1.0f - s)) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    alignas(16) T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_float<T>(v[j]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
}

// A CTA takes 256 columns and `rows_per` rows: 32 threads with eight columns each lie along a row, eight rows are worked on at
// once.  Column sums stay in registers over the rows, are added across the eight threads of a column in a fixed order and go
// to partial[row band][cols], which one more kernel adds up, again in order: the result does not depend on timing.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) act_backward_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ z8,
                                                                const float* __restrict__ zs, int act, T* __restrict__ dz,
                                                                long long ld_dz, float* __restrict__ partial, int rows, int cols,
                                                                int rows_per) {
    __shared__ float s_sum[8][264];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 256 + tx * 8;
    const int r_end = min(rows, int(blockIdx.y + 1) * rows_per);
    float sum[8] = {};
    if (c0 < cols) {
        const float* s_col = zs + (long long)(c0 / FP8_BLOCK) * rows;
        for (int r = blockIdx.y * rows_per + ty; r < r_end; r += 8) {
            const long long at = (long long)r * cols + c0;
            float g[8];
            if (VEC) {
                load8(dy + at, g);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = c0 + j < cols ? to_float(dy[at + j]) : 0.0f;
            }
            if (act != EPI_NONE) {
                uint8_t q[8];
                if (VEC) {
                    *reinterpret_cast<uint2*>(q) = __ldg(reinterpret_cast<const uint2*>(z8 + at));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) q[j] = c0 + j < cols ? z8[at + j] : uint8_t(0);
                }
                const float s = __ldg(s_col + r);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] *= act_slope(e4m3_value(q[j]) * s, act);
            }
            if (!VEC) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c0 + j >= cols) g[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
            if (dz != nullptr) store8(dz + r * ld_dz + c0, g);
        }
    }
    if (partial == nullptr) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) s_sum[ty][tx * 8 + j] = sum[j];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < cols) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += s_sum[i][threadIdx.x];
        partial[(long long)blockIdx.y * cols + c] = total;
    }
}

__global__ void __launch_bounds__(kThreads) add_bands_kernel(const float* __restrict__ partial, int bands, int cols,
                                                             float* __restrict__ out) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    float total = 0.0f;
    for (int b = 0; b < bands; ++b) total += partial[(long long)b * cols + c];
    out[c] = total;
}

__global__ void __launch_bounds__(kThreads) block_tops_kernel(const float* __restrict__ scales, int rows, float* __restrict__ top) {
    __shared__ float s_max[kThreads / 32];
    float m = 0.0f;
    for (int r = threadIdx.x; r < rows; r += kThreads) m = fmaxf(m, finite_abs(__ldg(scales + (long long)blockIdx.x * rows + r)));
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, s_max[w]);
    if (threadIdx.x == 0) top[blockIdx.x] = m > 0.0f ? m : 1.0f;
}

// Eight elements per thread, zeros behind cols up to the next multiple of eight.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) dequantize_rows_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scales,
                                                                   const float* __restrict__ top, int rows, int cols,
                                                                   T* __restrict__ y, long long ld_y) {
    const int units = (cols + 7) / 8;
    const long long total = (long long)rows * units;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / units;
        const int c0 = int(i - r * units) * 8;
        const int b = c0 / FP8_BLOCK;
        float s = __ldg(scales + (long long)b * rows + r);
        if (top != nullptr) s /= __ldg(top + b);
        uint8_t v[8];
        if (VEC) {
            *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(q + r * cols + c0));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c0 + j < cols ? q[r * cols + c0 + j] : uint8_t(0);
        }
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = e4m3_value(v[j]) * s;
        store8(y + r * ld_y + c0, f);
    }
}

template <typename T>
void act_backward_typed(const T* dy, const uint8_t* z8, const float* z_scales, int act, T* dz, long long ld_dz, float* db,
                        int rows, int cols, cudaStream_t stream) {
    const bool vec = cols % 8 == 0 && reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(z8) % 8 == 0;
    const int rows_per = rows > 2048 ? 128 : 32;
    const int bands = (rows + rows_per - 1) / rows_per;
    CB200_REQUIRE(bands <= 65535, "too many rows");
    Scratch partial;
    float* to = db;
    if (db != nullptr && bands > 1) {
        partial = Scratch(size_t(bands) * cols * sizeof(float), stream);
        to = static_cast<float*>(partial.ptr);
    }
    const dim3 grid((cols + 255) / 256, bands);
    if (vec) act_backward_kernel<T, true><<<grid, kThreads, 0, stream>>>(dy, z8, z_scales, act, dz, ld_dz, to, rows, cols, rows_per);
    else act_backward_kernel<T, false><<<grid, kThreads, 0, stream>>>(dy, z8, z_scales, act, dz, ld_dz, to, rows, cols, rows_per);
    CB200_CHECK_LAUNCH();
    if (to != db) {
        add_bands_kernel<<<(cols + kThreads - 1) / kThreads, kThreads, 0, stream>>>(to, bands, cols, db);
        CB200_CHECK_LAUNCH();
    }
}

unsigned pass_grid(long long items) {
    const long long most = 16ll * device_info().num_sms;
    const long long want = (items + kThreads - 1) / kThreads;
    return unsigned(want < most ? want : most);
}

template <typename T>
void quantize_typed(const T* x, long long rows, int cols, int block_rows, uint8_t* q, float* scales, cudaStream_t stream) {
    const bool vec = cols % 8 == 0 && (cols * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % 8 == 0;
    const unsigned blocks = unsigned((cols + FP8_BLOCK - 1) / FP8_BLOCK);
    const int rows_per = block_rows == 1 ? 32 : FP8_BLOCK;
    // gridDim.y holds 65535: more rows go in bands (their scales are addressed from the whole matrix's first row).
    CB200_REQUIRE((rows + rows_per - 1) / rows_per <= 65535, "quantize_fp8: too many rows");
    const unsigned bands = unsigned((rows + rows_per - 1) / rows_per);
    if (block_rows == 1) {
        const dim3 grid((blocks + 1) / 2, bands);
        if (vec) quantize_rows_kernel<T, true><<<grid, kThreads, 0, stream>>>(x, rows, cols, q, scales);
        else quantize_rows_kernel<T, false><<<grid, kThreads, 0, stream>>>(x, rows, cols, q, scales);
    } else {
        const dim3 grid(blocks, bands);
        if (vec) quantize_tiles_kernel<T, true><<<grid, kThreads, 0, stream>>>(x, rows, cols, q, scales);
        else quantize_tiles_kernel<T, false><<<grid, kThreads, 0, stream>>>(x, rows, cols, q, scales);
    }
    CB200_CHECK_LAUNCH();
}

}  // namespace

AlignedRows aligned_rows(const void* src, long long rows, int cols, int elem_size, cudaStream_t stream) {
    AlignedRows out;
    const int per_unit = 16 / elem_size;
    if (cols % per_unit == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0) {
        out.ptr = src;
        out.ld = cols;
        return out;
    }
    const int units = (cols + per_unit - 1) / per_unit;
    out.ld = (long long)units * per_unit;
    out.copy = Scratch(size_t(rows) * units * 16, stream);
    out.ptr = out.copy.ptr;
    if (elem_size == 1)
        pad_rows_kernel<uint8_t><<<pass_grid(rows * units), kThreads, 0, stream>>>(
            static_cast<const uint8_t*>(src), static_cast<uint8_t*>(out.copy.ptr), rows, cols, units);
    else
        pad_rows_kernel<uint16_t><<<pass_grid(rows * units), kThreads, 0, stream>>>(
            static_cast<const uint16_t*>(src), static_cast<uint16_t*>(out.copy.ptr), rows, cols, units);
    CB200_CHECK_LAUNCH();
    return out;
}

void quantize_fp8(const void* x, int x_type, long long rows, int cols, int block_rows, uint8_t* q, float* scales,
                  cudaStream_t stream) {
    if (x_type == TYPE_F32) quantize_typed(static_cast<const float*>(x), rows, cols, block_rows, q, scales, stream);
    else if (x_type == TYPE_F16) quantize_typed(static_cast<const __half*>(x), rows, cols, block_rows, q, scales, stream);
    else quantize_typed(static_cast<const __nv_bfloat16*>(x), rows, cols, block_rows, q, scales, stream);
}

void dequantize_fp8(const uint8_t* q, const float* scales, long long rows, int cols, int block_rows, void* y, int y_type,
                    cudaStream_t stream) {
    const unsigned grid = pass_grid(rows * cols);
    if (y_type == TYPE_F32)
        dequantize_kernel<<<grid, kThreads, 0, stream>>>(q, scales, rows, cols, block_rows, static_cast<float*>(y));
    else if (y_type == TYPE_F16)
        dequantize_kernel<<<grid, kThreads, 0, stream>>>(q, scales, rows, cols, block_rows, static_cast<__half*>(y));
    else
        dequantize_kernel<<<grid, kThreads, 0, stream>>>(q, scales, rows, cols, block_rows, static_cast<__nv_bfloat16*>(y));
    CB200_CHECK_LAUNCH();
}

void activation_backward_fp8(const void* dy, int type, const uint8_t* z8, const float* z_scales, int act, void* dz,
                             long long ld_dz, float* db, int rows, int cols, cudaStream_t stream) {
    if (type == TYPE_F16)
        act_backward_typed(static_cast<const __half*>(dy), z8, z_scales, act, static_cast<__half*>(dz), ld_dz, db, rows, cols,
                           stream);
    else
        act_backward_typed(static_cast<const __nv_bfloat16*>(dy), z8, z_scales, act, static_cast<__nv_bfloat16*>(dz), ld_dz, db,
                           rows, cols, stream);
}

void block_tops(const float* scales, int rows, int cols, float* top, cudaStream_t stream) {
    block_tops_kernel<<<(cols + FP8_BLOCK - 1) / FP8_BLOCK, kThreads, 0, stream>>>(scales, rows, top);
    CB200_CHECK_LAUNCH();
}

void dequantize_rows(const uint8_t* q, const float* scales, const float* top, int rows, int cols, void* y, long long ld_y,
                     int y_type, cudaStream_t stream) {
    const bool vec = cols % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
    const unsigned grid = pass_grid((long long)rows * ((cols + 7) / 8));
    if (y_type == TYPE_F16) {
        __half* out = static_cast<__half*>(y);
        if (vec) dequantize_rows_kernel<__half, true><<<grid, kThreads, 0, stream>>>(q, scales, top, rows, cols, out, ld_y);
        else dequantize_rows_kernel<__half, false><<<grid, kThreads, 0, stream>>>(q, scales, top, rows, cols, out, ld_y);
    } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(y);
        if (vec) dequantize_rows_kernel<__nv_bfloat16, true><<<grid, kThreads, 0, stream>>>(q, scales, top, rows, cols, out, ld_y);
        else dequantize_rows_kernel<__nv_bfloat16, false><<<grid, kThreads, 0, stream>>>(q, scales, top, rows, cols, out, ld_y);
    }
    CB200_CHECK_LAUNCH();
}

}  // namespace cudeep_b200
