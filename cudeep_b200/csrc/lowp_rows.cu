// One-pass kernels around the 8-bit and the grouped products: padding of rows for the TMA unit, quantisation to e4m3
// in blocks and back.  All are bound by HBM: each input is read once and each output written once.
//
// Each kernel waits for its predecessors itself and then lets its successor be set up, so that in a sequence of small
// launches (the backward pass of a short batch is five) the launches overlap.
#include "lowp_rows.h"

#include "device_flags.cuh"
#include "epilogue_math.cuh"
#include "launch_dependent.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

namespace cudeep_b200 {

namespace {

constexpr int kThreads = 256;

// The work of a CTA in prepare_kernel for one matrix to pad.
struct PadJob {
    const uint8_t* src;
    uint8_t* dst;
    long long rows;
    int row_bytes, ld;
    const int32_t* offsets;
    int rows_group;
    unsigned chunks;      // of 512 bytes, in a row of the result
    unsigned blocks;      // CTAs
};

// dst[r, 0..ld) = src[r, 0..row_bytes) followed by zeros, in bytes; ld is a multiple of 16 and dst aligned to it.  A warp
// takes 512 bytes of a row, a lane every 32nd word of the result, shifted together from the two aligned words of the source
// that hold it (loads byte by byte ran at 2 TB/s, 16 bytes a lane at a quarter of the requests' width).  Words that reach
// over the matrix's ends are put together from bytes.  With offsets, rows_group rows belong to each group, and those of
// groups without rows in their turn (the weights of experts that have no token) are left out.
__device__ __forceinline__ void pad_rows(const PadJob& job, unsigned block) {
    const uint8_t* __restrict__ src = job.src;
    uint8_t* __restrict__ dst = job.dst;
    const long long rows = job.rows;
    const int row_bytes = job.row_bytes, ld = job.ld;
    const int lane = threadIdx.x & 31;
    const long long r = block / job.chunks * (long long)(kThreads / 32) + (threadIdx.x >> 5);
    if (r >= rows) return;
    if (job.offsets != nullptr) {
        const int g = rows <= 0x7fffffff ? int(unsigned(r) / unsigned(job.rows_group)) : int(r / job.rows_group);
        if (__ldg(job.offsets + g + 1) <= __ldg(job.offsets + g)) return;
    }
    const uint8_t* row = src + r * row_bytes;
    const uint8_t* end = src + rows * row_bytes;
    const int shift = int(reinterpret_cast<uintptr_t>(row) & 3u);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(row - shift);
    uint32_t* out = reinterpret_cast<uint32_t*>(dst + r * ld);
    const int count = ld / 4;
    // Words that hold bytes outside the matrix (its first, its last) are put together from bytes.
    const int last = (row_bytes + shift - 1) / 4;      // word of the row's last byte
    const int from = row - shift >= src ? 0 : 1;
    const int to = row - shift + 4 * last + 4 <= end ? last : last - 1;
    auto word_of_bytes = [&](int w) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 4 * w + i - shift;
            if (at >= 0 && at < row_bytes) v |= uint32_t(row[at]) << (8 * i);
        }
        return v;
    };
    const int w0 = int(block % job.chunks) * 128;
    uint32_t lo[4], hi[4];
    if (from <= to) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int w = w0 + lane + 32 * j;
            lo[j] = __ldg(words + max(from, min(w, to)));
            hi[j] = __ldg(words + max(from, min(w + 1, to)));
        }
    }
    if (from != 0 || to != last) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int w = w0 + lane + 32 * j;
            if (w < from || w > to) lo[j] = word_of_bytes(w);
            if (w + 1 < from || w + 1 > to) hi[j] = word_of_bytes(w + 1);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int w = w0 + lane + 32 * j;
        if (w >= count) break;
        const int left = row_bytes - 4 * w;      // bytes of the row from this word on
        uint32_t v = __funnelshift_r(lo[j], hi[j], 8 * shift);
        if (left < 4) v = left <= 0 ? 0u : v & (0xffffffffu >> (8 * (4 - left)));
        out[w] = v;
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

// 16 bytes of input: 4 floats or 8 16-bit values.  The block's maximum is found on the bits of the magnitudes, which order as
// the magnitudes do with infinities and NaN on top: two instructions per word and no conversion.  A block that holds
// something that is not finite shows it by a maximum beyond the largest finite value and takes the long way.
template <typename T>
struct Unit {
    static constexpr int N = 16 / int(sizeof(T));
    uint4 w;
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
    __device__ __forceinline__ float value(int j) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(word(j));
        } else {
            const uint16_t h = uint16_t(word(j / 2) >> (16 * (j & 1)));
            return to_float(*reinterpret_cast<const T*>(&h));
        }
    }
    __device__ __forceinline__ uint32_t top(uint32_t m) const {      // packed for 16-bit types
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, word(i) & 0x7fffffffu);
            else m = __vmaxu2(m, word(i) & 0x7fff7fffu);
        }
        return m;
    }
};
// Magnitude bits of one value as top() packs them, and back to one value.
template <typename T>
__device__ __forceinline__ uint32_t unpack_top(uint32_t m) {
    return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
}
template <typename T>
__device__ __forceinline__ float top_value(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    const uint16_t h = uint16_t(bits);
    return to_float(*reinterpret_cast<const T*>(&h));
}
template <typename T>
__device__ __forceinline__ bool top_finite(uint32_t bits) {
    return bits < (sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
}

// Four values times the inverse of the scale (exact: a power of two) in e4m3, rounded to nearest even once.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float inv) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inv, d * inv), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
// NaN's code where a value is not finite.
__device__ __forceinline__ uint32_t nan_codes(uint32_t q, float a, float b, float c, float d) {
    const float v[4] = {a, b, c, d};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (!(fabsf(v[j]) <= 3.402823466e38f)) q = (q & ~(0xffu << (8 * j))) | 0x7fu << (8 * j);
    return q;
}

// A row's 128 elements of a block that start anywhere, across a warp: a lane takes every 32nd, so that loads and byte stores
// are contiguous across the lanes.  Loads are not conditional: lanes behind the row's end read its last element and drop it
// (a branch around each load kept the loads of a block from being under way together: 4100 x 11007 FP32 78 us instead of
// 50 us; four neighbouring elements a lane, to store their codes as a word, were four times as many requests to L1: 100 us).
struct RowSlice {
    float v[4];
    // The first `width` (1 to 128) elements of the block; zeros for a row that is not there (src then is some row that is).
    template <typename T>
    __device__ __forceinline__ void load(const T* src, int width, bool there, int lane) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_float(src[min(lane + 32 * j, width - 1)]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!there || lane + 32 * j >= width) v[j] = 0.0f;
    }
    __device__ __forceinline__ uint32_t top(uint32_t m) const {      // as Unit::top
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ float finite_top(float amax) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, finite_abs(v[j]));
        return amax;
    }
    __device__ __forceinline__ void store(uint8_t* dst, int width, int lane, float inv, bool finite) const {
        uint32_t codes = e4m3x4(v[0], v[1], v[2], v[3], inv);
        if (!finite) codes = nan_codes(codes, v[0], v[1], v[2], v[3]);
        if (width == FP8_BLOCK) {
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[lane + 32 * j] = uint8_t(codes >> (8 * j));
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < width) dst[lane + 32 * j] = uint8_t(codes >> (8 * j));
    }
};

// Blocks of 1 x 128.  Eight lanes own a block, 16 elements each in units of 16 bytes; a warp takes four neighbouring blocks of
// four rows, so a lane has 8 (16-bit types) or 16 independent loads under way, and a CTA 32 rows x 512 columns.  The
// scales lie [block][row], so the CTA collects its 32 x 4 scales in shared memory and writes runs of 32.
// 8192 x 16384 BF16, 407 MB: 61 us.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                 int grid_cols, uint8_t* __restrict__ q, float* __restrict__ scales) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int bx = int(blockIdx.x % unsigned(grid_cols)), by = int(blockIdx.x / unsigned(grid_cols));
    constexpr int N = Unit<T>::N, UNITS = 16 / N;
    __shared__ float s_scale[4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane >> 3, l8 = lane & 7;
    const int block = bx * 4 + sub;
    const int c0 = block * FP8_BLOCK + l8 * N;      // and 8 * N further on for each unit
    const long long row0 = (long long)by * 32 + warp * 4;
    Unit<T> u[4][UNITS];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int k = 0; k < UNITS; ++k) {
            const int c = c0 + 8 * N * k;
            u[i][k].w = make_uint4(0, 0, 0, 0);
            if (row0 + i < rows && c < cols) u[i][k].w = __ldg(reinterpret_cast<const uint4*>(x + (row0 + i) * cols + c));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < UNITS; ++k) m = u[i][k].top(m);
        m = unpack_top<T>(m);
#pragma unroll
        for (int d = 4; d >= 1; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        const bool finite = top_finite<T>(m);
        float amax = top_value<T>(m);
        if (__any_sync(0xffffffffu, !finite)) {
            amax = 0.0f;
#pragma unroll
            for (int k = 0; k < UNITS; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) amax = fmaxf(amax, finite_abs(u[i][k].value(j)));
#pragma unroll
            for (int d = 4; d >= 1; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        }
        const int e = scale_exponent(amax);
        const float inv = pow2(-e);
        if (l8 == 0) s_scale[sub][warp * 4 + i] = pow2(e);
        if (row0 + i < rows) {
            uint8_t* dst = q + (row0 + i) * cols + c0;
#pragma unroll
            for (int k = 0; k < UNITS; ++k) {
                if (c0 + 8 * N * k >= cols) break;
                uint32_t out[N / 4];
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    const Unit<T>& v = u[i][k];
                    out[j / 4] = e4m3x4(v.value(j), v.value(j + 1), v.value(j + 2), v.value(j + 3), inv);
                    if (!finite) out[j / 4] = nan_codes(out[j / 4], v.value(j), v.value(j + 1), v.value(j + 2), v.value(j + 3));
                }
                if constexpr (N == 8) *reinterpret_cast<uint2*>(dst + 8 * N * k) = make_uint2(out[0], out[1]);
                else *reinterpret_cast<uint32_t*>(dst + 8 * N * k) = out[0];
            }
        }
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        const long long r = (long long)by * 32 + lane;
        const int blk = bx * 4 + warp;
        if (r < rows && (long long)blk * FP8_BLOCK < cols) scales[(long long)blk * rows + r] = s_scale[warp][lane];
    }
}

// The same for rows that start anywhere: a warp takes four rows of a block at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_rows_any_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                     int grid_cols, uint8_t* __restrict__ q, float* __restrict__ scales) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int bx = int(blockIdx.x % unsigned(grid_cols)), by = int(blockIdx.x / unsigned(grid_cols));
    __shared__ float s_scale[4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row0 = (long long)by * 32 + warp * 4;
#pragma unroll 1
    for (int b = 0; b < 4; ++b) {
        const int c0 = (bx * 4 + b) * FP8_BLOCK;
        if (c0 >= cols) break;
        const int width = min(FP8_BLOCK, cols - c0);
        RowSlice slice[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            slice[i].load(x + min(row0 + i, rows - 1) * cols + c0, width, row0 + i < rows, lane);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = __reduce_max_sync(0xffffffffu, slice[i].top(0));
            const bool finite = top_finite<float>(m);
            if (!finite) m = __reduce_max_sync(0xffffffffu, __float_as_uint(slice[i].finite_top(0.0f)));
            const int e = scale_exponent(__uint_as_float(m));
            if (lane == 0) s_scale[b][warp * 4 + i] = pow2(e);
            const long long at = (row0 + i) * cols + c0;
            if (row0 + i < rows) slice[i].store(q + at, width, lane, pow2(-e), finite);
        }
    }
    __syncthreads();
    if (threadIdx.x < 128) {
        const long long r = (long long)by * 32 + lane;
        const int blk = bx * 4 + warp;
        if (r < rows && (long long)blk * FP8_BLOCK < cols) scales[(long long)blk * rows + r] = s_scale[warp][lane];
    }
}

// Blocks of 128 x 128, one CTA each, held in registers while the block's maximum is found: eight lanes along a row of the
// block, 32 rows at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_tiles_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                  int grid_cols, uint8_t* __restrict__ q, float* __restrict__ scales) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int bx = int(blockIdx.x % unsigned(grid_cols)), by = int(blockIdx.x / unsigned(grid_cols));
    constexpr int N = Unit<T>::N, UNITS = 16 / N;
    __shared__ float s_max[kThreads / 32];
    __shared__ uint32_t s_top[kThreads / 32];
    const int l8 = threadIdx.x & 7;
    const int c0 = bx * FP8_BLOCK + l8 * N;
    const long long row0 = (long long)by * FP8_BLOCK + (threadIdx.x >> 3);
    Unit<T> u[4][UNITS];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < UNITS; ++k) {
            const long long r = row0 + 32 * i;
            const int c = c0 + 8 * N * k;
            u[i][k].w = make_uint4(0, 0, 0, 0);
            if (r < rows && c < cols) u[i][k].w = __ldg(reinterpret_cast<const uint4*>(x + r * cols + c));
        }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < UNITS; ++k) m = u[i][k].top(m);
    m = __reduce_max_sync(0xffffffffu, unpack_top<T>(m));
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, s_top[w]);
    const bool finite = top_finite<T>(m);      // the same for the whole CTA
    float amax = top_value<T>(m);
    if (!finite) {
        amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int k = 0; k < UNITS; ++k)
#pragma unroll
                for (int j = 0; j < N; ++j) amax = fmaxf(amax, finite_abs(u[i][k].value(j)));
        amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) amax = fmaxf(amax, s_max[w]);
    }
    const int e = scale_exponent(amax);
    const float inv = pow2(-e);
    if (threadIdx.x == 0) scales[(long long)by * grid_cols + bx] = pow2(e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = row0 + 32 * i;
        if (r >= rows) break;
        uint8_t* dst = q + r * cols + c0;
#pragma unroll
        for (int k = 0; k < UNITS; ++k) {
            if (c0 + 8 * N * k >= cols) break;
            uint32_t out[N / 4];
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const Unit<T>& v = u[i][k];
                out[j / 4] = e4m3x4(v.value(j), v.value(j + 1), v.value(j + 2), v.value(j + 3), inv);
                if (!finite) out[j / 4] = nan_codes(out[j / 4], v.value(j), v.value(j + 1), v.value(j + 2), v.value(j + 3));
            }
            if constexpr (N == 8) *reinterpret_cast<uint2*>(dst + 8 * N * k) = make_uint2(out[0], out[1]);
            else *reinterpret_cast<uint32_t*>(dst + 8 * N * k) = out[0];
        }
    }
}

// The same for rows that start anywhere: a warp holds eight rows.  4100 x 11007 FP32, 226 MB: 50 us.
constexpr int kTileThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kTileThreads) quantize_tiles_any_kernel(const T* __restrict__ x, long long rows, int cols,
                                                                          int grid_cols, uint8_t* __restrict__ q, float* __restrict__ scales) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int bx = int(blockIdx.x % unsigned(grid_cols)), by = int(blockIdx.x / unsigned(grid_cols));
    __shared__ uint32_t s_top[kTileThreads / 32], s_finite_top[kTileThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c0 = bx * FP8_BLOCK;
    const int width = min(FP8_BLOCK, cols - c0);
    const long long row0 = (long long)by * FP8_BLOCK + warp * 8;
    RowSlice slice[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        slice[i].load(x + min(row0 + i, rows - 1) * cols + c0, width, row0 + i < rows, lane);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = slice[i].top(m);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_top[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kTileThreads / 32; ++w) m = max(m, s_top[w]);
    const bool finite = top_finite<float>(m);      // the same for the whole CTA
    if (!finite) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = slice[i].finite_top(amax);
        m = __reduce_max_sync(0xffffffffu, __float_as_uint(amax));
        if (lane == 0) s_finite_top[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTileThreads / 32; ++w) m = max(m, s_finite_top[w]);
    }
    const int e = scale_exponent(__uint_as_float(m));
    const float inv = pow2(-e);
    if (threadIdx.x == 0) scales[(long long)by * grid_cols + bx] = pow2(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long at = (row0 + i) * cols + c0;
        if (row0 + i < rows) slice[i].store(q + at, width, lane, inv, finite);
    }
}

__device__ __forceinline__ float e4m3_value(uint8_t q) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

// Eight of them, as they lie in memory.
__device__ __forceinline__ void e4m3_values(uint2 q, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t word = i < 2 ? q.x : q.y;
        const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t((word >> (16 * (i & 1))) & 0xffffu), __NV_E4M3));
        const float2 f = __half22float2(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Eight 16-bit values of a row from column c0 on; zeros behind cols.
template <typename T>
struct Unit8 {
    uint4 w;
    template <bool VEC>
    __device__ __forceinline__ void load(const T* row, int c0, int cols) {
        if (VEC) {
            w = __ldg(reinterpret_cast<const uint4*>(row + c0));
        } else {
            alignas(16) T t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t[j] = row[min(c0 + j, cols - 1)];
                if (c0 + j >= cols) t[j] = from_float<T>(0.0f);
            }
            w = *reinterpret_cast<const uint4*>(t);
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float(t[j]);
    }
};

// Eight codes of a row from column c0 on; zeros behind cols.
template <bool VEC>
__device__ __forceinline__ uint2 load_codes(const uint8_t* row, int c0, int cols) {
    if (VEC) return __ldg(reinterpret_cast<const uint2*>(row + c0));
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t code = row[min(c0 + j, cols - 1)];
        w[j / 4] |= (c0 + j < cols ? code : 0u) << (8 * (j % 4));
    }
    return make_uint2(w[0], w[1]);
}

template <typename T>
__global__ void dequantize_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scales, long long rows, int cols,
                                  int block_rows, T* __restrict__ y) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int col_blocks = (cols + FP8_BLOCK - 1) / FP8_BLOCK;
    const long long total = rows * cols;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / cols;
        const int b = int(i - r * cols) / FP8_BLOCK;
        const float s = __ldg(scales + (block_rows == 1 ? b * rows + r : (r / FP8_BLOCK) * col_blocks + b));
        y[i] = from_float<T>(e4m3_value(q[i]) * s);
    }
}

// Slope of the epilogue activations.  With s = sigmoid(t), t = 2 sqrt(2 / pi) (z + 0.044715 z^3): tanh-form GELU is z s, so its
// slope is s + z s (1 - s) dt/dz; SiLU the same with t = z.  s comes from the SFU's ex2 and rcp as in the forward epilogue
// (2 ulp; with expf and tanhf the pass was bound by arithmetic, 68 us for 8192 x 4096 instead of 34 us with the bands' sums).
template <int act>
__device__ __forceinline__ float act_slope(float z) {
    if (act == EPI_RELU) return z > 0.0f ? 1.0f : 0.0f;
    // At these bounds e reaches 2^126, so s (or 1 - s) FP32's least normal number, 2^-126; beyond them the slope differs from 0 or
    // 1 by no more than that times z dt/dz.  Inside them no power of z and no exponential overflows.
    constexpr float bound = act == EPI_GELU ? 10.0f : 87.33f;
    constexpr float a = act == EPI_GELU ? 2.0f * 0.7978845608028654f : 1.0f;
    constexpr float b = act == EPI_GELU ? a * 0.044715f : 0.0f;
    constexpr float log2e = 1.4426950408889634f;
    z = clamp_nan(z, -bound, bound);
    const float z2 = z * z;
    const float e = sfu_ex2(z * fmaf(-log2e * b, z2, -log2e * a));
    const float s = sfu_rcp(1.0f + e);
    const float rest = e * s;                                   // 1 - s without cancellation
    if (act == EPI_SIGMOID) return s * rest;
    return fmaf(z * rest * fmaf(3.0f * b, z2, a), s, s);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    alignas(16) T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_float<T>(v[j]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(t);
}

// A CTA takes 256 columns and `rows_per` rows: 32 threads with eight columns each lie along a row, eight rows side by side.
// Column sums stay in registers over the rows, are added across the eight threads of a column in a fixed order and go to
// partial[row band][cols], which one more kernel adds up, again in order: the result does not depend on timing.
template <typename T, bool VEC, int act>
__global__ void __launch_bounds__(kThreads) act_backward_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ z8,
                                                                const float* __restrict__ zs, T* __restrict__ dz,
                                                                long long ld_dz, float* __restrict__ partial, int rows, int cols,
                                                                int rows_per) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    __shared__ float s_sum[8][264];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c0 = blockIdx.x * 256 + tx * 8;
    const int r_end = min(rows, int(blockIdx.y + 1) * rows_per);
    float sum[8] = {};
    if (c0 < cols) {
        const float* s_col = zs + (long long)(c0 / FP8_BLOCK) * rows;
        // Four rows at a time, their loads under way together (rows behind the band read its last one).
        for (int r0 = blockIdx.y * rows_per + ty; r0 < r_end; r0 += 32) {
            Unit8<T> g8[4];
            uint2 z8s[4];
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = min(r0 + 8 * i, r_end - 1);
                g8[i].template load<VEC>(dy + (long long)r * cols, c0, cols);
                if (act != EPI_NONE) {
                    z8s[i] = load_codes<VEC>(z8 + (long long)r * cols, c0, cols);
                    s[i] = __ldg(s_col + r);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = r0 + 8 * i;
                if (r >= r_end) break;
                float g[8];
                g8[i].values(g);
                if (act != EPI_NONE) {
                    float z[8];
                    e4m3_values(z8s[i], z);
#pragma unroll
                    for (int j = 0; j < 8; ++j)      // rounded before the sum, whether dz is stored or not
                        g[j] = __fmul_rn(g[j], act_slope<act>(z[j] * s[i]));
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

// Column sums that still lie in bands of rows.
struct Bands {
    const float* partial;      // [bands][cols]
    int bands, cols;
    float* out;
    unsigned blocks;           // CTAs: one for 32 columns
};

// A CTA takes 32 columns, its eight warps every eighth band each; their sums are added in warp order.
__device__ __forceinline__ void add_bands(const Bands& p, unsigned block) {
    __shared__ float s_sum[8][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int c = int(block) * 32 + lane;
    float total = 0.0f;
    if (c < p.cols) {
#pragma unroll 4
        for (int b = warp; b < p.bands; b += 8) total += p.partial[(long long)b * p.cols + c];
    }
    s_sum[warp][lane] = total;
    __syncthreads();
    if (warp == 0 && c < p.cols) {
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) total += s_sum[i][lane];
        p.out[c] = total;
    }
}

__global__ void __launch_bounds__(kThreads) add_bands_kernel(const __grid_constant__ Bands p) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    add_bands(p, blockIdx.x);
}

// FP16 reaches from 448 * 2^0 down to steps of 2^-24, and e4m3's steps are 2^-9 of a scale: scales down to 2^-15 of the block's
// largest one fit.  Zero scales stand for zeros and do not count.  (A block of zeros has the scale 1, which counts: its codes
// are not looked at here.)
__device__ __forceinline__ void block_top(const float* __restrict__ scales, int rows, float* __restrict__ top,
                                          uint32_t* __restrict__ wide, unsigned block) {
    __shared__ float s_max[kThreads / 32], s_min[kThreads / 32];
    float m = 0.0f, least = __int_as_float(0x7f800000);
#pragma unroll 8
    for (int r = threadIdx.x; r < rows; r += kThreads) {
        const float s = finite_abs(__ldg(scales + (long long)block * rows + r));
        m = fmaxf(m, s);
        least = fminf(least, s > 0.0f ? s : __int_as_float(0x7f800000));
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, d));
    }
    if ((threadIdx.x & 31) == 0) {
        s_max[threadIdx.x >> 5] = m;
        s_min[threadIdx.x >> 5] = least;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        m = fmaxf(m, s_max[w]);
        least = fminf(least, s_min[w]);
    }
    if (threadIdx.x == 0) {
        top[block] = m > 0.0f ? m : 1.0f;
        wide[block] = least * 32768.0f < m ? 1u : 0u;
    }
}

// What a product needs before it, in one launch: each launch costs the host about 2 us, more than a small one of these takes
// (a grouped product of 64 rows with both operands to pad occupies the host for 11.6 us with a launch for each and 8.7 us so).
struct PrepareParams {
    PadJob pad[2];
    const float* scales;
    int scale_rows;
    float* top;
    uint32_t* wide;
};
__global__ void __launch_bounds__(kThreads) prepare_kernel(const __grid_constant__ PrepareParams p) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    unsigned block = blockIdx.x;
    if (block < p.pad[0].blocks) return pad_rows(p.pad[0], block);
    block -= p.pad[0].blocks;
    if (block < p.pad[1].blocks) return pad_rows(p.pad[1], block);
    block_top(p.scales, p.scale_rows, p.top, p.wide, block - p.pad[1].blocks);
}

// What dequantize_rows_kernel heeds for FP16.
struct WideRows {
    const float* top;           // nullptr for BF16
    const uint32_t* wide;       // [blocks]
    int blocks;
    const __half* split;        // a matrix to split (SplitRequest)
    long long ld_split, ld_parts;
    int split_cols;
    __nv_bfloat16* parts;
};

// Eight elements per thread, zeros behind cols up to the next multiple of eight; CTA `block` of `blocks`.
template <typename T, bool VEC>
__device__ __forceinline__ void dequantize_units(const uint8_t* __restrict__ q, const float* __restrict__ scales,
                                                 const float* __restrict__ top, int rows, int cols, T* __restrict__ y,
                                                 long long ld_y, unsigned block, unsigned blocks) {
    const int units = (cols + 7) / 8;
    const long long total = (long long)rows * units;
    for (long long i = block * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)blocks * blockDim.x) {
        const long long r = i / units;
        const int c0 = int(i - r * units) * 8;
        const int b = c0 / FP8_BLOCK;
        float s = __ldg(scales + (long long)b * rows + r);
        if (top != nullptr) s /= __ldg(top + b);
        float f[8];
        e4m3_values(load_codes<VEC>(q + r * cols, c0, cols), f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= s;
        store8(y + r * ld_y + c0, f);
    }
}

// The first CTAs add up column sums instead, of the pass before it (a launch less).  One load of codes a thread is under way, so
// that the pass lives on eight CTAs to an SM.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 8) dequantize_rows_kernel(const uint8_t* __restrict__ q, const float* __restrict__ scales,
                                                                   int rows, int cols, T* __restrict__ y, long long ld_y,
                                                                   const __grid_constant__ Bands sums,
                                                                   const __grid_constant__ WideRows w) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    if (blockIdx.x < sums.blocks) return add_bands(sums, blockIdx.x);
    const unsigned block = blockIdx.x - sums.blocks, blocks = gridDim.x - sums.blocks;
    if constexpr (std::is_same<T, __half>::value) {
        if (any_set(w.wide, w.blocks)) {
            dequantize_units<__nv_bfloat16, VEC>(q, scales, nullptr, rows, cols, reinterpret_cast<__nv_bfloat16*>(y), ld_y, block,
                                                 blocks);
            const int units = (w.split_cols + 7) / 8;
            const long long total = (long long)rows * units;
            for (long long i = block * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)blocks * blockDim.x) {
                const long long r = i / units;
                const int c0 = int(i - r * units) * 8;
                Unit8<__half> u;
                u.template load<true>(w.split + r * w.ld_split, c0, w.split_cols);
                float v[8], rest[8];
                u.values(v);
#pragma unroll
                for (int j = 0; j < 8; ++j)      // an infinity or NaN goes whole into the first part
                    rest[j] = fabsf(v[j]) <= 65504.0f ? v[j] - __bfloat162float(__float2bfloat16_rn(v[j])) : 0.0f;
                store8(w.parts + r * w.ld_parts + c0, v);
                store8(w.parts + (rows + r) * w.ld_parts + c0, rest);
            }
            return;
        }
    }
    dequantize_units<T, VEC>(q, scales, w.top, rows, cols, y, ld_y, block, blocks);
}

template <typename T>
ColumnSums act_backward_typed(const T* dy, const uint8_t* z8, const float* z_scales, int act, T* dz, long long ld_dz, float* db,
                              int rows, int cols, cudaStream_t stream) {
    const bool vec = cols % 8 == 0 && reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(z8) % 8 == 0;
    // Bands of the grid's second dimension (at most 65535); 64 rows keep the last wave of CTAs full for large matrices.
    const int least = (rows / 65535 + 32) / 32 * 32;
    const int rows_per = std::max(rows > 4096 ? 64 : 32, least);
    const int bands = (rows + rows_per - 1) / rows_per;
    ColumnSums sums;
    float* to = db;
    if (db != nullptr && bands > 1) {
        sums.partial = Scratch(size_t(bands) * cols * sizeof(float), stream);
        sums.bands = bands;
        sums.cols = cols;
        sums.out = db;
        to = static_cast<float*>(sums.partial.ptr);
    }
    const dim3 grid((cols + 255) / 256, bands);
    auto launch = [&](auto code) {
        constexpr int A = decltype(code)::value;
        if (vec) launch_dependent(act_backward_kernel<T, true, A>, dim3(grid), kThreads, stream, dy, z8, z_scales, dz, ld_dz, to, rows, cols, rows_per);
        else launch_dependent(act_backward_kernel<T, false, A>, dim3(grid), kThreads, stream, dy, z8, z_scales, dz, ld_dz, to, rows, cols, rows_per);
    };
    if (act == EPI_RELU) launch(std::integral_constant<int, EPI_RELU>{});
    else if (act == EPI_GELU) launch(std::integral_constant<int, EPI_GELU>{});
    else if (act == EPI_SILU) launch(std::integral_constant<int, EPI_SILU>{});
    else if (act == EPI_SIGMOID) launch(std::integral_constant<int, EPI_SIGMOID>{});
    else launch(std::integral_constant<int, EPI_NONE>{});
    CB200_CHECK_LAUNCH();
    return sums;
}

// The part of a pass over `sums`; none without any.
Bands bands_of(const ColumnSums& sums) {
    Bands p{};
    p.partial = static_cast<const float*>(sums.partial.ptr);
    p.bands = sums.bands;
    p.cols = sums.cols;
    p.out = sums.out;
    p.blocks = sums.out != nullptr ? unsigned((sums.cols + 31) / 32) : 0u;
    return p;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) add_parts_kernel(const float* __restrict__ part, int parts, int m, int n, long long ld,
                                                             T* __restrict__ out) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const long long units = ld / 4, total = m * units;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        float4 sum = __ldg(reinterpret_cast<const float4*>(part) + i);
        for (int p = 1; p < parts; ++p) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(part) + p * total + i);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        const long long r = i / units;
        const int c = int(i - r * units) * 4;
        T* dst = out + r * n + c;
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < n) dst[j] = from_float<T>(v[j]);
    }
}

template <typename S, typename D>
__global__ void __launch_bounds__(kThreads) cast_kernel(const S* __restrict__ src, D* __restrict__ dst, long long count) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
#pragma unroll 4
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < count; i += (long long)gridDim.x * blockDim.x)
        dst[i] = from_float<D>(to_float(src[i]));
}

unsigned pass_grid(long long items) {
    const long long most = 16ll * device_info().num_sms;
    const long long want = (items + kThreads - 1) / kThreads;
    return unsigned(want < most ? want : most);
}

template <typename T>
void quantize_typed(const T* x, long long rows, int cols, int block_rows, uint8_t* q, float* scales, cudaStream_t stream) {
    // Rows of whole 16-byte units that start on their boundaries, and codes (4 or 8 to a unit) likewise.
    const bool vec = (cols * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(q) % Unit<T>::N == 0;
    const unsigned blocks = unsigned((cols + FP8_BLOCK - 1) / FP8_BLOCK);
    const int rows_per = block_rows == 1 ? 32 : FP8_BLOCK;
    // One grid dimension, neighbours along a row first.
    const int grid_cols = int(block_rows == 1 ? (blocks + 3) / 4 : blocks);
    const long long ctas = (rows + rows_per - 1) / rows_per * grid_cols;
    CB200_REQUIRE(ctas <= 2147483647ll, "quantize_fp8: matrix too large");
    const dim3 grid{unsigned(ctas)};
    if (block_rows == 1) {
        if (vec) launch_dependent(quantize_rows_kernel<T>, grid, kThreads, stream, x, rows, cols, grid_cols, q, scales);
        else launch_dependent(quantize_rows_any_kernel<T>, grid, kThreads, stream, x, rows, cols, grid_cols, q, scales);
    } else {
        if (vec) launch_dependent(quantize_tiles_kernel<T>, grid, kThreads, stream, x, rows, cols, grid_cols, q, scales);
        else launch_dependent(quantize_tiles_any_kernel<T>, grid, kTileThreads, stream, x, rows, cols, grid_cols, q, scales);
    }
    CB200_CHECK_LAUNCH();
}

}  // namespace

PreparedRows prepare_rows(const RowsRequest& a, const RowsRequest& b, const ScaleTops& tops, cudaStream_t stream) {
    PreparedRows out;
    PrepareParams p{};
    long long blocks = 0;
    auto add = [&](const RowsRequest& m, AlignedRows& to, PadJob& job) {
        if (m.src == nullptr) return;
        const int per_unit = 16 / m.elem_size;
        if (m.ld != 0 || (m.cols % per_unit == 0 && reinterpret_cast<uintptr_t>(m.src) % 16 == 0)) {
            to.ptr = m.src;
            to.ld = m.ld != 0 ? m.ld : m.cols;
            return;
        }
        CB200_REQUIRE((long long)m.cols * m.elem_size <= 2147483647 - 1023, "a row of this many bytes cannot be copied to a padded one");
        const int units = (m.cols + per_unit - 1) / per_unit;
        to.ld = (long long)units * per_unit;
        to.copy = Scratch(size_t(m.rows) * units * 16, stream);
        to.ptr = to.copy.ptr;
        const long long chunks = (units + 31) / 32, ctas = (m.rows + kThreads / 32 - 1) / (kThreads / 32) * chunks;
        CB200_REQUIRE(ctas <= 1000000000ll, "matrix too large");      // two of them in a grid
        job = PadJob{static_cast<const uint8_t*>(m.src), static_cast<uint8_t*>(to.copy.ptr), m.rows, m.cols * m.elem_size, units * 16,
                     m.offsets, m.rows_group, unsigned(chunks), unsigned(ctas)};
        blocks += ctas;
    };
    add(a, out.a, p.pad[0]);
    add(b, out.b, p.pad[1]);
    if (tops.top != nullptr) {
        p.scales = tops.scales;
        p.scale_rows = tops.rows;
        p.top = tops.top;
        p.wide = tops.wide;
        blocks += tops.blocks();
    }
    if (blocks == 0) return out;
    launch_dependent(prepare_kernel, dim3(unsigned(blocks)), kThreads, stream, p);
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
        launch_dependent(dequantize_kernel<float>, dim3(grid), kThreads, stream, q, scales, rows, cols, block_rows,
                         static_cast<float*>(y));
    else if (y_type == TYPE_F16)
        launch_dependent(dequantize_kernel<__half>, dim3(grid), kThreads, stream, q, scales, rows, cols, block_rows,
                         static_cast<__half*>(y));
    else
        launch_dependent(dequantize_kernel<__nv_bfloat16>, dim3(grid), kThreads, stream, q, scales, rows, cols, block_rows,
                         static_cast<__nv_bfloat16*>(y));
    CB200_CHECK_LAUNCH();
}

ColumnSums activation_backward_fp8(const void* dy, int type, const uint8_t* z8, const float* z_scales, int act, void* dz,
                                   long long ld_dz, float* db, int rows, int cols, cudaStream_t stream) {
    if (type == TYPE_F16)
        return act_backward_typed(static_cast<const __half*>(dy), z8, z_scales, act, static_cast<__half*>(dz), ld_dz, db, rows,
                                  cols, stream);
    return act_backward_typed(static_cast<const __nv_bfloat16*>(dy), z8, z_scales, act, static_cast<__nv_bfloat16*>(dz), ld_dz, db,
                              rows, cols, stream);
}

void finish_sums(const ColumnSums& sums, cudaStream_t stream) {
    const Bands p = bands_of(sums);
    if (p.blocks == 0) return;
    launch_dependent(add_bands_kernel, dim3(p.blocks), kThreads, stream, p);
    CB200_CHECK_LAUNCH();
}

void dequantize_rows(const uint8_t* q, const float* scales, const ScaleTops& tops, int rows, int cols, void* y, long long ld_y,
                     int y_type, const ColumnSums& sums, const SplitRequest& split, cudaStream_t stream) {
    const Bands bands = bands_of(sums);
    const bool vec = cols % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
    const unsigned grid = bands.blocks + pass_grid((long long)rows * ((cols + 7) / 8));
    WideRows wide{};
    if (y_type == TYPE_F16) {
        wide = WideRows{tops.top, tops.wide, tops.blocks(), static_cast<const __half*>(split.src), split.ld, split.ld_parts,
                        split.cols, static_cast<__nv_bfloat16*>(split.parts)};
        __half* out = static_cast<__half*>(y);
        if (vec) launch_dependent(dequantize_rows_kernel<__half, true>, dim3(grid), kThreads, stream, q, scales, rows, cols, out, ld_y, bands, wide);
        else launch_dependent(dequantize_rows_kernel<__half, false>, dim3(grid), kThreads, stream, q, scales, rows, cols, out, ld_y, bands, wide);
    } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(y);
        if (vec) launch_dependent(dequantize_rows_kernel<__nv_bfloat16, true>, dim3(grid), kThreads, stream, q, scales, rows, cols, out, ld_y, bands, wide);
        else launch_dependent(dequantize_rows_kernel<__nv_bfloat16, false>, dim3(grid), kThreads, stream, q, scales, rows, cols, out, ld_y, bands, wide);
    }
    CB200_CHECK_LAUNCH();
}

void add_parts(const float* part, int parts, int m, int n, long long ld, void* out, int type, cudaStream_t stream) {
    const unsigned grid = pass_grid(m * (ld / 4));
    if (type == TYPE_F32)
        launch_dependent(add_parts_kernel<float>, dim3(grid), kThreads, stream, part, parts, m, n, ld, static_cast<float*>(out));
    else if (type == TYPE_F16)
        launch_dependent(add_parts_kernel<__half>, dim3(grid), kThreads, stream, part, parts, m, n, ld, static_cast<__half*>(out));
    else
        launch_dependent(add_parts_kernel<__nv_bfloat16>, dim3(grid), kThreads, stream, part, parts, m, n, ld,
                         static_cast<__nv_bfloat16*>(out));
}

void cast(const void* src, int src_type, void* dst, int dst_type, long long count, cudaStream_t stream) {
    const unsigned grid = pass_grid(count);
    auto from = [&](auto* s) {
        using S = std::remove_pointer_t<decltype(s)>;
        const S* in = static_cast<const S*>(src);
        if (dst_type == TYPE_F32) launch_dependent(cast_kernel<S, float>, dim3(grid), kThreads, stream, in, static_cast<float*>(dst), count);
        else if (dst_type == TYPE_F16) launch_dependent(cast_kernel<S, __half>, dim3(grid), kThreads, stream, in, static_cast<__half*>(dst), count);
        else launch_dependent(cast_kernel<S, __nv_bfloat16>, dim3(grid), kThreads, stream, in, static_cast<__nv_bfloat16*>(dst), count);
    };
    if (src_type == TYPE_F32) from(static_cast<float*>(nullptr));
    else if (src_type == TYPE_F16) from(static_cast<__half*>(nullptr));
    else from(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace cudeep_b200
