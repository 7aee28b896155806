// Microscaled 4-bit matrices: quantisation, the way back, and row-major scales into tiles (include/zc_ffn.h has the format).
//
// All three are bound by memory: a value is read once (2 or 4 bytes) and 17/32 byte written, or the other way round. Nothing is
// rounded but the value itself: the scale is a power of two, so x 2^-e is exact in FP32 wherever it does not fall below half of the
// smallest e2m1 value's threshold, and the conversion instruction rounds it to nearest, ties to even.
#include "ffn.cuh"

namespace zc {
namespace {

constexpr int QT_ROWS = 32, QT_COLS = 256;      // one CTA: a quarter (every fourth word) of two scale tiles
constexpr int FLIGHT = 4;                       // rows of a warp, all of their loads in flight

// A CTA takes 32 rows x 256 columns, whose scales are every fourth 32-bit word of two tiles (gathered in shared memory; words of rows and
// columns past the last one are written 0, so the grid covers whole tiles). Four lanes share a block of 32: lane l holds columns 8 l .. 8 l + 7 of
// the 256, a warp its four rows at once.
template <typename T, bool VEC> __global__ void __launch_bounds__(256) quantize_kernel(const T* x, uint32_t rows, uint32_t cols, uint64_t ld,
                                                                                      uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ uint32_t words[2][QT_ROWS];
    const uint32_t row0 = blockIdx.x * QT_ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = blockIdx.y * QT_COLS + lane * 8;
    const uint32_t r0 = row0 + warp * FLIGHT;
    pdl_wait();
    pdl_launch_dependents();
    float v[FLIGHT][8];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (r0 + i < rows && col < cols) load8<T, VEC>(x + uint64_t(r0 + i) * ld + col, v[i]);      // cols is a multiple of 32: the four lanes of a block agree
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
        uint32_t top = 0;                                // magnitudes as integers: ordered like the values, NaN above all
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t s = mx4_scale(top);               // 0 where there is nothing
        if (r0 + i < rows && col < cols) *reinterpret_cast<uint32_t*>(codes + uint64_t(r0 + i) * (cols >> 1) + (col >> 1)) = mx4_codes8(v[i], s);
        if ((lane & 3) == 0) reinterpret_cast<uint8_t*>(&words[lane >> 4][warp * FLIGHT + i])[(lane >> 2) & 3] = uint8_t(s);
    }
    __syncthreads();
    const uint32_t tiles = (cols + 127) / 128, t = blockIdx.y * 2 + (threadIdx.x >> 5);
    if (threadIdx.x < 64 && t < tiles)
        *reinterpret_cast<uint32_t*>(scales + (uint64_t(row0 / 128) * tiles + t) * 512 + (threadIdx.x & 31) * 16 + (row0 % 128) / 32 * 4) = words[threadIdx.x >> 5][threadIdx.x & 31];
}

// The same shape the other way: 32 rows x 256 columns a CTA, eight columns a lane.
template <typename T, bool VEC> __global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t rows,
                                                                                        uint32_t cols, T* __restrict__ out, uint64_t ld) {
    const uint32_t lane = threadIdx.x & 31, r0 = blockIdx.x * QT_ROWS + (threadIdx.x >> 5) * FLIGHT, col = blockIdx.y * QT_COLS + lane * 8;
    pdl_wait();
    pdl_launch_dependents();
    if (col >= cols || r0 >= rows) return;
    uint32_t word[FLIGHT], s[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
        const uint32_t r = min(r0 + i, rows - 1);
        word[i] = __ldcg(reinterpret_cast<const uint32_t*>(codes + uint64_t(r) * (cols >> 1) + (col >> 1)));
        s[i] = __ldca(scales + mx4_scale_at(r, col / 32, (cols + 127) / 128));
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
        if (r0 + i >= rows) break;
        const float f = mx4_factor(s[i]);
        alignas(16) T v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = mx4_values2((word[i] >> (8 * j)) & 0xffu);
            v[2 * j] = from_f32<T>(p.x * f);
            v[2 * j + 1] = from_f32<T>(p.y * f);
        }
        T* to = out + uint64_t(r0 + i) * ld + col;
        if constexpr (VEC) {
#pragma unroll
            for (uint32_t j = 0; j < sizeof(T) * 8 / 16; ++j) reinterpret_cast<uint4*>(to)[j] = reinterpret_cast<const uint4*>(v)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = v[j];
        }
    }
}

__global__ void __launch_bounds__(128) tile_scales_kernel(const uint8_t* __restrict__ from, uint32_t rows, uint32_t blocks, uint8_t* __restrict__ to) {
    const uint32_t row = blockIdx.x * 128 + threadIdx.x, b0 = blockIdx.y * 4;
    uint32_t word = 0;
    pdl_wait();
    pdl_launch_dependents();
    for (uint32_t j = 0; j < 4; ++j)
        if (row < rows && b0 + j < blocks) word |= uint32_t(__ldca(from + uint64_t(row) * blocks + b0 + j)) << (8 * j);
    *reinterpret_cast<uint32_t*>(to + (uint64_t(blockIdx.x) * gridDim.y + blockIdx.y) * 512 + (threadIdx.x & 31) * 16 + (threadIdx.x >> 5) * 4) = word;
}

template <typename T> int quantize_as(const void* x, uint32_t rows, uint32_t cols, uint64_t ld, void* codes, void* scales, cudaStream_t s) {
    const dim3 grid((rows + 127) / 128 * (128 / QT_ROWS), (cols + QT_COLS - 1) / QT_COLS);      // whole tiles
    auto kernel = rows16(x, ld, sizeof(T)) ? quantize_kernel<T, true> : quantize_kernel<T, false>;
    return launched(launch_after(kernel, grid, 256, 0, 1, s, static_cast<const T*>(x), rows, cols, ld, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)), "mx4 quantisation");
}
template <typename T> int dequantize_as(const void* codes, const void* scales, uint32_t rows, uint32_t cols, void* out, uint64_t ld, cudaStream_t s) {
    const dim3 grid((rows + QT_ROWS - 1) / QT_ROWS, (cols + QT_COLS - 1) / QT_COLS);
    auto kernel = rows16(out, ld, sizeof(T)) ? dequantize_kernel<T, true> : dequantize_kernel<T, false>;
    return launched(launch_after(kernel, grid, 256, 0, 1, s, static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, cols, static_cast<T*>(out), ld), "mx4 dequantisation");
}

}  // namespace

int launch_mx4_quantize(const void* x, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, void* codes, void* scales, cudaStream_t s) {
    if (dtype == ZC_BF16) return quantize_as<__nv_bfloat16>(x, rows, cols, ld, codes, scales, s);
    if (dtype == ZC_F16) return quantize_as<__half>(x, rows, cols, ld, codes, scales, s);
    return quantize_as<float>(x, rows, cols, ld, codes, scales, s);
}
}  // namespace zc

using namespace zc;

extern "C" {

int zc_mx4_scale_bytes(uint32_t rows, uint32_t cols, uint64_t* bytes) {
    if (!bytes) return fail(nullptr, ZC_EINVAL, "missing buffer");
    *bytes = mx4_scale_bytes(rows, cols);
    return ZC_OK;
}

int zc_mx4_quantize(const void* x, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, void* codes, void* scales, void* stream) {
    int rc = check_mx4("zc_mx4_quantize", codes, scales, rows, cols);
    if (rc == ZC_OK) rc = check_matrix("zc_mx4_quantize: x", x, dtype, rows, cols, ld, false);
    if (rc != ZC_OK) return rc;
    if (!rows) return ZC_OK;
    if (rows == 1) ld = cols;
    const Span xs{x, matrix_bytes(dtype, rows, cols, ld)}, cs{codes, uint64_t(rows) * cols / 2}, ss{scales, mx4_scale_bytes(rows, cols)};
    if (overlap(cs, xs) || overlap(ss, xs) || overlap(cs, ss)) return fail(nullptr, ZC_EINVAL, "zc_mx4_quantize: overlapping buffers");
    return launch_mx4_quantize(x, dtype, rows, cols, ld, codes, scales, static_cast<cudaStream_t>(stream));
}

int zc_mx4_dequantize(const void* codes, const void* scales, uint32_t rows, uint32_t cols, void* out, int dtype, uint64_t ld, void* stream) {
    int rc = check_mx4("zc_mx4_dequantize", codes, scales, rows, cols);
    if (rc == ZC_OK) rc = check_matrix("zc_mx4_dequantize: out", out, dtype, rows, cols, ld, false);
    if (rc != ZC_OK) return rc;
    if (!rows) return ZC_OK;
    if (rows == 1) ld = cols;
    const Span os{out, matrix_bytes(dtype, rows, cols, ld)}, cs{codes, uint64_t(rows) * cols / 2}, ss{scales, mx4_scale_bytes(rows, cols)};
    if (overlap(cs, os) || overlap(ss, os)) return fail(nullptr, ZC_EINVAL, "zc_mx4_dequantize: overlapping buffers");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ZC_BF16) return dequantize_as<__nv_bfloat16>(codes, scales, rows, cols, out, ld, s);
    if (dtype == ZC_F16) return dequantize_as<__half>(codes, scales, rows, cols, out, ld, s);
    return dequantize_as<float>(codes, scales, rows, cols, out, ld, s);
}

int zc_mx4_tile_scales(const void* row_scales, uint32_t rows, uint32_t cols, void* scales, void* stream) {
    const int rc = check_mx4("zc_mx4_tile_scales", scales, scales, rows, cols);
    if (rc != ZC_OK) return rc;
    if (!rows) return ZC_OK;
    if (!row_scales) return fail(nullptr, ZC_EINVAL, "zc_mx4_tile_scales: missing buffer");
    if (overlap({row_scales, uint64_t(rows) * (cols / 32)}, {scales, mx4_scale_bytes(rows, cols)}))
        return fail(nullptr, ZC_EINVAL, "zc_mx4_tile_scales: overlapping buffers");
    return launched(launch_after(tile_scales_kernel, dim3((rows + 127) / 128, (cols + 127) / 128), 128, 0, 1, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(row_scales), rows, cols / 32,
                                 static_cast<uint8_t*>(scales)), "mx4 scale tiling");
}

}  // extern "C"
