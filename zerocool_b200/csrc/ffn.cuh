// What the dense feed-forward operators (include/zc_ffn.h) share: the microscaled format and the checks of their arguments.
#pragma once
#include "common.cuh"
#include "../../include/zc_ffn.h"

namespace zc {

// ---------------------------------------------------------------------------------------------
// Microscaled values
// ---------------------------------------------------------------------------------------------
inline uint64_t mx4_scale_bytes(uint32_t rows, uint32_t cols) { return uint64_t((uint64_t(rows) + 127) / 128) * ((uint64_t(cols) + 127) / 128) * 512; }
// Byte of the scale of (row, block of 32 columns); ktiles = ceil(cols / 128).
__host__ __device__ inline uint64_t mx4_scale_at(uint32_t row, uint32_t block, uint32_t ktiles) {
    return (uint64_t(row / 128) * ktiles + block / 4) * 512 + (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4;
}
#ifdef __CUDACC__
// Scale byte of a block whose largest magnitude has these bits: floor(log2) - 2 from the exponent field (zero and subnormal values:
// the smallest scale), 255 where a value is infinite or NaN.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top_bits) {
    const uint32_t field = top_bits >> 23;
    return field == 255 ? 255u : field > 2 ? field - 2 : 0u;
}
__device__ __forceinline__ float mx4_factor(uint32_t s) { return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u); }   // 2^(s - 127)
// Eight values -> eight codes, the first in the lowest bits. 2^(127 - s) is exact for every s that mx4_scale gives (0..252).
__device__ __forceinline__ uint32_t mx4_codes8(const float (&v)[8], uint32_t s) {
    const float f = __uint_as_float((254u - s) << 23);
    uint32_t word;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(word) : "f"(v[0] * f), "f"(v[1] * f), "f"(v[2] * f), "f"(v[3] * f), "f"(v[4] * f), "f"(v[5] * f), "f"(v[6] * f), "f"(v[7] * f));
    return s == 255 ? 0u : word;
}
__device__ __forceinline__ float2 mx4_values2(uint32_t byte) {      // low half first
    uint32_t h2;
    asm("{\n\t.reg .b8 a, z;\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tmov.b16 {a, z}, h;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h2) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(float v) { return v; }

// Eight consecutive values of a row. VEC: the row is 16-byte aligned. Not through the read-only path: a kernel of these starts while the kernel
// before it still writes (programmatic launch), and that path may keep what it read before.
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    alignas(16) T raw[8];
    if constexpr (VEC) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) * 8 / 16; ++i) reinterpret_cast<uint4*>(raw)[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) reinterpret_cast<float*>(raw)[i] = __ldca(reinterpret_cast<const float*>(p) + i);
            else reinterpret_cast<unsigned short*>(raw)[i] = __ldca(reinterpret_cast<const unsigned short*>(p) + i);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(raw[i]);
}
#endif

// ---------------------------------------------------------------------------------------------
// Arguments
// ---------------------------------------------------------------------------------------------
struct Span { const void* p; uint64_t bytes; uint64_t width = 0, pitch = 0; };      // a matrix of several rows: bytes of a row, and from one to the next
// Columns side by side in the rows of one buffer share no byte, though the one's rows lie between the other's.
inline bool overlap(const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    if (!a.p || !b.p || !a.bytes || !b.bytes || x >= y + b.bytes || y >= x + a.bytes) return false;
    const uint64_t pitch = a.pitch ? a.pitch : b.pitch;
    if (!pitch || (a.pitch && b.pitch && a.pitch != b.pitch)) return true;
    const uint64_t after = x >= y ? (x - y) % pitch : (pitch - (y - x) % pitch) % pitch;      // where a row of a starts, from the start of b's row before it
    return after < (b.pitch ? b.width : b.bytes) || after + (a.pitch ? a.width : a.bytes) > pitch;
}
inline uint64_t dtype_bytes(int dtype) { return dtype == ZC_F32 ? 4 : 2; }
inline uint64_t matrix_bytes(int dtype, uint64_t rows, uint64_t cols, uint64_t ld) { return rows ? ((rows - 1) * ld + cols) * dtype_bytes(dtype) : 0; }
inline Span matrix_span(const void* p, int dtype, uint64_t rows, uint64_t cols, uint64_t ld) {
    return rows > 1 ? Span{p, matrix_bytes(dtype, rows, cols, ld), cols * dtype_bytes(dtype), ld * dtype_bytes(dtype)} : Span{p, matrix_bytes(dtype, rows, cols, ld)};
}
inline bool misaligned(const void* p, uintptr_t to = 16) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }
// Whether every row of a matrix starts on 16 bytes.
inline bool rows16(const void* p, uint64_t ld, uint64_t elem) { return !misaligned(p) && ld * elem % 16 == 0; }

constexpr uint32_t MAX_COLS = 1u << 20;      // columns of any matrix here; rows are limited to 2^31 - 1 (TMA coordinates are signed)
// A microscaled matrix: pointers (needed where rows > 0), alignment, sizes.
int check_mx4(const char* who, const void* codes, const void* scales, uint32_t rows, uint32_t cols);
// A plain matrix: type, row stride, and alignment to 16 bytes (rows and all: `tma`) or to its elements.
int check_matrix(const char* who, const void* p, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, bool tma);

#ifdef __CUDACC__
// A launch that may start while the kernel before it on the stream still runs (the rules of launch_chained: everything up to pdl_wait()
// reads and writes no global memory, and pdl_launch_dependents() comes after it). `cluster`: CTAs of a cluster.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, uint32_t block, size_t smem, uint32_t cluster, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}
inline int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return ZC_OK;
    cudaGetLastError();
    return fail(nullptr, ZC_EEXEC, std::string("CUDA launch of ") + what + ": " + cudaGetErrorString(e));
}
#endif

int launch_mx4_quantize(const void* x, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, void* codes, void* scales, cudaStream_t s);

}  // namespace zc
