// Products of the dense feed-forward operators (include/zc_ffn.h): microscaled 4-bit and 16-bit matrices on the tensor cores.
//
// One kernel, five forms. D[M, N] = A . B^T with A and B either MX4 (tcgen05 kind::mxf4, two e8m0 scales per row and 64 k) or 16-bit
// (kind::f16), each 16-bit operand with K or with M / N along its rows, so that none is ever transposed in memory:
//     products of MX4 matrices      A = x, B = w                    the same, gated:  B = 128 rows of gate and 128 of up, side by side
//     gated block, 16 bits          A = x, B = gate | up
//     its dx                        A = dg, du (K = ffn, one after the other), B = gate, up read with N along the rows
//     its dgate, dup                A = dg or du, B = x, both with K = tokens across the rows; the two outputs are tiles of one launch
// Either type has 128 bytes of K per row and pipeline stage and four tensor-core steps of 32 bytes in it, so the loop is the same.
//
// A persistent CTA per SM walks 128 x 256 tiles: one thread issues TMA loads into a ring of four stages, one issues the products into
// tensor memory, eight warps drain it, apply the epilogue in FP32 and store. 128 x 256 is the widest tile a single CTA can issue: a
// step reads 12 KB of shared memory for 128 clocks of tensor work. 16-bit products alternate between two accumulators of 256 columns,
// so the drain is hidden; MX4 products keep their scales in tensor memory too (32 columns a stage), which leaves one, and the drain
// (all of it into registers before the first store) is what the next tile waits for.
// Every wait is bounded (POLL_LIMIT): one that runs out raises ZC_STATUS_TIMEOUT and the CTA's abort flag; its roles leave their
// loops, wait for the copies and products in flight, and the tensor memory is freed.
#include "ffn.cuh"
#include "tcgen05.cuh"
#include <atomic>

namespace zc {

int check_mx4(const char* who, const void* codes, const void* scales, uint32_t rows, uint32_t cols) {
    auto bad = [&](const char* why) { return fail(nullptr, ZC_EINVAL, std::string(who) + ": " + why); };
    if (!cols || cols % 32 || cols > MAX_COLS) return bad("columns must be a multiple of 32, from 32 to 1048576");
    if (rows > 0x7fffffffu) return bad("too many rows");
    if (!rows) return ZC_OK;
    if (!codes || !scales) return bad("missing buffer");
    if (misaligned(codes) || misaligned(scales)) return bad("codes and scales must be 16-byte aligned");
    return ZC_OK;
}

int check_matrix(const char* who, const void* p, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, bool tma) {
    auto bad = [&](const char* why) { return fail(nullptr, ZC_EINVAL, std::string(who) + ": " + why); };
    if (dtype != ZC_BF16 && dtype != ZC_F16 && (dtype != ZC_F32 || tma)) return bad(tma ? "dtype must be BF16 or F16" : "dtype must be BF16, F16 or F32");
    if (!cols || rows > 0x7fffffffu) return bad("invalid shape");
    if (rows > 1 && ld < cols) return bad("row stride below the row's length");
    if (ld > (1ull << 40)) return bad("row stride above 2^40");
    if (!rows) return ZC_OK;
    if (!p) return bad("missing buffer");
    if (misaligned(p, tma ? 16 : dtype_bytes(dtype))) return bad(tma ? "buffers must be 16-byte aligned" : "buffer is not aligned to its elements");
    if (tma && ld * dtype_bytes(dtype) % 16) return bad("row stride must be a multiple of 16 bytes");
    return ZC_OK;
}

namespace {

__device__ uint32_t ffn_status_word;     // the device's status word of these operators (zc_ffn_status)

constexpr uint32_t TILE_M = 128, TILE_N = 256, STAGES = 4, THREADS = 320;
constexpr uint32_t A_BYTES = TILE_M * 128, B_BYTES = TILE_N * 128, SF_BYTES = 3 * 1024;
constexpr uint32_t SF_COLUMN = 256, SF_COLUMNS = 32;      // MX4: first column of the scales, columns a stage: A 2 x 4, B 2 x 8 (of 32)

struct TileMaps { CUtensorMap a[2], b[2]; };

struct TilePlan {
    uint32_t M, N;                      // rows and columns of an output (gated: N = ffn)
    uint32_t kblocks, ksteps;           // blocks of 128 bytes of K; steps of 32 bytes in the last one
    uint32_t segs, outs;                // pairs (a[s], b[s]) whose products add up; outputs a[z] . b[0]
    uint32_t mtiles, ntiles, tiles;
    uint32_t idesc;
    uint32_t ktiles, brows;             // MX4: scale tiles along K; rows of B
    const uint8_t *sfa, *sfb[2];
    void* out[2];
    uint64_t ldo;
    void *g, *u;                        // gated: where the two products go as well, or null
    int out_type;
    bool vec;                           // the output's rows are 16-byte aligned
};

struct Tile { uint32_t z, m0, n0; };

// Bands of eight row tiles, walked column by column: what runs at one time shares few rows of A and of B in L2.
__device__ __forceinline__ Tile tile_at(const TilePlan& p, uint32_t t, uint32_t width) {
    const uint32_t per = p.mtiles * p.ntiles, z = t / per, i = t % per, band = i / (8 * p.ntiles), j = i % (8 * p.ntiles);
    const uint32_t rows = min(8u, p.mtiles - band * 8);
    return {z, (band * 8 + j % rows) * TILE_M, j / rows * width};
}

// `valid` leading values of v to a row.
template <typename T, int NC> __device__ __forceinline__ void store_row(T* to, uint32_t valid, bool vec, const float (&v)[NC]) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < NC; c += PER) {
        if (vec && c + PER <= valid) {
            alignas(16) T w[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) w[j] = from_f32<T>(v[c + j]);
            *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(w);
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (c + j < valid) to[c + j] = from_f32<T>(v[c + j]);
        }
    }
}
template <int NC> __device__ __forceinline__ void store_as(void* out, int type, uint64_t at, uint32_t valid, bool vec, const float (&v)[NC]) {
    if (type == ZC_BF16) store_row(static_cast<__nv_bfloat16*>(out) + at, valid, vec, v);
    else if (type == ZC_F16) store_row(static_cast<__half*>(out) + at, valid, vec, v);
    else store_row(static_cast<float*>(out) + at, valid, vec, v);
}
__device__ __forceinline__ float silu(float v) { return __fdiv_rn(v, 1.0f + expf(-v)); }

template <bool MX4> struct TileSmem {
    static constexpr uint32_t stage = A_BYTES + B_BYTES + (MX4 ? SF_BYTES : 0), bytes = STAGES * stage + 1024;
};

template <bool MX4, bool A_MN, bool B_MN, bool GATED>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ TileMaps maps, const TilePlan p) {
    constexpr uint32_t ACC = MX4 ? 1 : 2, STAGE = TileSmem<MX4>::stage, KB = MX4 ? 128 : 64;      // KB: TMA elements of K a block (bytes of codes, 16-bit values)
    constexpr uint32_t WIDTH = GATED ? TILE_N / 2 : TILE_N;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[ACC], acc_empty[ACC], drain;
    __shared__ uint32_t tmem_s, abort_s;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t* const status = &ffn_status_word;
    volatile uint32_t* const abort_flag = &abort_s;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (uint32_t i = 0; i < ACC; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 8); }
        mbar_init(&drain, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_s;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
                const Tile c = tile_at(p, t, WIDTH);
                for (uint32_t s = 0; ok && s < p.segs; ++s) {
                    const CUtensorMap* const ma = &maps.a[p.outs == 2 ? c.z : s];
                    const CUtensorMap* const mb = &maps.b[s];
                    for (uint32_t kb = 0; kb < p.kblocks; ++kb, ++it) {
                        const uint32_t slot = it % STAGES, a = ring + slot * STAGE, b = a + A_BYTES;
                        if (it >= STAGES && !mbar_wait(&empty[slot], (it / STAGES - 1) & 1, abort_flag, status)) { ok = false; break; }
                        const uint32_t atoms = MX4 ? min(2u, p.ktiles - kb * 2) : 0;
                        const uint32_t second = GATED ? 0 : c.n0 + 128;      // MX4: row of B whose scale tile follows (gated: up's own)
                        const bool two = GATED || second < p.brows;
                        mbar_expect(&full[slot], A_BYTES + B_BYTES + atoms * 512 * (two ? 3 : 2));
                        if constexpr (A_MN) {
                            for (uint32_t i = 0; i < 2; ++i) tma_load_2d(a + i * 8192, ma, &full[slot], c.m0 + i * 64, kb * 64);
                        } else {
                            tma_load_2d(a, ma, &full[slot], kb * KB, c.m0);
                        }
                        if constexpr (B_MN) {
                            for (uint32_t i = 0; i < 4; ++i) tma_load_2d(b + i * 8192, mb, &full[slot], c.n0 + i * 64, kb * 64);
                        } else if constexpr (GATED) {
                            tma_load_2d(b, &maps.b[0], &full[slot], kb * KB, c.n0);
                            tma_load_2d(b + 16384, &maps.b[1], &full[slot], kb * KB, c.n0);
                        } else {
                            tma_load_2d(b, mb, &full[slot], kb * KB, c.n0);
                            tma_load_2d(b + 16384, mb, &full[slot], kb * KB, c.n0 + 128);
                        }
                        if constexpr (MX4) {
                            const uint32_t sf = b + B_BYTES;
                            const uint64_t at = uint64_t(c.n0 / 128) * p.ktiles + kb * 2;
                            bulk_load(sf, p.sfa + (uint64_t(c.m0 / 128) * p.ktiles + kb * 2) * 512, atoms * 512, &full[slot]);
                            bulk_load(sf + 1024, p.sfb[0] + at * 512, atoms * 512, &full[slot]);
                            if (two) bulk_load(sf + 2048, GATED ? p.sfb[1] + at * 512 : p.sfb[0] + (at + p.ktiles) * 512, atoms * 512, &full[slot]);
                        }
                    }
                }
            }
            if (!ok)      // the last copies into every slot land before the CTA may end
                for (uint32_t f = it > STAGES ? it - STAGES : 0; f < it; ++f)
                    for (uint32_t i = 0; i < POLL_LIMIT && !mbar_try(&full[f % STAGES], (f / STAGES) & 1); ++i) {}
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t it = 0, n = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++n) {
                const uint32_t buf = n % ACC, acc = tmem + buf * 256;
                if (n >= ACC && !mbar_wait(&acc_empty[buf], (n / ACC - 1) & 1, abort_flag, status)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t more = 0;
                for (uint32_t s = 0; ok && s < p.segs; ++s) {
                    for (uint32_t kb = 0; kb < p.kblocks; ++kb, ++it) {
                        const uint32_t slot = it % STAGES, a = ring + slot * STAGE, b = a + A_BYTES;
                        if (!mbar_wait(&full[slot], (it / STAGES) & 1, abort_flag, status)) { ok = false; break; }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t da = desc_at(A_MN ? DESC_MN_MAJOR : DESC_K_MAJOR, a), db = desc_at(B_MN ? DESC_MN_MAJOR : DESC_K_MAJOR, b);
                        const uint32_t steps = kb + 1 == p.kblocks ? p.ksteps : 4;
                        const uint32_t sf = tmem + SF_COLUMN + slot * SF_COLUMNS;
                        if constexpr (MX4) {
                            // 128 k of scales: four columns for A's rows, eight for B's (its two blocks of 128 rows)
                            for (uint32_t j = 0; j < (steps + 1) / 2; ++j) {
                                tmem_copy_scales(sf + j * 4, desc_at(DESC_SCALES, b + B_BYTES + j * 512));
                                tmem_copy_scales(sf + 8 + j * 8, desc_at(DESC_SCALES, b + B_BYTES + 1024 + j * 512));
                                tmem_copy_scales(sf + 12 + j * 8, desc_at(DESC_SCALES, b + B_BYTES + 2048 + j * 512));
                            }
                        }
                        for (uint32_t k = 0; k < steps; ++k, more = 1) {
                            if constexpr (MX4) {
                                const uint32_t id = (k & 1) * 2;         // which two of a column's four scales
                                umma_mx4(acc, da + k * 2, db + k * 2, p.idesc | id << 29 | id << 4, sf + (k >> 1) * 4, sf + 8 + (k >> 1) * 8, more);
                            } else {
                                umma_f16(acc, da + k * (A_MN ? 128 : 2), db + k * (B_MN ? 128 : 2), p.idesc, more);
                            }
                        }
                        umma_commit(&empty[slot]);
                    }
                }
                if (ok) umma_commit(&acc_full[buf]);
            }
            if (abort_s) {       // products in flight read shared memory and write tensor memory: they end first
                umma_commit(&drain);
                for (uint32_t i = 0; i < POLL_LIMIT && !mbar_try(&drain, 0); ++i) {}
            }
        }
    } else {
        const uint32_t half = (warp - 2) >> 2, quarter = warp & 3;      // columns; the 32 lanes of tensor memory a warp can read
        uint32_t n = 0;
        for (uint32_t t = blockIdx.x; t < p.tiles; t += gridDim.x, ++n) {
            const Tile c = tile_at(p, t, WIDTH);
            const uint32_t buf = n % ACC, acc = tmem + buf * 256 + (quarter << 21);
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (n / ACC) & 1, abort_flag, status))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float v[128];      // gated: 64 of gate, then 64 of up
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld32(acc + (GATED ? (i >> 1) * 128 + half * 64 + (i & 1) * 32 : half * 128 + i * 32), v + i * 32);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
            const uint32_t row = c.m0 + quarter * 32 + lane, col = c.n0 + half * (WIDTH / 2);
            if (row >= p.M || col >= p.N) continue;
            const uint64_t at = uint64_t(row) * p.ldo + col;
            const uint32_t valid = p.N - col;
            if constexpr (GATED) {
                float gate[64], up[64];
#pragma unroll
                for (int i = 0; i < 64; ++i) { gate[i] = v[i]; up[i] = v[64 + i]; }
                if (p.g) {
                    store_as(p.g, p.out_type, at, valid, p.vec, gate);
                    store_as(p.u, p.out_type, at, valid, p.vec, up);
                }
#pragma unroll
                for (int i = 0; i < 64; ++i) gate[i] = silu(gate[i]) * up[i];
                store_as(p.out[0], p.out_type, at, valid, p.vec, gate);
            } else {
                store_as(c.z ? p.out[1] : p.out[0], p.out_type, at, valid, p.vec, v);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// dg = dh u s (1 + g (1 - s)), du = dh g s; eight values a thread. Bound by memory: three reads and two writes of 16 bits a value.
template <typename T> __global__ void __launch_bounds__(256) gated_gradient_kernel(const T* __restrict__ dh, uint64_t dh_ld, const T* __restrict__ g, const T* __restrict__ u, uint32_t tokens,
                                                                                   uint32_t ffn, T* __restrict__ dg, T* __restrict__ du) {
    const uint32_t per_row = ffn / 8;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < uint64_t(tokens) * per_row; i += uint64_t(gridDim.x) * 256) {
        const uint64_t row = i / per_row, col = i % per_row;
        alignas(16) T a[8], b[8], c[8], d[8], e[8];
        *reinterpret_cast<uint4*>(a) = __ldg(reinterpret_cast<const uint4*>(dh + row * dh_ld) + col);
        *reinterpret_cast<uint4*>(b) = __ldg(reinterpret_cast<const uint4*>(g) + i);
        *reinterpret_cast<uint4*>(c) = __ldg(reinterpret_cast<const uint4*>(u) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gv = float(b[j]), s = __fdividef(1.0f, 1.0f + __expf(-gv)), dv = float(a[j]);
            d[j] = from_f32<T>(dv * float(c[j]) * s * (1.0f + gv * (1.0f - s)));
            e[j] = from_f32<T>(dv * gv * s);
        }
        reinterpret_cast<uint4*>(dg)[i] = *reinterpret_cast<const uint4*>(d);
        reinterpret_cast<uint4*>(du)[i] = *reinterpret_cast<const uint4*>(e);
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                           CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode tensor_map_encoder() {
    static const Encode encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
        if (e != cudaSuccess) cudaGetLastError();
        return reinterpret_cast<Encode>(e == cudaSuccess && q == cudaDriverEntryPointSuccess ? p : nullptr);
    }();
    return encode;
}
// A view of `rows` rows of `inner` elements (bytes, or 16-bit values), `stride` bytes apart, in boxes of 128 bytes x box_rows.
bool make_map(CUtensorMap& m, const void* base, bool bytes, uint64_t inner, uint64_t rows, uint64_t stride, uint32_t box_rows) {
    const Encode encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {inner, rows}, strides[1] = {stride};
    const cuuint32_t box[2] = {bytes ? 128u : 64u, box_rows}, elem[2] = {1, 1};
    return encode(&m, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool map_codes(CUtensorMap& m, const void* codes, uint32_t rows, uint32_t cols) { return make_map(m, codes, true, cols / 2, rows, cols / 2, 128); }
// A 16-bit operand [rows, cols]: K along its rows (boxes of 64 k x 128 rows), or across them (boxes of 64 columns x 64 k).
bool map_rows(CUtensorMap& m, const void* p, uint32_t rows, uint32_t cols, uint64_t ld, bool k_across) { return make_map(m, p, false, cols, rows, ld * 2, k_across ? 64 : 128); }

// Instruction descriptors. Both: N / 8 from bit 17, M / 16 from bit 24.
uint32_t idesc_f16(int dtype, bool a_mn, bool b_mn) {      // FP32 accumulators; operand types; which operand has M / N along its rows
    const uint32_t t = dtype == ZC_BF16 ? 1 : 0;
    return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | ((TILE_N / 8) << 17) | ((TILE_M / 16) << 24);
}
uint32_t idesc_mx4() { return (1u << 7) | (1u << 10) | ((TILE_N / 8) << 17) | (1u << 23) | ((TILE_M / 16) << 24); }      // e2m1 both, e8m0 scales

struct Device { int index = -1; uint32_t sms = 0; };
int current_device(Device& d) {
    static std::atomic<uint32_t> sms[MAX_DEVICES];
    cudaError_t e = cudaGetDevice(&d.index);
    if (e == cudaSuccess && (d.index < 0 || d.index >= MAX_DEVICES)) e = cudaErrorInvalidDevice;
    if (e == cudaSuccess && !(d.sms = sms[d.index].load(std::memory_order_relaxed))) {
        int n = 0;
        e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d.index);
        sms[d.index].store(d.sms = uint32_t(n), std::memory_order_relaxed);
    }
    if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("no CUDA device: ") + cudaGetErrorString(e)); }
    return ZC_OK;
}

template <bool MX4, bool A_MN, bool B_MN, bool GATED> int launch_tiles(const TileMaps& maps, TilePlan& p, cudaStream_t s) {
    Device d;
    const int rc = current_device(d);
    if (rc != ZC_OK) return rc;
    auto kernel = tile_kernel<MX4, A_MN, B_MN, GATED>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(TileSmem<MX4>::bytes));
    if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e)); }
    constexpr uint32_t width = GATED ? TILE_N / 2 : TILE_N;
    p.mtiles = (p.M + TILE_M - 1) / TILE_M;
    p.ntiles = (p.N + width - 1) / width;
    const uint64_t tiles = uint64_t(p.mtiles) * p.ntiles * p.outs;
    if (tiles > 0x7fffffffu) return fail(nullptr, ZC_EINVAL, "too many output tiles");
    p.tiles = uint32_t(tiles);
    p.vec = rows16(p.out[0], p.ldo, dtype_bytes(p.out_type)) && (!p.out[1] || rows16(p.out[1], p.ldo, dtype_bytes(p.out_type)));
    kernel<<<p.tiles < d.sms ? p.tiles : d.sms, THREADS, TileSmem<MX4>::bytes, s>>>(maps, p);
    return check_launch(nullptr, "dense product");
}

void set_k(TilePlan& p, uint32_t k, uint32_t block) {
    p.kblocks = (k + block - 1) / block;
    const uint32_t left = k - (p.kblocks - 1) * block, step = block / 4;
    p.ksteps = (left + step - 1) / step;
}

int no_maps() { return fail(nullptr, ZC_EEXEC, "the driver did not encode a tensor map"); }

struct Mx4Arg { const void *codes, *scales; };

// x . w[0]^T, or the gated block of w[0] and w[1].
int mx4_product(const char* who, const void* x, int x_dtype, uint64_t x_ld, void* x_codes, void* x_scales, uint32_t tokens, uint32_t cols, const Mx4Arg* w, int mats,
                uint32_t rows, void* out, int out_dtype, uint64_t out_ld, void* stream) {
    int rc = check_mx4(who, x_codes, x_scales, tokens, cols);
    if (rc == ZC_OK && x) rc = check_matrix((std::string(who) + ": x").c_str(), x, x_dtype, tokens, cols, x_ld, false);
    for (int i = 0; rc == ZC_OK && i < mats; ++i) rc = check_mx4(who, w[i].codes, w[i].scales, rows, cols);
    if (rc == ZC_OK && !rows) rc = fail(nullptr, ZC_EINVAL, std::string(who) + ": no rows in the weights");
    if (rc == ZC_OK) rc = check_matrix((std::string(who) + ": output").c_str(), out, out_dtype, tokens, rows, out_ld, false);
    if (rc != ZC_OK || !tokens) return rc;
    const Span os{out, matrix_bytes(out_dtype, tokens, rows, out_ld)}, cs{x_codes, uint64_t(tokens) * cols / 2}, ss{x_scales, mx4_scale_bytes(tokens, cols)};
    const Span xs{x, x ? matrix_bytes(x_dtype, tokens, cols, x_ld) : 0};
    bool bad = overlap(os, cs) || overlap(os, ss) || overlap(os, xs) || (x && (overlap(cs, ss) || overlap(cs, xs) || overlap(ss, xs)));
    for (int i = 0; i < mats; ++i)
        for (const Span& t : {Span{w[i].codes, uint64_t(rows) * cols / 2}, Span{w[i].scales, mx4_scale_bytes(rows, cols)}})
            bad = bad || overlap(os, t) || (x && (overlap(cs, t) || overlap(ss, t)));
    if (bad) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x && (rc = launch_mx4_quantize(x, x_dtype, tokens, cols, x_ld, x_codes, x_scales, s)) != ZC_OK) return rc;
    TileMaps maps{};
    TilePlan p{};
    if (!map_codes(maps.a[0], x_codes, tokens, cols)) return no_maps();
    for (int i = 0; i < mats; ++i)
        if (!map_codes(maps.b[i], w[i].codes, rows, cols)) return no_maps();
    p.M = tokens; p.N = rows; p.segs = 1; p.outs = 1;
    set_k(p, cols, 256);
    p.idesc = idesc_mx4();
    p.ktiles = (cols + 127) / 128; p.brows = rows;
    p.sfa = static_cast<const uint8_t*>(x_scales);
    for (int i = 0; i < mats; ++i) p.sfb[i] = static_cast<const uint8_t*>(w[i].scales);
    p.out[0] = out; p.ldo = out_ld; p.out_type = out_dtype;
    return mats == 2 ? launch_tiles<true, false, false, true>(maps, p, s) : launch_tiles<true, false, false, false>(maps, p, s);
}

int check_gated(const char* who, int dtype, uint32_t hidden, uint32_t ffn) {
    if (dtype != ZC_BF16 && dtype != ZC_F16) return fail(nullptr, ZC_EINVAL, std::string(who) + ": dtype must be BF16 or F16");
    if (!hidden || hidden % 8 || hidden > MAX_COLS || !ffn || ffn % 8 || ffn > MAX_COLS)
        return fail(nullptr, ZC_EINVAL, std::string(who) + ": hidden and ffn must be multiples of 8, from 8 to 1048576");
    return ZC_OK;
}

}  // namespace
}  // namespace zc

using namespace zc;

extern "C" {

int zc_mx4_linear(const void* x, int x_dtype, uint64_t x_ld, void* x_codes, void* x_scales, uint32_t tokens, uint32_t cols, const void* w_codes, const void* w_scales,
                  uint32_t rows, void* out, int out_dtype, uint64_t out_ld, void* stream) {
    const Mx4Arg w[1] = {{w_codes, w_scales}};
    return mx4_product("zc_mx4_linear", x, x_dtype, x_ld, x_codes, x_scales, tokens, cols, w, 1, rows, out, out_dtype, out_ld, stream);
}

int zc_mx4_gated(const void* x, int x_dtype, uint64_t x_ld, void* x_codes, void* x_scales, uint32_t tokens, uint32_t cols, const void* gate_codes, const void* gate_scales,
                 const void* up_codes, const void* up_scales, uint32_t ffn, void* h, int out_dtype, uint64_t out_ld, void* stream) {
    const Mx4Arg w[2] = {{gate_codes, gate_scales}, {up_codes, up_scales}};
    return mx4_product("zc_mx4_gated", x, x_dtype, x_ld, x_codes, x_scales, tokens, cols, w, 2, ffn, h, out_dtype, out_ld, stream);
}

int zc_gated_forward(const void* x, uint64_t x_ld, const void* gate, const void* up, int dtype, uint32_t tokens, uint32_t hidden, uint32_t ffn, void* h, void* g, void* u,
                     void* stream) {
    const char* who = "zc_gated_forward";
    int rc = check_gated(who, dtype, hidden, ffn);
    if (rc == ZC_OK) rc = check_matrix(who, x, dtype, tokens, hidden, x_ld, true);
    for (const void* w : {gate, up}) if (rc == ZC_OK) rc = check_matrix(who, w, dtype, ffn, hidden, hidden, true);
    if (rc == ZC_OK) rc = check_matrix(who, h, dtype, tokens, ffn, ffn, true);
    if (rc == ZC_OK && tokens && !g != !u) rc = fail(nullptr, ZC_EINVAL, std::string(who) + ": g and u go together");
    for (const void* v : {g, u}) if (rc == ZC_OK && v) rc = check_matrix(who, v, dtype, tokens, ffn, ffn, true);
    if (rc != ZC_OK || !tokens) return rc;
    const uint64_t tf = uint64_t(tokens) * ffn * 2, fh = uint64_t(ffn) * hidden * 2;
    const Span in[3] = {{x, matrix_bytes(dtype, tokens, hidden, x_ld)}, {gate, fh}, {up, fh}}, to[3] = {{h, tf}, {g, tf}, {u, tf}};
    for (int i = 0; i < 3; ++i) {
        for (const Span& v : in) if (overlap(to[i], v)) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
        for (int j = 0; j < i; ++j) if (overlap(to[i], to[j])) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    }
    TileMaps maps{};
    TilePlan p{};
    if (!map_rows(maps.a[0], x, tokens, hidden, x_ld, false) || !map_rows(maps.b[0], gate, ffn, hidden, hidden, false) || !map_rows(maps.b[1], up, ffn, hidden, hidden, false))
        return no_maps();
    p.M = tokens; p.N = ffn; p.segs = 1; p.outs = 1;
    set_k(p, hidden, 64);
    p.idesc = idesc_f16(dtype, false, false);
    p.out[0] = h; p.g = g; p.u = u; p.ldo = ffn; p.out_type = dtype;
    return launch_tiles<false, false, false, true>(maps, p, static_cast<cudaStream_t>(stream));
}

int zc_gated_backward(const void* dh, uint64_t dh_ld, const void* x, uint64_t x_ld, const void* gate, const void* up, const void* g, const void* u, int dtype, uint32_t tokens,
                      uint32_t hidden, uint32_t ffn, void* dg, void* du, void* dx, void* dgate, void* dup, void* stream) {
    const char* who = "zc_gated_backward";
    int rc = check_gated(who, dtype, hidden, ffn);
    if (rc == ZC_OK) rc = check_matrix(who, dh, dtype, tokens, ffn, dh_ld, true);
    if (rc == ZC_OK) rc = check_matrix(who, x, dtype, tokens, hidden, x_ld, true);
    for (const void* w : {gate, up}) if (rc == ZC_OK) rc = check_matrix(who, w, dtype, ffn, hidden, hidden, true);
    for (const void* v : {g, u, static_cast<const void*>(dg), static_cast<const void*>(du)}) if (rc == ZC_OK) rc = check_matrix(who, v, dtype, tokens, ffn, ffn, true);
    if (rc == ZC_OK && dx) rc = check_matrix(who, dx, dtype, tokens, hidden, hidden, true);
    if (rc == ZC_OK && !dgate != !dup) rc = fail(nullptr, ZC_EINVAL, std::string(who) + ": dgate and dup go together");
    for (const void* v : {dgate, dup}) if (rc == ZC_OK && v) rc = check_matrix(who, v, dtype, ffn, hidden, hidden, true);
    if (rc != ZC_OK) return rc;
    const uint64_t tf = uint64_t(tokens) * ffn * 2, fh = uint64_t(ffn) * hidden * 2, th = uint64_t(tokens) * hidden * 2;
    const Span in[6] = {{dh, matrix_bytes(dtype, tokens, ffn, dh_ld)}, {x, matrix_bytes(dtype, tokens, hidden, x_ld)}, {gate, fh}, {up, fh}, {g, tf}, {u, tf}};
    const Span to[5] = {{dg, tf}, {du, tf}, {dx, th}, {dgate, fh}, {dup, fh}};
    for (int i = 0; i < 5; ++i) {
        for (const Span& v : in) if (overlap(to[i], v)) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
        for (int j = 0; j < i; ++j) if (overlap(to[i], to[j])) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!tokens) {
        for (void* v : {dgate, dup}) {
            const cudaError_t e = v ? cudaMemsetAsync(v, 0, fh, s) : cudaSuccess;
            if (e != cudaSuccess) return fail(nullptr, ZC_EEXEC, std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
        }
        return ZC_OK;
    }
    const uint64_t blocks = (uint64_t(tokens) * (ffn / 8) + 255) / 256;
    const uint32_t grid = uint32_t(blocks < 148 * 16 ? blocks : 148 * 16);
    if (dtype == ZC_BF16) {
        typedef __nv_bfloat16 T;
        gated_gradient_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(dh), dh_ld, static_cast<const T*>(g), static_cast<const T*>(u), tokens, ffn, static_cast<T*>(dg), static_cast<T*>(du));
    } else {
        typedef __half T;
        gated_gradient_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(dh), dh_ld, static_cast<const T*>(g), static_cast<const T*>(u), tokens, ffn, static_cast<T*>(dg), static_cast<T*>(du));
    }
    if ((rc = check_launch(nullptr, "gated gradient")) != ZC_OK) return rc;
    if (dx) {
        TileMaps maps{};
        TilePlan p{};
        if (!map_rows(maps.a[0], dg, tokens, ffn, ffn, false) || !map_rows(maps.a[1], du, tokens, ffn, ffn, false) ||
            !map_rows(maps.b[0], gate, ffn, hidden, hidden, true) || !map_rows(maps.b[1], up, ffn, hidden, hidden, true)) return no_maps();
        p.M = tokens; p.N = hidden; p.segs = 2; p.outs = 1;
        set_k(p, ffn, 64);
        p.idesc = idesc_f16(dtype, false, true);
        p.out[0] = dx; p.ldo = hidden; p.out_type = dtype;
        if ((rc = launch_tiles<false, false, true, false>(maps, p, s)) != ZC_OK) return rc;
    }
    if (dgate) {
        TileMaps maps{};
        TilePlan p{};
        if (!map_rows(maps.a[0], dg, tokens, ffn, ffn, true) || !map_rows(maps.a[1], du, tokens, ffn, ffn, true) || !map_rows(maps.b[0], x, tokens, hidden, x_ld, true)) return no_maps();
        p.M = ffn; p.N = hidden; p.segs = 1; p.outs = 2;
        set_k(p, tokens, 64);
        p.idesc = idesc_f16(dtype, true, true);
        p.out[0] = dgate; p.out[1] = dup; p.ldo = hidden; p.out_type = dtype;
        rc = launch_tiles<false, true, true, false>(maps, p, s);
    }
    return rc;
}

int zc_ffn_status(void* stream, uint32_t* status) {
    if (!status) return fail(nullptr, ZC_EINVAL, "missing buffer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint32_t zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, ffn_status_word, 4, 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(ffn_status_word, &zero, 4, 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("status: ") + cudaGetErrorString(e)); }
    return ZC_OK;
}

}  // extern "C"
