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
// A pair of CTAs (cta_group::2) walks tiles of 256 rows x 256 (or 128) columns: either CTA stages its 128 rows of A and its half of B's
// rows by TMA into a ring, one thread of the leading CTA issues the products of both, and eight warps of either drain its 128 rows from
// tensor memory, apply the epilogue in FP32 and store. The pair halves B's traffic: 32 KB from L2 per SM for 512 clocks of tensor work, not
// the 48 KB of a single CTA's widest tile, whose loop L2 bounded (11 TB/s: 150 us for MX4 8192 x 8192 x 4096).
// Two accumulators where they fit, so that the drain is hidden. MX4 products keep their scales in tensor memory too (32 columns a stage),
// which leaves one of 256: the next tile waits until it is in registers, not until it is stored.
// Every wait is bounded (POLL_LIMIT polls, unless zc_ffn_wait_limit says otherwise): one that runs out raises ZC_STATUS_TIMEOUT and the abort
// flag, of both CTAs of a pair and all pairs of a tile; the roles leave their loops, and no CTA frees its tensor memory or ends before the
// copies and products that it has started have ended. A copy has ended when its stage is released; the copying thread therefore waits for the
// last stage too (while the others drain the last tile), and where that is cut short, for the bytes themselves.
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
    if (rows > 1 && ld > (1ull << 30)) return bad("row stride above 2^30");
    if (!rows) return ZC_OK;
    if (!p) return bad("missing buffer");
    if (misaligned(p, tma ? 16 : dtype_bytes(dtype))) return bad(tma ? "buffers must be 16-byte aligned" : "buffer is not aligned to its elements");
    if (tma && rows > 1 && ld * dtype_bytes(dtype) % 16) return bad("row stride must be a multiple of 16 bytes");
    return ZC_OK;
}

namespace {

__device__ uint32_t ffn_status_word;     // the device's status word of these operators (zc_ffn_status)
static_assert(POLL_LIMIT == ZC_FFN_WAIT_POLLS, "the limit that zc_ffn.h states");
std::atomic<uint32_t> wait_polls{POLL_LIMIT};      // of the launches that follow (zc_ffn_wait_limit)

constexpr uint32_t TILE_M = 128, THREADS = 320;           // rows of a CTA
constexpr uint32_t A_BYTES = TILE_M * 128;
constexpr uint32_t SF_COLUMNS = 32;                        // MX4: tensor-memory columns of a stage's scales: A 2 x 4, B 2 x 8 at most

struct TileMaps { CUtensorMap a[2], b[2], sfa, sfb[2], o[3]; };

// Division of n < 2^31 by a divisor known on the host, by the method of Granlund and Montgomery ("Division by invariant integers using multiplication",
// 1994): (umulhi(mul, n) + n) >> shift with mul = 2^32 (2^shift - d) / d + 1, 2^shift >= d. The tile of an index takes two; as divisions they stopped the copying thread for 1,000 clocks a tile.
struct Divisor {
    uint32_t d, mul, shift;
    void set(uint32_t by) {
        d = by;
        for (shift = 0; (1ull << shift) < d; ++shift) {}
        mul = uint32_t((((1ull << shift) - d) << 32) / d + 1);
    }
};
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& by) { return (__umulhi(by.mul, n) + n) >> by.shift; }

struct TilePlan {
    uint32_t M, N;                      // rows and columns of an output (gated: N = ffn)
    uint32_t kblocks, ksteps;           // stages of K; steps of 32 bytes in the last one
    uint32_t segs, outs;                // pairs (a[s], b[s]) whose products add up; outputs a[z] . b[0]
    uint32_t mtiles, ntiles, tiles;     // of 256 rows
    Divisor band, last;                 // tiles of a band of eight row tiles; row tiles of the last, shorter band
    uint32_t splits, kown;              // pairs that share a tile's K (then a cluster has one tile), stages of each
    uint32_t idesc;
    uint32_t polls;                     // of a wait
    uint32_t ktiles;                    // MX4: scale tiles along K
    void* out[2];
    uint64_t ldo;
    void *g, *u;                        // gated: where the two products go as well, or null
    int out_type, saved_type;           // of the outputs; of g and u
    bool aligned;                       // the output's rows start and end on 16 bytes: o[] are views of out[0], and of out[1], or of g and u
};

struct Tile { uint32_t z, m0, n0; };

// Bands of eight row tiles, walked column by column: what runs at one time shares few rows of A and of B in L2.
__device__ __forceinline__ Tile tile_at(const TilePlan& p, uint32_t t, uint32_t width) {
    const uint32_t per = p.mtiles * p.ntiles, z = t >= per, i = z ? t - per : t;      // (at most two outputs)
    const uint32_t band = quotient(i, p.band), j = i - band * p.band.d;
    const bool whole = band * 8 + 8 <= p.mtiles;
    const uint32_t column = whole ? j >> 3 : quotient(j, p.last), row = j - column * (whole ? 8 : p.last.d);
    return {z, (band * 8 + row) * 2 * TILE_M, column * width};
}

// A warp's 32 rows (one a lane) of eight columns, from (row, col) of the output on, turned through shared memory, so that eight lanes store
// consecutive columns; rows and columns past the last one are left out.
template <typename T> __device__ __forceinline__ void store_eight(T* out, const TilePlan& p, uint32_t row, uint32_t col, uint8_t* patch, const float (&v)[8]) {
    float* const turned = reinterpret_cast<float*>(patch);
    const uint32_t lane = threadIdx.x & 31, at = col + lane % 8;
    if (row >= p.M) return;
    const uint32_t rows = min(32u, p.M - row);
#pragma unroll
    for (int j = 0; j < 8; ++j) turned[lane * 9 + j] = v[j];
    __syncwarp();
    if (at < p.N)
        for (uint32_t r = lane / 8; r < rows; r += 4) out[uint64_t(row + r) * p.ldo + at] = from_f32<T>(turned[r * 9 + lane % 8]);
    __syncwarp();
}
__device__ __forceinline__ void store_eight_as(void* out, int type, const TilePlan& p, uint32_t row, uint32_t col, uint8_t* patch, const float (&v)[8]) {
    if (type == ZC_BF16) store_eight(static_cast<__nv_bfloat16*>(out), p, row, col, patch, v);
    else if (type == ZC_F16) store_eight(static_cast<__half*>(out), p, row, col, patch, v);
    else store_eight(static_cast<float*>(out), p, row, col, patch, v);
}
// The same for NC columns of rows that start anywhere: 128 bytes of each row as 32 words, row by row out of shared memory (33 words a row), a word a
// lane. A 16-bit row that starts between two words is shifted by half of one on the way; its first and its last value are stored alone. Eight
// rows at a time and without branches: what bounds it is how long a warp waits for its own instructions (8192 x 8191 of BF16 over 1024 k: 58 us, sixteen
// columns a round in FP32 98; aligned rows, by TMA, 37).
template <typename T, int NC> __device__ __forceinline__ void store_turned(T* out, const TilePlan& p, uint32_t row, uint32_t col, uint8_t* patch, const float (&v)[NC]) {
    constexpr int PER = 4 / sizeof(T), CHUNK = 32 * PER;      // values of a word, columns of a round
    uint32_t* const words = reinterpret_cast<uint32_t*>(patch);
    const uint32_t lane = threadIdx.x & 31, rows = min(32u, p.M - row);
#pragma unroll
    for (int c = 0; c < NC; c += CHUNK) {
        if (col + c >= p.N) break;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            alignas(4) T w[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) w[k] = from_f32<T>(v[c + j * PER + k]);
            words[lane * 33 + j] = *reinterpret_cast<const uint32_t*>(w);
        }
        __syncwarp();
        const uint32_t limit = min(uint32_t(CHUNK), p.N - col - c);
        T* to = out + uint64_t(row) * p.ldo + col + c;
#pragma unroll 1
        for (uint32_t r0 = 0; r0 < rows; r0 += 8) {
            uint32_t w[8], next[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) w[i] = words[(r0 + i) * 33 + lane];
            if constexpr (PER == 2) {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) next[i] = __shfl_down_sync(0xffffffffu, w[i], 1);
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i, to += p.ldo) {
                const uint32_t end = r0 + i < rows ? limit : 0;
                if constexpr (PER == 1) {
                    if (lane < end) *reinterpret_cast<uint32_t*>(to + lane) = w[i];
                } else {
                    uint16_t* const half = reinterpret_cast<uint16_t*>(to);
                    const uint32_t odd = uint32_t(reinterpret_cast<uintptr_t>(to) >> 1) & 1, at = lane * 2 + odd;
                    const uint32_t pair = odd ? __funnelshift_r(w[i], next[i], 16) : w[i];
                    if (at + 1 < end) *reinterpret_cast<uint32_t*>(half + at) = pair;
                    if (at + 1 == end) half[at] = uint16_t(pair);
                    if (odd && lane == 0 && end) half[0] = uint16_t(w[i]);
                }
            }
        }
        __syncwarp();
    }
}
// A warp's 32 rows (one a lane) of NC columns, from (row, col) of the output on; rows and columns past the last one are left out. Rows that start and
// end on 16 bytes leave by TMA: 128 (or 64) bytes of each through shared memory, swizzled so that neither side meets a bank twice.
// Stored by the lanes, 16 bytes of a row each, they took 6,200 clocks a tile, and the waits of the copying and the issuing
// thread queued behind them. Others (only results of MX4 products can have such rows: ANY) are turned.
template <bool ANY, typename T, int NC> __device__ __forceinline__ void store_rows(T* out, const CUtensorMap* map, const TilePlan& p, uint32_t row, uint32_t col, uint8_t* patch, const float (&v)[NC]) {
    const uint32_t lane = threadIdx.x & 31;
    if (row >= p.M) return;
    if (!ANY || p.aligned) {
        constexpr int GROUP = NC * int(sizeof(T)) < 128 ? NC : 128 / int(sizeof(T)), CHUNK = 16 / sizeof(T), BYTES = GROUP * sizeof(T);
#pragma unroll
        for (int c = 0; c < NC; c += GROUP) {
            if (col + c >= p.N) break;
            if (lane == 0) tma_store_read();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < GROUP / CHUNK; ++j) {
                alignas(16) T w[CHUNK];
#pragma unroll
                for (int k = 0; k < CHUNK; ++k) w[k] = from_f32<T>(v[c + j * CHUNK + k]);
                const uint32_t turn = BYTES == 128 ? lane & 7 : (lane >> 1) & 3;
                *reinterpret_cast<uint4*>(patch + lane * BYTES + ((j ^ turn) << 4)) = *reinterpret_cast<const uint4*>(w);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(map, smem_addr(patch), col + c, row);
        }
        return;
    }
    if constexpr (ANY) store_turned(out, p, row, col, patch, v);
}
template <bool ANY, int NC> __device__ __forceinline__ void store_as(void* out, int type, const CUtensorMap* map, const TilePlan& p, uint32_t row, uint32_t col, uint8_t* patch, const float (&v)[NC]) {
    if (type == ZC_BF16) store_rows<ANY>(static_cast<__nv_bfloat16*>(out), map, p, row, col, patch, v);
    else if (type == ZC_F16) store_rows<ANY>(static_cast<__half*>(out), map, p, row, col, patch, v);
    else store_rows<ANY>(static_cast<float*>(out), map, p, row, col, patch, v);
}
// The quotient by the fast reciprocal (2 ulp): with the rounded division the epilogue of a gated tile took 26,000 clocks, more than the products
// of 3,300 k. It gives 0 for a denominator beyond 2^126, so far below zero, where 1 + e^-v is e^-v to the last bit, silu(v) = v e^v, its exponential in two
// factors: neither of them leaves FP32's normal range before the result does.
constexpr float FAR_GATE = -64.0f;
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.0f + expf(-v)); }
__device__ __forceinline__ float silu_far(float v) {
    const float t = expf(0.5f * v);
    return v * t * t;
}
// v = silu(v) w. One branch for all values: chosen value by value, the far form cost the gated block of 2048 x 2048, 64 tokens, 2.8 us of 9.2.
template <int N> __device__ __forceinline__ void activate(float (&v)[N], const float (&w)[N]) {
    float low = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) low = fminf(low, v[i]);
    if (low < FAR_GATE) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (v[i] < FAR_GATE ? silu_far(v[i]) : silu(v[i])) * w[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = silu(v[i]) * w[i];
    }
}

// A stage is `depth` blocks of K, loaded and released together: with 128 columns a block is worth 256 clocks of products, and waiting for it,
// releasing it and going round cost the issuing thread 300 beside its products' 40 each.
//
// A CTA that waits for tensor memory while others wait for it could close a circle over two SMs (two clusters, each with one CTA that has its
// columns and one that has not). So no CTA here ever waits for another's columns: each takes at least the share of its SM's shared memory that it
// takes of the tensor memory, so that those that fit an SM together find their columns free. A tile CTA takes all 512, hence all of the shared memory: it
// has its SM alone, whatever else runs. A CTA of few tokens may meet those of other libraries; it holds its columns while it waits for nothing
// but its own copies and products.
constexpr uint32_t SM_SMEM = 228 * 1024, CTA_RESERVED = 1024, CTA_STATIC = 256, CTA_SMEM_MAX = 227 * 1024 - CTA_STATIC;
constexpr uint32_t smem_share(uint32_t tmem_columns) { return tmem_columns * (SM_SMEM / 512) - CTA_RESERVED - CTA_STATIC; }

template <bool MX4, bool GATED, int N> struct TileSmem {
    static constexpr uint32_t patch = MX4 ? 5120 : 4096;      // a warp's, of the epilogue: 32 rows of 128 bytes (of 33 words where rows are turned), on 1024 bytes
    static constexpr uint32_t b = N / 2 * 128, block = A_BYTES + b + (MX4 ? (1 + N / 128) * 1024 : 0), depth = N == 256 ? 1 : 2, stage = depth * block;
    static constexpr uint32_t stages = MX4 ? (N == 256 ? 5 : 3) : N == 256 ? 6 : 4, used = stages * stage + 8 * patch + 1024;
    static constexpr uint32_t bytes = smem_share(512);
    static constexpr bool shared = N == 128 || (MX4 && GATED);      // whether pairs may share a tile's K (the others are narrow where tiles are few)
    static_assert(used <= bytes && bytes <= CTA_SMEM_MAX, "shared memory of a tile CTA");
};

// The copying thread of a pair's leader, once a wait has run out: the leader's barriers count the bytes of both CTAs, which may have started different
// numbers of stages, `mine` and what the other CTA's thread leaves in *others, plus one, when it stops. What the other has started alone is expected
// here, what it has not started is counted off, so that every barrier of the last round flips when its copies have landed. (Without an answer the other
// has started all, and all of them have been used.) Until the leader is here, neither CTA passes the barrier behind which it ends.
__device__ __noinline__ void end_copies(uint64_t* full, uint32_t mine, const volatile uint32_t* others, uint32_t stages, uint32_t bytes) {
    for (uint32_t i = 0; i < POLL_LIMIT && !*others; ++i) {}
    const uint32_t theirs = *others ? *others - 1 : mine, most = max(mine, theirs);
    for (uint32_t f = most > stages ? most - stages : 0; f < most; ++f) {
        uint64_t* const bar = &full[f % stages];
        if (f >= mine) mbar_expect(bar, bytes);
        else if (f >= theirs) mbar_complete(bar, bytes);
        mbar_await(bar, (f / stages) & 1);
    }
}

template <bool MX4, bool A_MN, bool B_MN, bool GATED, int N>
__global__ void __launch_bounds__(THREADS, 1) tile_kernel(const __grid_constant__ TileMaps maps, const TilePlan p) {
    typedef TileSmem<MX4, GATED, N> Smem;
    constexpr uint32_t STAGES = Smem::stages, STAGE = Smem::stage, DEPTH = Smem::depth, ACC = MX4 && N == 256 ? 1 : 2, SF_COLUMN = ACC * N;
    constexpr uint32_t KB = MX4 ? 128 : 64;               // TMA elements of K a block (bytes of codes, 16-bit values)
    constexpr uint32_t WIDTH = GATED ? N / 2 : N;         // output columns of a tile
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[ACC], acc_empty[ACC], drain;       // (CTA_STATIC bytes at most)
    __shared__ uint32_t tmem_s, abort_s, others_s;       // others_s: see end_copies
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank() & 1, part = cluster_rank() >> 1, lead = part * 2;            // lead: the leader's rank in the cluster
    const uint32_t pair = cluster_index(), pairs = cluster_count();
    const uint32_t k0 = part * p.kown, k1 = min(k0 + p.kown, p.segs * p.kblocks);                     // of the stages of all segments
    const uint32_t seg0 = k0 >= p.kblocks, kb0 = k0 - (seg0 ? p.kblocks : 0);                         // (at most two segments)
    uint32_t* const status = &ffn_status_word;
    volatile uint32_t* const abort_flag = &abort_s;
    const auto give_up = [&] {      // by one thread of a role whose wait ran out: no other CTA of the cluster waits for its limit as well
        for (uint32_t r = 0; r < 2 * p.splits; ++r) store_cluster_word(map_to(smem_addr(&abort_s), r), 1);
    };
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (uint32_t i = 0; i < ACC; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 16); }
        mbar_init(&drain, 1);
        abort_s = others_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_s;
    pdl_wait();
    pdl_launch_dependents();

    if (warp == 0) {
        if (elect_one()) {
            uint32_t it = 0, slot = 0, round = 0;
            bool ok = true;
            for (uint32_t t = pair; ok && t < p.tiles; t += pairs) {
                const Tile c = tile_at(p, t, WIDTH);
                const int row = c.m0 + rank * TILE_M;                                       // of A
                const int col = GATED ? c.n0 : c.n0 + rank * (N / 2);                       // row of B (gated: the leader has gate's, the other up's)
                uint32_t seg = seg0, kb = kb0;
                for (uint32_t left = k1 - k0; left; --left, ++it) {
                    const CUtensorMap* const ma = &maps.a[p.outs == 2 ? c.z : seg];
                    const CUtensorMap* const mb = &maps.b[GATED ? rank : seg];
                    if (round && !mbar_wait(&empty[slot], (round - 1) & 1, abort_flag, status, p.polls)) { ok = false; break; }
                    const uint32_t bar = map_to(smem_addr(&full[slot]), lead);          // the leader counts the bytes of both
                    if (rank == 0) mbar_expect(&full[slot], 2 * STAGE);
#pragma unroll
                    for (uint32_t d = 0; d < DEPTH; ++d) {
                        const uint32_t a = ring + slot * STAGE + d * Smem::block, b = a + A_BYTES, k = kb * DEPTH + d;      // k: block of K (one past the end is zeros)
                        if constexpr (A_MN) {
                            for (uint32_t i = 0; i < 2; ++i) tma_load_2d_pair(a + i * 8192, ma, bar, row + i * 64, k * 64);
                        } else {
                            tma_load_2d_pair(a, ma, bar, k * KB, row);
                        }
                        if constexpr (B_MN) {
                            for (uint32_t i = 0; i < N / 128; ++i) tma_load_2d_pair(b + i * 8192, mb, bar, col + i * 64, k * 64);
                        } else {
                            tma_load_2d_pair(b, mb, bar, k * KB, col);
                        }
                        if constexpr (MX4) {      // two scale tiles (256 k) of this CTA's rows of A and of all rows of B
                            const uint32_t sf = b + Smem::b;
                            const int at = (c.n0 / 128) * p.ktiles + k * 2;
                            tma_load_2d_pair(sf, &maps.sfa, bar, 0, (row / 128) * p.ktiles + k * 2);
                            tma_load_2d_pair(sf + 1024, &maps.sfb[0], bar, 0, at);
                            if (N == 256) tma_load_2d_pair(sf + 2048, &maps.sfb[GATED ? 1 : 0], bar, 0, GATED ? at : at + p.ktiles);
                        }
                    }
                    if (++slot == STAGES) { slot = 0; ++round; }
                    if (++kb == p.kblocks) { kb = 0; ++seg; }
                }
            }
            const uint32_t last = slot ? slot - 1 : STAGES - 1;
            if (ok) ok = mbar_spin(&empty[last], (slot ? round : round - 1) & 1, abort_flag, status, p.polls);
            if (!ok) {
                give_up();
                if (rank) store_cluster_word(map_to(smem_addr(&others_s), lead), it + 1);
                else end_copies(full, it, &others_s, STAGES, STAGE);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            uint32_t n = 0, slot = 0, phase = 0;
            bool ok = true, ready = mbar_test(&full[0], 0);      // a stage ahead: the answer arrives while the products before it are issued
            for (uint32_t t = pair; ok && t < p.tiles; t += pairs, ++n) {
                const uint32_t buf = n % ACC, acc = tmem + buf * N;
                if (n >= ACC && !mbar_wait(&acc_empty[buf], (n / ACC - 1) & 1, abort_flag, status, p.polls)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t more = 0, kb = kb0;
                for (uint32_t left = k1 - k0; left; --left) {
                    const uint32_t stage = ring + slot * STAGE, now = slot;
                    if (!ready && !mbar_wait(&full[slot], phase, abort_flag, status, p.polls)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (++slot == STAGES) { slot = 0; phase ^= 1; }
                    ready = mbar_test(&full[slot], phase);
                    const uint32_t steps = kb + 1 == p.kblocks ? p.ksteps : 4 * DEPTH;
#pragma unroll
                    for (uint32_t d = 0; d < DEPTH; ++d) {
                        if (d * 4 >= steps) break;
                        const uint32_t a = stage + d * Smem::block, b = a + A_BYTES;
                        const uint64_t da = desc_at(A_MN ? DESC_MN_MAJOR : DESC_K_MAJOR, a), db = desc_at(B_MN ? DESC_MN_MAJOR : DESC_K_MAJOR, b);
                        const uint32_t sf = tmem + SF_COLUMN + now * SF_COLUMNS + d * (SF_COLUMNS / 2), sf_b = sf + 8, sf_step = N / 32;
                        if constexpr (MX4) {
                            // 128 k of scales: four columns for A's rows, four or eight for B's
                            const uint64_t ds = desc_at(DESC_SCALES, b + Smem::b);
#pragma unroll
                            for (uint32_t j = 0; j < 2; ++j) {
                                if (d * 4 + j * 2 >= steps) break;
                                tmem_copy_scales_pair(sf + j * 4, ds + j * 32);
#pragma unroll
                                for (uint32_t i = 0; i < N / 128; ++i) tmem_copy_scales_pair(sf_b + j * sf_step + i * 4, ds + 64 * (i + 1) + j * 32);
                            }
                        }
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) {
                            if (d * 4 + k >= steps) break;
                            if constexpr (MX4) {
                                constexpr uint32_t odd = 2u << 29 | 2u << 4;      // the upper two of a column's four scales
                                umma_mx4_pair(acc, da + k * 2, db + k * 2, k & 1 ? p.idesc | odd : p.idesc, sf + (k >> 1) * 4, sf_b + (k >> 1) * sf_step, more);
                            } else {
                                umma_f16_pair(acc, da + k * (A_MN ? 128 : 2), db + k * (B_MN ? 128 : 2), p.idesc, more);
                            }
                            more = 1;
                        }
                    }
                    if (++kb == p.kblocks) kb = 0;
                    umma_commit_pair(&empty[now], lead);
                }
                if (ok) umma_commit_pair(&acc_full[buf], lead);
            }
            if (!ok) give_up();
            umma_commit_lead(&drain);       // products read shared memory of both CTAs and write their tensor memory
            mbar_await(&drain, 0);
        }
        __syncwarp();
    } else {
        constexpr int COLS = WIDTH / 2;                                 // output columns of a warp
        const uint32_t half = (warp - 2) >> 2, quarter = warp & 3;      // which columns; the 32 lanes of tensor memory a warp can read
        uint8_t* const patch = raw + (ring - smem_addr(raw)) + STAGES * STAGE + (warp - 2) * Smem::patch;
        uint32_t n = 0;
        for (uint32_t t = pair; t < p.tiles; t += pairs, ++n) {
            const Tile c = tile_at(p, t, WIDTH);
            const uint32_t buf = n % ACC, acc = tmem + buf * N + (quarter << 21);
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (n / ACC) & 1, abort_flag, status, p.polls))) {
                if (lane == 0) give_up();
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float v[COLS], w[GATED ? COLS : 1];
#pragma unroll
            for (int i = 0; i < COLS; i += 32) {
                tmem_ld32(acc + half * COLS + i, v + i);
                if constexpr (GATED) tmem_ld32(acc + N / 2 + half * COLS + i, w + i);
            }
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_at(map_to(smem_addr(&acc_empty[buf]), lead));
            const uint32_t row = c.m0 + rank * TILE_M + quarter * 32, col = c.n0 + half * COLS;
            if (Smem::shared && p.splits > 1) {
                // The sums of this part of K, [column][row]; every stage of the ring has been read.
                float* const mine = reinterpret_cast<float*>(raw + (ring - smem_addr(raw))) + half * COLS * TILE_M + quarter * 32 + lane;
#pragma unroll
                for (int i = 0; i < COLS; ++i) {
                    mine[i * TILE_M] = v[i];
                    if constexpr (GATED) mine[(N / 2 + i) * TILE_M] = w[i];
                }
                continue;
            }
            if constexpr (GATED) {
                if (p.g) {
                    store_as<MX4>(p.g, p.saved_type, &maps.o[1], p, row, col, patch, v);
                    store_as<MX4>(p.u, p.saved_type, &maps.o[2], p, row, col, patch, w);
                }
                activate(v, w);
            }
            store_as<MX4>(c.z ? p.out[1] : p.out[0], p.out_type, &maps.o[c.z], p, row, col, patch, v);
        }
        if (lane == 0) tma_store_done();
        __syncwarp();
    }
    if constexpr (Smem::shared) {
        if (p.splits > 1) {
            // Every pair adds a part of the tile's columns over the pairs, in their order, eight columns a warp at a time.
            cluster_sync();
            if (warp >= 2 && __all_sync(0xffffffffu, !*abort_flag)) {
                const uint32_t quarter = warp & 3, share = WIDTH / p.splits;
                uint8_t* const patch = raw + (ring - smem_addr(raw)) + STAGES * STAGE + (warp - 2) * Smem::patch;
                const Tile c = tile_at(p, pair, WIDTH);
                const uint32_t row = c.m0 + rank * TILE_M + quarter * 32;
                // A warp without rows loads nothing, the others use all that they load: cluster_leave waits for no load.
                const uint32_t end = row < p.M ? (part + 1) * share : 0;
                for (uint32_t j = part * share + ((warp - 2) >> 2) * 8; j < end; j += 16) {
                    float v[8], w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = w[i] = 0.0f;
                    for (uint32_t r = 0; r < p.splits; ++r) {
                        const uint32_t from = map_to(ring + (j * TILE_M + quarter * 32 + lane) * 4, r * 2 + rank);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            v[i] += load_cluster(from + i * TILE_M * 4);
                            if constexpr (GATED) w[i] += load_cluster(from + (N / 2 + i) * TILE_M * 4);
                        }
                    }
                    if constexpr (GATED) {
                        if (p.g) {
                            store_eight_as(p.g, p.saved_type, p, row, c.n0 + j, patch, v);
                            store_eight_as(p.u, p.saved_type, p, row, c.n0 + j, patch, w);
                        }
                        activate(v, w);
                    }
                    store_eight_as(c.z ? p.out[1] : p.out[0], p.out_type, p, row, c.n0 + j, patch, v);
                }
            }
            __syncwarp();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (Smem::shared && p.splits > 1) cluster_leave();       // (the arrivals at the leader's barriers came before the sums)
    else cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---------------------------------------------------------------------------------------------
// Few tokens
// ---------------------------------------------------------------------------------------------
// D[M, tokens] = W . X^T: the weights are the 128 rows of a product, the tokens (64 at most, padded to a multiple of 16) its columns, so a single
// token costs the tensor cores an eighth of what 128 would and the launch is what its bytes are: the weights, once. A CTA owns one tile of 128 weight
// rows (of gate and of up) and one run of blocks of K; the CTAs of a cluster share a tile's K and add their partial sums through
// distributed shared memory, in the order of their ranks. The lanes of the epilogue hold consecutive output columns of a token, so plain
// stores are coalesced whatever the row stride.
// A handful of plain tokens: every CTA quantises its own part of their K into shared memory (the epilogue warps, while the weights arrive),
// in the swizzle TMA would have written; more are quantised by a launch of their own.
// The kernel before may still run while this one starts (programmatic launch): until it has ended nothing is read but into L2, where a later write
// of it would arrive too.
// What bounds it: one token, MX4 8192 x 4096, replayed back to back 6.1 us a call for 17.8 MB (2.7 us of HBM): 1.7 us until the first stage is there
// (all CTAs ask for all weights at once: 10 TB/s out of L2), 1.3 for the products, 0.7 for the sums, 0.6 to leave the cluster, 1.5 until the next
// kernel is let go. Sums written to the ranks that add them, one cluster barrier the less, came to 0.2 us more. (With all ends of copies and products
// waited for, 6.2.)
constexpr uint32_t FEW_THREADS = 192;
// Which calls: up to 64 tokens, unless K is short, where the tokens' sums over the cluster cost more than the weights. Rows x K, here / in tiles of pairs, us,
// of MX4 product | MX4 block (tokens microscaled) | 16-bit block. 2048 x 512: 25 tokens 4.1 / 3.7 | 5.7 / 6.2 | 7.2 / 7.2, 32 tokens 4.1 / 3.9 | 6.2 / 6.2 |
// 7.3 / 7.2, 33 tokens 4.6 / 3.9 | 6.7 / 6.2 | 8.2 / 7.3, 64 tokens 5.9 / 4.1 | 8.7 / 6.2 | 9.4 / 7.2. 1024 x 1024: 48 tokens 4.4 / 4.4 | 6.5 / 6.9 | 7.3 / 8.3,
// 64 tokens 5.1 / 4.4 | 7.2 / 6.7 | 8.2 / 8.2. 2048 x 2048: 33 tokens 5.2 / 4.9 | 7.7 / 8.2 | 9.9 / 10.3, 64 tokens 6.2 / 5.4 | 9.2 / 8.2 | 12.2 / 11.3.
// 1024 x 4096, 64 tokens: 5.4 / 6.7 | 7.7 / 8.7 | 11.3 / 12.3. 8192 x 8192, 64 tokens: 11.8 / 13.8 | 19.5 / 19.9 | 50 / 55. One rule for forms that cross over
// at different places; what it gives away: the MX4 product above (2048 x 2048, 33 tokens), few rows of K = 2048 (512 x 2048, 49 tokens 4.6 / 4.9 | 6.7 / 8.0 |
// 8.3 / 8.2; 64 tokens 4.9 / 5.1 | 7.2 / 8.2 | 9.3 / 8.2). dx, whose K is two segments, stays here up to 64 tokens (hidden x ffn, 2048 x 1024 9.3 / 11.3,
// 4096 x 4096 20 / 26, 2048 x 512 8.3 / 9.3).
constexpr uint32_t FEW_TOKENS = 64;
bool takes_few(uint32_t tokens, uint32_t k) { return tokens <= 32 || (tokens <= 48 && k > 512) || (tokens <= FEW_TOKENS && k > 2048); }
// What a ring may take where SMs have two CTAs, and its stages at most. A CTA that has its SM alone takes what there is (16-bit block of 16384 x 4096,
// 64 tokens: two stages 65 us, five 52), unless it is one of a cluster: sixteen clusters of eight such do not all fit (2048 x 2048: 9.9 us, 6.5).
constexpr uint32_t FEW_SMEM = 110 * 1024, FEW_STAGES = 6;
// x is quantised inside where a CTA has at most so many rows of 256 of its columns (tokens x blocks; the four warps share them): MX4 2048 x 512, one block a
// CTA, 1 / 4 / 8 / 12 / 16 tokens 3.1 / 3.2 / 4.0 / 4.7 / 5.2 us, by a launch of its own 4.1 / 4.1 / 4.2 / 4.7 / 4.9; 8192 x 4096, four blocks, 2 / 3 / 4
// tokens 7.0 / 7.6 / 8.2 and 8.2 / 8.4 / 8.4.
constexpr uint32_t FEW_PLAIN_ROWS = 12;
constexpr uint64_t FEW_AHEAD = 32ull << 20;                               // bytes of weights requested into L2 before the kernel before has ended

struct FewPlan {
    uint32_t M, tokens, n;              // weight rows, tokens, tokens padded
    uint32_t splits, kown;              // CTAs of a cluster, blocks of K of each
    uint32_t kblocks, segs, ksteps;     // blocks of a segment, segments, steps of a segment's last block
    uint32_t stages, stage, resident;   // ring; byte offset of the quantised tokens (0: they come through the ring)
    uint32_t smem;
    uint32_t tmem_columns, sf_column, sf_columns;
    uint32_t prefetch;                  // blocks of K to request into L2 ahead
    uint32_t idesc, ktiles, polls;
    const uint8_t *sfw[2], *sfx;
    const void* x;
    uint64_t x_ld;
    uint32_t x_dtype, cols;
    bool x_vec, out_vec;                // rows of x and of the output are aligned
    void *out, *g, *u;
    uint64_t ldo;
    int out_type, saved_type;
};

__device__ __forceinline__ void store_one(void* out, int type, uint64_t at, float v) {
    if (type == ZC_BF16) static_cast<__nv_bfloat16*>(out)[at] = from_f32<__nv_bfloat16>(v);
    else if (type == ZC_F16) static_cast<__half*>(out)[at] = from_f32<__half>(v);
    else static_cast<float*>(out)[at] = v;
}
// Four consecutive columns of a row, `valid` of which exist.
template <typename T> __device__ __forceinline__ void store_four(void* out, uint64_t at, uint32_t valid, bool vec, const float4& v) {
    T* const to = static_cast<T*>(out) + at;
    alignas(16) const T w[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    if (vec && valid >= 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(w);
        else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(w);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (j < valid) to[j] = w[j];
    }
}
__device__ __forceinline__ void store_four_as(void* out, int type, const FewPlan& p, uint64_t at, uint32_t valid, const float4& v) {
    if (type == ZC_BF16) store_four<__nv_bfloat16>(out, at, valid, p.out_vec, v);
    else if (type == ZC_F16) store_four<__half>(out, at, valid, p.out_vec, v);
    else store_four<float>(out, at, valid, p.out_vec, v);
}
template <bool GATED> __device__ __forceinline__ void few_store4(const FewPlan& p, uint64_t at, uint32_t valid, float4 a, const float4& b) {
    if constexpr (GATED) {
        if (p.g) { store_four_as(p.g, p.saved_type, p, at, valid, a); store_four_as(p.u, p.saved_type, p, at, valid, b); }
        float v[4] = {a.x, a.y, a.z, a.w};
        activate(v, {b.x, b.y, b.z, b.w});
        a = make_float4(v[0], v[1], v[2], v[3]);
    }
    store_four_as(p.out, p.out_type, p, at, valid, a);
}
__device__ __forceinline__ float4 load_peer(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_to(addr, rank)) : "memory");
    return v;
}
// The tokens' blocks [k0, k0 + blocks) of 256 columns into shared memory: per block n rows of 128 bytes, then two scale tiles. A warp takes a
// row of a block at a time, eight values a lane (four lanes share a scale). Padding rows stay as they are (their columns are not stored);
// columns past the last one become zero codes with a zero scale byte. The loop is not unrolled: a launch of a few microseconds waits for
// its instructions too (gated block of 512 x 2048, one token: 4.0 us, with four rows in flight 4.7).
template <typename T> __device__ __forceinline__ void quantise_tokens(const FewPlan& p, uint32_t k0, uint32_t blocks, uint8_t* to) {
    const uint32_t lane = threadIdx.x & 31, size = p.n * 128 + 1024, left = p.cols - k0 * 256;
    const T* const x = static_cast<const T*>(p.x) + uint64_t(k0) * 256;
#pragma unroll 1
    for (uint32_t t = 0, block = (threadIdx.x >> 5) - 2;; block += 4) {       // rows of blocks, token by token, dealt to the four warps in turn
        while (block >= blocks) { block -= blocks; ++t; }
        if (t >= p.tokens) break;
        const T* const row = x + uint64_t(t) * p.x_ld;
        const uint32_t at = block * 256 + lane * 8;
        float v[8] = {};
        if (at < left) p.x_vec ? load8<T, true>(row + at, v) : load8<T, false>(row + at, v);
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t s = mx4_scale(top);
        uint8_t* const b = to + block * size;
        *reinterpret_cast<uint32_t*>(b + t * 128 + (((lane >> 2) ^ (t & 7)) << 4) + (lane & 3) * 4) = mx4_codes8(v, s);
        if ((lane & 3) == 0) b[p.n * 128 + (lane >> 4) * 512 + (t & 31) * 16 + (t >> 5) * 4 + ((lane >> 2) & 3)] = uint8_t(s);
    }
}

template <bool MX4, bool A_MN, int MATS>
__global__ void __launch_bounds__(FEW_THREADS) few_kernel(const __grid_constant__ TileMaps maps, const FewPlan p) {
    constexpr uint32_t KB = MX4 ? 128 : 64;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t full[FEW_STAGES], empty[FEW_STAGES], acc_full, tokens_ready, drain;     // (CTA_STATIC bytes at most)
    __shared__ uint32_t tmem_s, abort_s;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* const ring_p = raw + (ring - smem_addr(raw));
    const uint32_t rank = cluster_rank(), m0 = cluster_index() * TILE_M;                // (a launch without clusters has clusters of one)
    const uint32_t k0 = rank * p.kown, k1 = min(k0 + p.kown, p.kblocks * p.segs);
    const uint32_t seg0 = k0 >= p.kblocks, kb0 = k0 - (seg0 ? p.kblocks : 0);           // (at most two segments)
    const bool fused = p.resident != 0;
    uint32_t* const status = &ffn_status_word;
    volatile uint32_t* const abort_flag = &abort_s;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < p.stages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&tokens_ready, 128);
        mbar_init(&drain, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_s)), "r"(p.tmem_columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 0 && elect_one()) {
        uint32_t seg = seg0, kb = kb0;
        for (uint32_t k = k0; k < min(k0 + p.prefetch, k1); ++k) {
            for (uint32_t i = 0; i < MATS; ++i) {
                if constexpr (A_MN) {
                    prefetch_2d(&maps.a[seg], m0, kb * 64);
                    if (m0 + 64 < p.M) prefetch_2d(&maps.a[seg], m0 + 64, kb * 64);
                } else {
                    prefetch_2d(&maps.a[i], kb * KB, m0);
                }
                if constexpr (MX4) prefetch_bulk(p.sfw[i] + (uint64_t(m0 / 128) * p.ktiles + kb * 2) * 512, min(2u, p.ktiles - kb * 2) * 512);
            }
            if (++kb == p.kblocks) { kb = 0; ++seg; }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_s;
    pdl_wait();
    pdl_launch_dependents();

    const uint32_t b_bytes = fused ? 0 : p.n * 128;      // token rows of a stage
    const uint32_t sf_off = MATS * A_BYTES + b_bytes;
    if (warp == 0) {
        if (elect_one()) {
            // slot, its round, segment and block are counted, not divided for: a division a stage is what the loop would wait for
            uint32_t it = 0, slot = 0, round = 0, seg = seg0, kb = kb0;
            bool ok = true;
            for (uint32_t k = k0; k < k1; ++k, ++it) {
                const uint32_t a = ring + slot * p.stage;
                if (round && !mbar_wait(&empty[slot], (round - 1) & 1, abort_flag, status, p.polls)) { ok = false; break; }
                const uint32_t atoms = MX4 ? min(2u, p.ktiles - kb * 2) : 0;
                mbar_expect(&full[slot], MATS * A_BYTES + b_bytes + atoms * 512 * (MATS + (fused ? 0 : 1)));
#pragma unroll
                for (uint32_t i = 0; i < MATS; ++i) {
                    if constexpr (A_MN) {
                        tma_load_2d(a, &maps.a[seg], &full[slot], m0, kb * 64);
                        tma_load_2d(a + 8192, &maps.a[seg], &full[slot], m0 + 64, kb * 64);
                    } else {
                        tma_load_2d(a + i * A_BYTES, &maps.a[i], &full[slot], kb * KB, m0);
                    }
                    if constexpr (MX4) bulk_load(a + sf_off + i * 1024, p.sfw[i] + (uint64_t(m0 / 128) * p.ktiles + kb * 2) * 512, atoms * 512, &full[slot]);
                }
                if (!fused) {
                    tma_load_2d(a + MATS * A_BYTES, &maps.b[seg], &full[slot], kb * KB, 0);
                    if constexpr (MX4) bulk_load(a + sf_off + MATS * 1024, p.sfx + uint64_t(kb) * 1024, atoms * 512, &full[slot]);
                }
                if (++slot == p.stages) { slot = 0; ++round; }
                if (++kb == p.kblocks) { kb = 0; ++seg; }
            }
            const uint32_t last = slot ? slot - 1 : p.stages - 1;
            if (ok) ok = mbar_spin(&empty[last], (slot ? round : round - 1) & 1, abort_flag, status, p.polls);
            if (!ok)
                for (uint32_t f = it > p.stages ? it - p.stages : 0; f < it; ++f) mbar_await(&full[f % p.stages], (f / p.stages) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            bool ok = !fused || mbar_wait(&tokens_ready, 0, abort_flag, status, p.polls);
            uint32_t slot = 0, phase = 0, kb = kb0, more = 0;
            uint32_t quantised = ring + p.resident;
            bool ready = mbar_test(&full[0], 0);
            for (uint32_t k = k0; ok && k < k1; ++k) {
                const uint32_t a = ring + slot * p.stage, now = slot;
                if (!ready && !mbar_wait(&full[slot], phase, abort_flag, status, p.polls)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (++slot == p.stages) { slot = 0; phase ^= 1; }
                ready = mbar_test(&full[slot], phase);
                const uint32_t b = fused ? quantised : a + MATS * A_BYTES;
                const uint32_t sfb = fused ? b + p.n * 128 : a + sf_off + MATS * 1024;
                const uint32_t steps = kb + 1 == p.kblocks ? p.ksteps : 4, sf = tmem + p.sf_column + now * p.sf_columns;
                const uint64_t db = desc_at(DESC_K_MAJOR, b), da = desc_at(A_MN ? DESC_MN_MAJOR : DESC_K_MAJOR, a);
                if constexpr (MX4) {
                    const uint64_t dsa = desc_at(DESC_SCALES, a + sf_off), dsb = desc_at(DESC_SCALES, sfb);
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j) {
                        if (j * 2 >= steps) break;
#pragma unroll
                        for (uint32_t i = 0; i < MATS; ++i) tmem_copy_scales(sf + i * 8 + j * 4, dsa + i * 64 + j * 32);
                        tmem_copy_scales(sf + MATS * 8 + j * 4, dsb + j * 32);
                    }
                }
#pragma unroll
                for (uint32_t s = 0; s < 4; ++s) {
                    if (s >= steps) break;
#pragma unroll
                    for (uint32_t i = 0; i < MATS; ++i) {
                        if constexpr (MX4) {
                            constexpr uint32_t odd = 2u << 29 | 2u << 4;
                            umma_mx4(tmem + i * p.n, da + i * (A_BYTES >> 4) + s * 2, db + s * 2, s & 1 ? p.idesc | odd : p.idesc, sf + i * 8 + (s >> 1) * 4,
                                     sf + MATS * 8 + (s >> 1) * 4, more);
                        } else {
                            umma_f16(tmem + i * p.n, da + i * (A_BYTES >> 4) + s * (A_MN ? 128 : 2), db + s * 2, p.idesc, more);
                        }
                    }
                    more = 1;
                }
                umma_commit(&empty[now]);
                if (++kb == p.kblocks) kb = 0;
                quantised += p.n * 128 + 1024;
            }
            uint64_t* const end = ok ? &acc_full : &drain;
            umma_commit(end);
            mbar_await(end, 0);
        }
        __syncwarp();
    } else {
        if (MX4 && fused) {
            uint8_t* const to = ring_p + p.resident;
            if (p.x_dtype == ZC_BF16) quantise_tokens<__nv_bfloat16>(p, k0, k1 - k0, to);
            else if (p.x_dtype == ZC_F16) quantise_tokens<__half>(p, k0, k1 - k0, to);
            else quantise_tokens<float>(p, k0, k1 - k0, to);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&tokens_ready);
        }
        const uint32_t quarter = warp & 3, row = quarter * 32 + lane;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full, 0, abort_flag, status, p.polls));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float* const part = reinterpret_cast<float*>(ring_p);        // [matrix][token][row]: every stage has been read when the products are done
        for (uint32_t t0 = 0; ok && t0 < p.tokens; t0 += 16) {
            uint32_t bits[MATS][16];
#pragma unroll
            for (uint32_t i = 0; i < MATS; ++i) tmem_ld16(tmem + (quarter << 21) + i * p.n + t0, bits[i]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            float v[MATS][16];
#pragma unroll
            for (uint32_t i = 0; i < MATS; ++i)
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) v[i][j] = __uint_as_float(bits[i][j]);
            if (p.splits > 1) {
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    if (t0 + j >= p.tokens) break;
#pragma unroll
                    for (uint32_t i = 0; i < MATS; ++i) part[(i * p.tokens + t0 + j) * 128 + row] = v[i][j];
                }
            } else if (m0 + row < p.M) {
                const uint64_t to = uint64_t(t0) * p.ldo + m0 + row;
                if constexpr (MATS == 2) {
                    if (p.g) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) {
                            if (t0 + j >= p.tokens) break;
                            store_one(p.g, p.saved_type, to + j * p.ldo, v[0][j]);
                            store_one(p.u, p.saved_type, to + j * p.ldo, v[1][j]);
                        }
                    }
                    activate(v[0], v[1]);       // (padding too, which is not stored)
                }
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    if (t0 + j >= p.tokens) break;
                    store_one(p.out, p.out_type, to + j * p.ldo, v[0][j]);
                }
            }
            __syncwarp();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    // The columns go back as soon as they are read, before the cluster is waited for: a kernel of another library that waits for them, on a CTA of whose
    // cluster another CTA here waits, gets them. (The warps that read them only arrive; with a barrier of the whole CTA a call took 0.1 us more.)
    if (warp == 1) {
        if (p.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("bar.sync 1, 160;" ::: "memory");
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_columns) : "memory");
        if (p.splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        if (warp >= 2) asm volatile("bar.arrive 1, 160;" ::: "memory");
        if (p.splits > 1) cluster_sync();
    }
    if (p.splits > 1) {
        // Sums that are not stored are not loaded either: cluster_leave waits for no load, so each of them has to be used before it.
        const uint32_t row = lane * 4;               // four rows a lane, a token a warp
        if (warp >= 2 && m0 + row < p.M && !*abort_flag) {
            for (uint32_t t = rank + (warp - 2) * p.splits; t < p.tokens; t += 4 * p.splits) {
                float4 v[MATS];
#pragma unroll
                for (uint32_t i = 0; i < MATS; ++i) {
                    float4 each[8];
#pragma unroll
                    for (uint32_t r = 0; r < 8; ++r)
                        if (r < p.splits) each[r] = load_peer(ring + ((i * p.tokens + t) * 128 + row) * 4, r);
                    v[i] = each[0];
#pragma unroll
                    for (uint32_t r = 1; r < 8; ++r)
                        if (r < p.splits) { v[i].x += each[r].x; v[i].y += each[r].y; v[i].z += each[r].z; v[i].w += each[r].w; }
                }
                few_store4<MATS == 2>(p, uint64_t(t) * p.ldo + m0 + row, p.M - m0 - row, v[0], v[MATS - 1]);
            }
        }
        __syncwarp();
        cluster_leave();         // no CTA leaves while another may still read its sums
    }
}

// dg = dh u s (1 + g (1 - s)), du = dh g s, in FP32; rounded to the operands' type, as the tensor cores take them (the gradients' error is that
// rounding and their own). Bound by memory: 14 bytes a value with g and u in FP32, 10 with 16 bits. A warp takes 256 columns of a row: 8191 x 8192
// 141 us (6.7 TB/s), 106 us with 16 bits; two or four rows a warp 111 and 145 us with 16 bits.
template <typename T, typename S> __global__ void __launch_bounds__(256) gated_gradient_kernel(const T* __restrict__ dh, uint64_t dh_ld, const S* __restrict__ g, const S* __restrict__ u,
                                                                                               uint32_t tokens, uint32_t ffn, T* __restrict__ dg, T* __restrict__ du) {
    const uint32_t col = blockIdx.y * 256 + (threadIdx.x & 31) * 8;
    const uint64_t row = uint64_t(blockIdx.x) * 8 + (threadIdx.x >> 5), at = row * ffn + col;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= tokens || col >= ffn) return;
    float a[8], b[8], c[8];
    alignas(16) T d[8], e[8];
    load8<T, true>(dh + row * dh_ld + col, a);
    load8<S, true>(g + at, b);
    load8<S, true>(u + at, c);
    float low = b[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) low = fminf(low, b[j]);
    if (low < FAR_GATE) {       // (one branch, as in activate: chosen value by value the far form took 12 us more with g and u in 16 bits)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool far = b[j] < FAR_GATE;       // there s = t^2, multiplied in one factor at a time, and 1 - s is 1
            const float t = __expf(far ? 0.5f * b[j] : -b[j]), s = far ? t : __fdividef(1.0f, 1.0f + t), rest = far ? t : 1.0f;
            d[j] = from_f32<T>(a[j] * c[j] * s * (1.0f + b[j] * (1.0f - (far ? 0.0f : s))) * rest);
            e[j] = from_f32<T>(a[j] * b[j] * s * rest);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float s = __fdividef(1.0f, 1.0f + __expf(-b[j]));
            d[j] = from_f32<T>(a[j] * c[j] * s * (1.0f + b[j] * (1.0f - s)));
            e[j] = from_f32<T>(a[j] * b[j] * s);
        }
    }
    *reinterpret_cast<uint4*>(dg + at) = *reinterpret_cast<const uint4*>(d);
    *reinterpret_cast<uint4*>(du + at) = *reinterpret_cast<const uint4*>(e);
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
bool map_codes(CUtensorMap& m, const void* codes, uint32_t rows, uint32_t cols, uint32_t box) { return make_map(m, codes, true, cols / 2, rows, cols / 2, box); }
// Scale tiles as rows of 512 bytes, two a box.
bool map_scales(CUtensorMap& m, const void* scales, uint32_t rows, uint32_t cols) {
    const Encode encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {128, mx4_scale_bytes(rows, cols) / 512}, strides[1] = {512};
    const cuuint32_t box[2] = {128, 2}, elem[2] = {1, 1};
    return encode(&m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A 16-bit operand [rows, cols]: K along its rows (boxes of 64 k x `box` rows), or across them (boxes of 64 columns x 64 k).
bool map_rows(CUtensorMap& m, const void* p, uint32_t rows, uint32_t cols, uint64_t ld, uint32_t box) { return make_map(m, p, false, cols, rows, ld * 2, box); }
constexpr uint32_t ACROSS = 64;

// Instruction descriptors. Both: N / 8 from bit 17, M / 16 from bit 24 (M = 128 of one CTA, 256 of a pair).
uint32_t idesc_f16(int dtype, bool a_mn, bool b_mn, uint32_t m, uint32_t n) {      // FP32 accumulators; operand types; which operand has M / N along its rows
    const uint32_t t = dtype == ZC_BF16 ? 1 : 0;
    return (1u << 4) | (t << 7) | (t << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | ((n / 8) << 17) | ((m / 16) << 24);
}
uint32_t idesc_mx4(uint32_t m, uint32_t n) { return (1u << 7) | (1u << 10) | ((n / 8) << 17) | (1u << 23) | ((m / 16) << 24); }      // e2m1 both, e8m0 scales

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

int no_maps() { return fail(nullptr, ZC_EEXEC, "the driver did not encode a tensor map"); }
// The output in boxes of 32 rows x 128 bytes, or of what a warp has of a row.
bool map_output(CUtensorMap& m, void* out, int type, const TilePlan& p, uint32_t columns) {
    const Encode encode = tensor_map_encoder();
    if (!encode) return false;
    const uint32_t elem_bytes = uint32_t(dtype_bytes(type)), most = 128 / elem_bytes;
    const cuuint64_t dims[2] = {p.N, p.M}, strides[1] = {p.ldo * elem_bytes};
    const cuuint32_t box[2] = {columns < most ? columns : most, 32}, elem[2] = {1, 1};
    return encode(&m, elem_bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, out, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  columns < most ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The opt-in to large shared memory of one kernel, and the clusters of 4 and 8 CTAs of it that the device holds at a time, once per device.
struct Configured {
    std::atomic<bool> done[MAX_DEVICES] = {};
    std::atomic<uint32_t> clusters[MAX_DEVICES][2] = {};
    template <typename Kernel> int once(Kernel kernel, int device, size_t smem, uint32_t threads, bool count) {
        if (done[device].load(std::memory_order_acquire)) return ZC_OK;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        for (int i = 0; e == cudaSuccess && count && i < 2; ++i) {
            cudaLaunchConfig_t cfg{};
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 4u << i; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
            cfg.gridDim = dim3(4u << i); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.attrs = &attr; cfg.numAttrs = 1;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
            clusters[device][i].store(uint32_t(n), std::memory_order_relaxed);
        }
        if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("dense product set-up: ") + cudaGetErrorString(e)); }
        done[device].store(true, std::memory_order_release);
        return ZC_OK;
    }
};

template <bool MX4, bool A_MN, bool B_MN, bool GATED, int N> int launch_tiles(TileMaps& maps, TilePlan& p, const Device& d, cudaStream_t s) {
    static Configured configured;
    auto kernel = tile_kernel<MX4, A_MN, B_MN, GATED, N>;
    constexpr uint32_t smem = TileSmem<MX4, GATED, N>::bytes;
    const int rc = configured.once(kernel, d.index, smem, THREADS, TileSmem<MX4, GATED, N>::shared);
    if (rc != ZC_OK) return rc;
    void* const to[3] = {p.out[0], p.g ? p.g : p.out[1], p.u};
    // A TMA store writes whole 16-byte pieces: rows start and end on one (the other outputs are contiguous and aligned wherever they are given).
    p.aligned = rows16(p.out[0], p.ldo, dtype_bytes(p.out_type)) && p.N * dtype_bytes(p.out_type) % 16 == 0;
    for (int i = 0; i < 3 && p.aligned; ++i)
        if (to[i] && !map_output(maps.o[i], to[i], p.g && i ? p.saved_type : p.out_type, p, GATED ? N / 4 : N / 2)) return no_maps();
    p.polls = wait_polls.load(std::memory_order_relaxed);
    const uint32_t pairs = d.sms / 2, total = p.segs * p.kblocks;
    // K is shared by four or two pairs where all of the tiles still run at once and it is long enough to pay for the sums: narrow tiles, four pairs
    // from 12 stages on (16-bit 256 x 2048 x 512, 16 stages 8.6 us, shared by none 9.8; of 12 stages 8.3 and 8.7; of 8 stages 7.8 and 7.2), two from 18
    // (512 x 3000 x 1000, 24 stages 14.5 and 18.6; of 20 stages 11.3 and 12.3; of 12 stages 9.8 and 9.2); wide ones, whose sums are twice as many, 16 (MX4
    // gated 300 x 4000 x 600 11.3 and 12.8; of 8 stages 10.1 and 8.7) and 32 (512 x 8192 x 1536 15.0 and 16.4; of 16 stages 12.3 and 10.9).
    typedef TileSmem<MX4, GATED, N> Smem;
    p.splits = 1;
    if (Smem::shared && p.tiles <= configured.clusters[d.index][1] && total >= (Smem::depth == 2 ? 12 : 16)) p.splits = 4;
    else if (Smem::shared && p.tiles <= configured.clusters[d.index][0] && total >= (Smem::depth == 2 ? 18 : 32)) p.splits = 2;
    p.kown = (total + p.splits - 1) / p.splits;
    return launched(launch_after(kernel, dim3(2 * p.splits * (p.splits > 1 || p.tiles < pairs ? p.tiles : pairs)), THREADS, smem, 2 * p.splits, s, maps, p), "dense product");
}

// Tiles of `width` output columns; the number of them, or 0 where there are too many.
uint32_t set_tiles(TilePlan& p, uint32_t width) {
    p.mtiles = uint32_t((uint64_t(p.M) + 2 * TILE_M - 1) / (2 * TILE_M));
    p.ntiles = (p.N + width - 1) / width;
    const uint64_t tiles = uint64_t(p.mtiles) * p.ntiles * p.outs;
    p.band.set(p.ntiles <= 0x0fffffffu ? 8 * p.ntiles : 1);
    p.last.set(p.mtiles % 8 ? p.mtiles % 8 : 8);
    return p.tiles = tiles > 0x7fffffffu ? 0 : uint32_t(tiles);
}
// Whether 128 columns a tile: where 256 leave half of the pairs without one.
bool narrow_tiles(TilePlan& p, const Device& d, uint32_t per_output) {
    return set_tiles(p, 256 / per_output) <= d.sms / 4;
}
int too_many() { return fail(nullptr, ZC_EINVAL, "too many output tiles"); }

// K in blocks of `block` (`steps` steps of the tensor cores each); the steps of the last one.
template <typename Plan> void set_k(Plan& p, uint32_t k, uint32_t block, uint32_t steps = 4) {
    p.kblocks = (k + block - 1) / block;
    const uint32_t left = k - (p.kblocks - 1) * block, step = block / steps;
    p.ksteps = (left + step - 1) / step;
}
void set_tile_k(TilePlan& p, uint32_t k, uint32_t block, bool narrow) { narrow ? set_k(p, k, 2 * block, 8) : set_k(p, k, block); }

// Cuts a call of few tokens. kblocks, ksteps, segs, M, tokens, cols are set; plain: x is to be quantised.
void plan_few(FewPlan& p, bool mx4, uint32_t mats, bool plain, uint32_t sms) {
    p.n = (p.tokens + 15) / 16 * 16;
    const uint32_t total = p.kblocks * p.segs, mtiles = (p.M + TILE_M - 1) / TILE_M;
    // Two CTAs an SM: 8192 x 4096, one token 6.4 us, with one CTA an SM 7.5. Where the tiles alone fill three quarters of the SMs, more than sixteen
    // tokens are not split: their sums cost more than the second CTA brings. Rows x K, in two / in one, us, of MX4 product | MX4 block (tokens microscaled) |
    // 16-bit block | dx: 14336 x 512, 17 tokens 5.1 / 3.6 | 7.2 / 5.9 | 9.3 / 8.6 | 10.3 / 9.3; 16384 x 2048, 17 tokens 6.7 / 5.7 | 10.2 / 9.3 |
    // 26.6 / 25.6 | 27.7 / 26.7, 32 tokens 7.1 / 6.1 | 10.5 / 9.6 | 27.7 / 26.0; 16384 x 8192, 64 tokens 19.3 / 16.9 | 32.8 / 30.0 | 92.3 / 87.2; against
    // the rule 18904 x 1024, 17 tokens 5.7 / 4.1 | 8.2 / 7.5 | 17.6 / 18.3 | 20.5 / 19.9. Up to sixteen it depends: 16384 x 2048, one token 5.8 / 5.7 |
    // 8.3 / 8.3 | 24.9 / 25.0, 16 tokens of dx 26.8 / 26.2, but one plain token, of which every CTA would quantise twice as much, 5.7 / 6.2 | 8.3 / 10.7.
    uint32_t splits = p.tokens > 16 && mtiles >= sms * 3 / 4 ? 1 : 2 * sms / mtiles;
    splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;
    if (splits > total) splits = total;
    p.kown = (total + splits - 1) / splits;
    p.splits = (total + p.kown - 1) / p.kown;
    const uint32_t quantised = p.kown * (p.n * 128 + 1024);
    const bool fused = plain && p.tokens * p.kown <= FEW_PLAIN_ROWS;
    p.stage = mats * (A_BYTES + (mx4 ? 1024 : 0)) + (fused ? 0 : p.n * 128 + (mx4 ? 1024 : 0));
    const uint32_t room = (p.splits == 1 && mtiles <= sms ? CTA_SMEM_MAX : FEW_SMEM) - 1024 - (fused ? quantised : 0);
    p.stages = room / p.stage;
    if (p.stages > FEW_STAGES) p.stages = FEW_STAGES;
    if (p.stages > p.kown) p.stages = p.kown;
    uint32_t bytes = p.stages * p.stage;
    const uint32_t sums = p.splits > 1 ? mats * p.tokens * 512 : 0;
    if (!fused && bytes < sums) bytes = sums;
    p.resident = fused ? (bytes > sums ? bytes : (sums + 1023) / 1024 * 1024) : 0;
    p.smem = 1024 + (fused ? p.resident + quantised : bytes);
    p.sf_column = mats * p.n;
    p.sf_columns = mx4 ? mats * 8 + 8 : 0;
    p.tmem_columns = 32;
    while (p.tmem_columns < p.sf_column + p.stages * p.sf_columns) p.tmem_columns *= 2;
    if (p.smem < smem_share(p.tmem_columns)) p.smem = smem_share(p.tmem_columns);
    const uint64_t ahead = FEW_AHEAD / (uint64_t(mtiles) * p.splits * mats * A_BYTES);
    p.prefetch = ahead < p.kown ? uint32_t(ahead) : p.kown;
}

template <bool MX4, bool A_MN, int MATS> int launch_few(const TileMaps& maps, FewPlan& p, const Device& d, cudaStream_t s) {
    static Configured configured;
    p.out_vec = rows16(p.out, p.ldo, dtype_bytes(p.out_type));
    p.polls = wait_polls.load(std::memory_order_relaxed);
    auto kernel = few_kernel<MX4, A_MN, MATS>;
    const int rc = configured.once(kernel, d.index, CTA_SMEM_MAX, FEW_THREADS, false);
    if (rc != ZC_OK) return rc;
    return launched(launch_after(kernel, dim3((p.M + TILE_M - 1) / TILE_M * p.splits), FEW_THREADS, p.smem, p.splits, s, maps, p), "dense product of few tokens");
}

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
    if (tokens == 1) { x_ld = cols; out_ld = rows; }
    const Span os = matrix_span(out, out_dtype, tokens, rows, out_ld), cs{x_codes, uint64_t(tokens) * cols / 2}, ss{x_scales, mx4_scale_bytes(tokens, cols)};
    const Span xs = x ? matrix_span(x, x_dtype, tokens, cols, x_ld) : Span{nullptr, 0};
    bool bad = overlap(os, cs) || overlap(os, ss) || overlap(os, xs) || (x && (overlap(cs, ss) || overlap(cs, xs) || overlap(ss, xs)));
    for (int i = 0; i < mats; ++i)
        for (const Span& t : {Span{w[i].codes, uint64_t(rows) * cols / 2}, Span{w[i].scales, mx4_scale_bytes(rows, cols)}})
            bad = bad || overlap(os, t) || (x && (overlap(cs, t) || overlap(ss, t)));
    if (bad) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Device d;
    if ((rc = current_device(d)) != ZC_OK) return rc;
    TileMaps maps{};
    if (takes_few(tokens, cols)) {
        FewPlan p{};
        p.M = rows; p.tokens = tokens; p.segs = 1;
        set_k(p, cols, 256);
        plan_few(p, true, mats, x != nullptr, d.sms);
        if (x && !p.resident && (rc = launch_mx4_quantize(x, x_dtype, tokens, cols, x_ld, x_codes, x_scales, s)) != ZC_OK) return rc;
        for (int i = 0; i < mats; ++i) {
            if (!map_codes(maps.a[i], w[i].codes, rows, cols, TILE_M)) return no_maps();
            p.sfw[i] = static_cast<const uint8_t*>(w[i].scales);
        }
        if (!p.resident && !map_codes(maps.b[0], x_codes, tokens, cols, p.n)) return no_maps();
        p.idesc = idesc_mx4(TILE_M, p.n);
        p.ktiles = (cols + 127) / 128;
        p.sfx = static_cast<const uint8_t*>(x_scales);
        p.x = x; p.x_ld = x_ld; p.x_dtype = x_dtype; p.cols = cols;
        p.x_vec = x && rows16(x, x_ld, dtype_bytes(x_dtype));
        p.out = out; p.ldo = out_ld; p.out_type = out_dtype;
        return mats == 2 ? launch_few<true, false, 2>(maps, p, d, s) : launch_few<true, false, 1>(maps, p, d, s);
    }
    if (x && (rc = launch_mx4_quantize(x, x_dtype, tokens, cols, x_ld, x_codes, x_scales, s)) != ZC_OK) return rc;
    TilePlan p{};
    p.M = tokens; p.N = rows; p.segs = 1; p.outs = 1;
    p.ktiles = (cols + 127) / 128;
    p.out[0] = out; p.ldo = out_ld; p.out_type = out_dtype;
    const bool narrow = mats == 1 && narrow_tiles(p, d, 1);        // gated: 64 rows each of gate and up would share a scale tile
    const uint32_t n = narrow ? 128 : 256;
    if (!set_tiles(p, n / mats)) return too_many();
    set_tile_k(p, cols, 256, narrow);
    p.idesc = idesc_mx4(256, n);
    if (!map_codes(maps.a[0], x_codes, tokens, cols, TILE_M) || !map_scales(maps.sfa, x_scales, tokens, cols)) return no_maps();
    for (int i = 0; i < mats; ++i)
        if (!map_codes(maps.b[i], w[i].codes, rows, cols, n / 2) || !map_scales(maps.sfb[i], w[i].scales, rows, cols)) return no_maps();
    if (mats == 2) return launch_tiles<true, false, false, true, 256>(maps, p, d, s);
    return narrow ? launch_tiles<true, false, false, false, 128>(maps, p, d, s) : launch_tiles<true, false, false, false, 256>(maps, p, d, s);
}

int check_gated(const char* who, int dtype, uint32_t hidden, uint32_t ffn) {
    if (dtype != ZC_BF16 && dtype != ZC_F16) return fail(nullptr, ZC_EINVAL, std::string(who) + ": dtype must be BF16 or F16");
    if (!hidden || hidden % 8 || hidden > MAX_COLS || !ffn || ffn % 8 || ffn > MAX_COLS)
        return fail(nullptr, ZC_EINVAL, std::string(who) + ": hidden and ffn must be multiples of 8, from 8 to 1048576");
    return ZC_OK;
}
// g and u: where the operands' type or FP32.
int check_saved(const char* who, const void* g, const void* u, int dtype, int saved_dtype) {
    if (saved_dtype != dtype && saved_dtype != ZC_F32) return fail(nullptr, ZC_EINVAL, std::string(who) + ": g and u must be F32 or of the operands' dtype");
    if (misaligned(g) || misaligned(u)) return fail(nullptr, ZC_EINVAL, std::string(who) + ": buffers must be 16-byte aligned");
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
                     int saved_dtype, void* stream) {
    const char* who = "zc_gated_forward";
    int rc = check_gated(who, dtype, hidden, ffn);
    if (rc == ZC_OK) rc = check_matrix(who, x, dtype, tokens, hidden, x_ld, true);
    for (const void* w : {gate, up}) if (rc == ZC_OK) rc = check_matrix(who, w, dtype, ffn, hidden, hidden, true);
    if (rc == ZC_OK) rc = check_matrix(who, h, dtype, tokens, ffn, ffn, true);
    if (rc == ZC_OK && tokens && !g != !u) rc = fail(nullptr, ZC_EINVAL, std::string(who) + ": g and u go together");
    if (rc == ZC_OK && (g || u)) rc = check_saved(who, g, u, dtype, saved_dtype);
    if (rc != ZC_OK || !tokens) return rc;
    if (tokens == 1) x_ld = hidden;
    const uint64_t tf = uint64_t(tokens) * ffn * 2, fh = uint64_t(ffn) * hidden * 2, ts = uint64_t(tokens) * ffn * dtype_bytes(saved_dtype);
    const Span in[3] = {{x, matrix_bytes(dtype, tokens, hidden, x_ld)}, {gate, fh}, {up, fh}}, to[3] = {{h, tf}, {g, ts}, {u, ts}};
    for (int i = 0; i < 3; ++i) {
        for (const Span& v : in) if (overlap(to[i], v)) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
        for (int j = 0; j < i; ++j) if (overlap(to[i], to[j])) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    }
    Device d;
    if ((rc = current_device(d)) != ZC_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    TileMaps maps{};
    if (takes_few(tokens, hidden)) {
        FewPlan p{};
        p.M = ffn; p.tokens = tokens; p.segs = 1;
        set_k(p, hidden, 64);
        plan_few(p, false, 2, false, d.sms);
        if (!map_rows(maps.a[0], gate, ffn, hidden, hidden, TILE_M) || !map_rows(maps.a[1], up, ffn, hidden, hidden, TILE_M) || !map_rows(maps.b[0], x, tokens, hidden, x_ld, p.n))
            return no_maps();
        p.idesc = idesc_f16(dtype, false, false, TILE_M, p.n);
        p.out = h; p.g = g; p.u = u; p.ldo = ffn; p.out_type = dtype; p.saved_type = saved_dtype;
        return launch_few<false, false, 2>(maps, p, d, s);
    }
    TilePlan p{};
    p.M = tokens; p.N = ffn; p.segs = 1; p.outs = 1;
    p.out[0] = h; p.g = g; p.u = u; p.ldo = ffn; p.out_type = dtype; p.saved_type = saved_dtype;
    const bool narrow = narrow_tiles(p, d, 2);
    set_tile_k(p, hidden, 64, narrow);
    const uint32_t n = narrow ? 128 : 256;
    if (!set_tiles(p, n / 2)) return too_many();
    p.idesc = idesc_f16(dtype, false, false, 256, n);
    if (!map_rows(maps.a[0], x, tokens, hidden, x_ld, TILE_M) || !map_rows(maps.b[0], gate, ffn, hidden, hidden, n / 2) || !map_rows(maps.b[1], up, ffn, hidden, hidden, n / 2)) return no_maps();
    return narrow ? launch_tiles<false, false, false, true, 128>(maps, p, d, s) : launch_tiles<false, false, false, true, 256>(maps, p, d, s);
}

int zc_gated_backward(const void* dh, uint64_t dh_ld, const void* x, uint64_t x_ld, const void* gate, const void* up, const void* g, const void* u, int saved_dtype, int dtype, uint32_t tokens,
                      uint32_t hidden, uint32_t ffn, void* dg, void* du, void* dx, void* dgate, void* dup, void* stream) {
    const char* who = "zc_gated_backward";
    int rc = check_gated(who, dtype, hidden, ffn);
    if (rc == ZC_OK) rc = check_matrix(who, dh, dtype, tokens, ffn, dh_ld, true);
    if (rc == ZC_OK) rc = check_matrix(who, x, dtype, tokens, hidden, x_ld, true);
    for (const void* w : {gate, up}) if (rc == ZC_OK) rc = check_matrix(who, w, dtype, ffn, hidden, hidden, true);
    for (const void* v : {g, u, static_cast<const void*>(dg), static_cast<const void*>(du)}) if (rc == ZC_OK) rc = check_matrix(who, v, dtype, tokens, ffn, ffn, true);
    if (rc == ZC_OK) rc = check_saved(who, g, u, dtype, saved_dtype);
    if (rc == ZC_OK && dx) rc = check_matrix(who, dx, dtype, tokens, hidden, hidden, true);
    if (rc == ZC_OK && !dgate != !dup) rc = fail(nullptr, ZC_EINVAL, std::string(who) + ": dgate and dup go together");
    for (const void* v : {dgate, dup}) if (rc == ZC_OK && v) rc = check_matrix(who, v, dtype, ffn, hidden, hidden, true);
    if (rc != ZC_OK) return rc;
    if (tokens == 1) { x_ld = hidden; dh_ld = ffn; }
    const uint64_t tf = uint64_t(tokens) * ffn * 2, fh = uint64_t(ffn) * hidden * 2, th = uint64_t(tokens) * hidden * 2, ts = uint64_t(tokens) * ffn * dtype_bytes(saved_dtype);
    const Span in[6] = {{dh, matrix_bytes(dtype, tokens, ffn, dh_ld)}, {x, matrix_bytes(dtype, tokens, hidden, x_ld)}, {gate, fh}, {up, fh}, {g, ts}, {u, ts}};
    const Span to[5] = {{dg, tf}, {du, tf}, {dx, th}, {dgate, fh}, {dup, fh}};
    for (int i = 0; i < 5; ++i) {
        for (const Span& v : in) if (overlap(to[i], v)) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
        for (int j = 0; j < i; ++j) if (overlap(to[i], to[j])) return fail(nullptr, ZC_EINVAL, std::string(who) + ": overlapping buffers");
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!tokens) {
        for (void* v : {dgate, dup}) {
            const cudaError_t e = v ? cudaMemsetAsync(v, 0, fh, s) : cudaSuccess;
            if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("cudaMemsetAsync: ") + cudaGetErrorString(e)); }
        }
        return ZC_OK;
    }
    const dim3 grid((tokens + 7) / 8, (ffn + 255) / 256);
    const auto gradient = [&](auto type, auto saved) {
        typedef decltype(type) T;
        typedef decltype(saved) S;
        return launch_after(gated_gradient_kernel<T, S>, grid, 256, 0, 1, s, static_cast<const T*>(dh), dh_ld, static_cast<const S*>(g), static_cast<const S*>(u), tokens, ffn,
                            static_cast<T*>(dg), static_cast<T*>(du));
    };
    const bool full = saved_dtype == ZC_F32;
    rc = launched(dtype == ZC_BF16 ? (full ? gradient(__nv_bfloat16(), float()) : gradient(__nv_bfloat16(), __nv_bfloat16()))
                                   : (full ? gradient(__half(), float()) : gradient(__half(), __half())), "gated gradient");
    if (rc != ZC_OK) return rc;
    Device d;
    if ((rc = current_device(d)) != ZC_OK) return rc;
    if (dx) {
        TileMaps maps{};
        if (tokens <= FEW_TOKENS) {
            FewPlan p{};
            p.M = hidden; p.tokens = tokens; p.segs = 2;
            set_k(p, ffn, 64);
            plan_few(p, false, 1, false, d.sms);
            if (!map_rows(maps.a[0], gate, ffn, hidden, hidden, ACROSS) || !map_rows(maps.a[1], up, ffn, hidden, hidden, ACROSS) ||
                !map_rows(maps.b[0], dg, tokens, ffn, ffn, p.n) || !map_rows(maps.b[1], du, tokens, ffn, ffn, p.n)) return no_maps();
            p.idesc = idesc_f16(dtype, true, false, TILE_M, p.n);
            p.out = dx; p.ldo = hidden; p.out_type = dtype;
            rc = launch_few<false, true, 1>(maps, p, d, s);
        } else {
            TilePlan p{};
            p.M = tokens; p.N = hidden; p.segs = 2; p.outs = 1;
            p.out[0] = dx; p.ldo = hidden; p.out_type = dtype;
            const bool narrow = narrow_tiles(p, d, 1);
            set_tile_k(p, ffn, 64, narrow);
            if (!set_tiles(p, narrow ? 128 : 256)) return too_many();
            p.idesc = idesc_f16(dtype, false, true, 256, narrow ? 128 : 256);
            if (!map_rows(maps.a[0], dg, tokens, ffn, ffn, TILE_M) || !map_rows(maps.a[1], du, tokens, ffn, ffn, TILE_M) ||
                !map_rows(maps.b[0], gate, ffn, hidden, hidden, ACROSS) || !map_rows(maps.b[1], up, ffn, hidden, hidden, ACROSS)) return no_maps();
            rc = narrow ? launch_tiles<false, false, true, false, 128>(maps, p, d, s) : launch_tiles<false, false, true, false, 256>(maps, p, d, s);
        }
        if (rc != ZC_OK) return rc;
    }
    if (dgate) {
        TileMaps maps{};
        TilePlan p{};
        p.M = ffn; p.N = hidden; p.segs = 1; p.outs = 2;
        p.out[0] = dgate; p.out[1] = dup; p.ldo = hidden; p.out_type = dtype;
        const bool narrow = narrow_tiles(p, d, 1);
        set_tile_k(p, tokens, 64, narrow);
        if (!set_tiles(p, narrow ? 128 : 256)) return too_many();
        p.idesc = idesc_f16(dtype, true, true, 256, narrow ? 128 : 256);
        if (!map_rows(maps.a[0], dg, tokens, ffn, ffn, ACROSS) || !map_rows(maps.a[1], du, tokens, ffn, ffn, ACROSS) || !map_rows(maps.b[0], x, tokens, hidden, x_ld, ACROSS)) return no_maps();
        rc = narrow ? launch_tiles<false, true, true, false, 128>(maps, p, d, s) : launch_tiles<false, true, true, false, 256>(maps, p, d, s);
    }
    return rc;
}

int zc_ffn_wait_limit(uint32_t polls, uint32_t* before) {
    if (polls > 1u << 27) return fail(nullptr, ZC_EINVAL, "zc_ffn_wait_limit: more than 2^27 polls");
    const uint32_t old = wait_polls.exchange(polls);
    if (before) *before = old;
    return ZC_OK;
}

int zc_ffn_status(void* stream, uint32_t* status) {
    if (!status) return fail(nullptr, ZC_EINVAL, "missing buffer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint32_t zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(status, ffn_status_word, 4, 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    // Cleared only where it was found set: what another stream raises after the read is then either left in the word, or the same bit as the one that
    // this call returns. (Its only bit is ZC_STATUS_TIMEOUT.)
    if (e == cudaSuccess && *status) {
        e = cudaMemcpyToSymbolAsync(ffn_status_word, &zero, 4, 0, cudaMemcpyHostToDevice, s);
        if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    }
    if (e != cudaSuccess) { cudaGetLastError(); return fail(nullptr, ZC_EEXEC, std::string("status: ") + cudaGetErrorString(e)); }
    return ZC_OK;
}

}  // extern "C"
