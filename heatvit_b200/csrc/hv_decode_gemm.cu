// hv_decode_gemm.cu — e4m3 matrix product with a scale for each block of 128.
//
//   C[m][n] = sum_g as[m][g] * bs[n / 128][g] * sum_{k in group g} A[m][k] B[n][k],
//   g the groups of 128 along K; sums in 32 bits, one rounding to C's type.
//
// A CTA computes 128 rows x BN columns of the product of two K-major operands, X (rows) and
// Y (columns).  Roles: one thread issues the TMA copies (128-byte swizzled boxes of one
// group) into a ring of stages; one thread issues tcgen05.mma kind::f8f6f4, four of K = 32
// for a group, into one of several TMEM accumulators; eight warps read each finished
// accumulator and add it, times its scale, to sums in their registers, since the tensor core
// itself cannot scale by 32-bit numbers.  Reading and adding a 128 x BN block takes half the
// time of its MMAs, and runs beside those of the next group.
//
// Two ways round.  Many tokens: X = A, Y = B.  Few tokens (SWAP): X = B, Y = A, so that the
// 128 rows that an MMA has anyway are weights; the time is that of reading the weights once.
// Where the tiles are fewer than the SMs, K is split over the CTAs of a cluster, which join
// their sums through distributed shared memory, in the order of their ranks.
//
// Every mbarrier wait is bounded: after a timeout the CTA waits for what it has in flight,
// releases its TMEM and sets the device's error word.
#include <cudaTypedefs.h>

#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr int BM = 128, GK = 128;  // rows of a tile; a group of K, in elements and bytes
constexpr int EPI_WARPS = 8, EPI_THREADS = EPI_WARPS * 32;
constexpr int THREADS = EPI_THREADS + 64;
constexpr uint32_t WAIT_ITERS = 1u << 22;

struct GemmFp8Args {
    const float *xs, *ys;  // scales of the row and column operands
    long long xs_row, xs_group, ys_row, ys_group;
    void *out;
    long long ldc;
    int x_rows, y_rows, groups, tiles_x, split, out_dtype, vec;
    int *err;
};

template <int BN>
struct Lay {
    static constexpr int A_ST = BM * GK, B_ST = BN * GK, STAGE = A_ST + B_ST;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int BUFS = BN == 256 ? 2 : 4;  // TMEM accumulators
    static constexpr int COLS = BN < 32 ? 32 : BN;  // TMEM columns of one
    static constexpr int TMEM = BUFS * COLS;
    static constexpr int BARS = STAGES * STAGE;  // full[STAGES] empty[STAGES] tfull[BUFS] tempty[BUFS] drain
    static constexpr int BYTES = BARS + 256 + 1024;  // and room to align the ring to 1024
};

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint64_t *mbar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::
            "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(tc05::smem_u32(mbar))
        : "memory");
}
__device__ __forceinline__ void expect_tx(uint64_t *mbar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(tc05::smem_u32(mbar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void arrive(uint64_t *mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc05::smem_u32(mbar)) : "memory");
}
// K-major operand, 128-byte swizzle: eight rows of 128 bytes per 1024-byte atom.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// kind::f8f6f4, e4m3 x e4m3 -> f32, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// Bounded wait that also ends when another role of the CTA has given up.
__device__ __forceinline__ bool wait_or_stop(uint64_t *bar, uint32_t parity, volatile int *stop) {
    for (uint32_t i = 0; i < WAIT_ITERS / 64; ++i) {
        if (tc05::mbar_wait(bar, parity, 64)) return true;
        if (*stop) return false;
    }
    *stop = 1;
    return false;
}

template <typename T>
__device__ __forceinline__ void put(void *out, long long i, float v) {
    ((T *)out)[i] = from_f32<T>(v);
}
__device__ __forceinline__ void put_any(void *out, int dtype, long long i, float v) {
    if (dtype == HV_BF16) put<__nv_bfloat16>(out, i, v);
    else if (dtype == HV_F16) put<__half>(out, i, v);
    else put<float>(out, i, v);
}
__device__ __forceinline__ void put8_any(void *out, int dtype, long long i, bool vec, int n, const float (&v)[8]) {
    if (dtype == HV_BF16) store8((__nv_bfloat16 *)out + i, n, vec, v);
    else if (dtype == HV_F16) store8((__half *)out + i, n, vec, v);
    else store8((float *)out + i, n, vec, v);
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ float ld_peer(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// gridDim.x = tiles * split, the CTAs of a cluster next to one another.
template <int BN, bool SWAP>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmy, const GemmFp8Args a) {
    using L = Lay<BN>;
    extern __shared__ uint8_t raw[];
    __shared__ uint32_t tslot;
    __shared__ volatile int stop;
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    uint64_t *full = (uint64_t *)(smem + L::BARS), *empty = full + L::STAGES;
    uint64_t *tfull = empty + L::STAGES, *tempty = tfull + L::BUFS, *drain = tempty + L::BUFS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = a.split, rank = blockIdx.x % split, tile = blockIdx.x / split;
    const int tx = tile % a.tiles_x, ty = tile / a.tiles_x;
    const int x0 = tx * BM, y0 = ty * BN;
    const int g0 = (int)((long long)a.groups * rank / split), g1 = (int)((long long)a.groups * (rank + 1) / split);
    const int n_groups = g1 - g0;

    if (warp == EPI_WARPS) {
        tc05::tmem_alloc(&tslot, L::TMEM);
        tc05::tmem_relinquish();
    }
    if (tid == 0) {
        stop = 0;
        for (int i = 0; i < L::STAGES; ++i) {
            tc05::mbar_init(&full[i], 1);
            tc05::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < L::BUFS; ++i) {
            tc05::mbar_init(&tfull[i], 1);
            tc05::mbar_init(&tempty[i], EPI_WARPS);
        }
        tc05::mbar_init(drain, 1);
        tc05::fence_mbar_init();
    }
    tc05::fence_before();
    __syncthreads();
    tc05::fence_after();
    griddep_wait();
    griddep_launch();
    const uint32_t tmem = tslot;

    if (warp == EPI_WARPS && lane == 0) {  // copies
        int i = 0;
        for (; i < n_groups; ++i) {
            const int s = i % L::STAGES;
            if (i >= L::STAGES && !wait_or_stop(&empty[s], (i / L::STAGES - 1) & 1, &stop)) break;
            const uint32_t dst = tc05::smem_u32(smem + s * L::STAGE);
            expect_tx(&full[s], L::STAGE);
            tma_box(dst, &tmx, (g0 + i) * GK, x0, &full[s]);
            tma_box(dst + L::A_ST, &tmy, (g0 + i) * GK, y0, &full[s]);
        }
        if (i < n_groups)  // gave up: what was issued has to land before shared memory goes
            for (int k = max(0, i - L::STAGES); k < i; ++k) tc05::mbar_wait(&full[k % L::STAGES], (k / L::STAGES) & 1, WAIT_ITERS);
    } else if (warp == EPI_WARPS + 1 && lane == 0) {  // products
        constexpr uint32_t idesc = idesc_e4m3(BM, BN);
        int i = 0;
        for (; i < n_groups; ++i) {
            const int s = i % L::STAGES, b = i % L::BUFS;
            if (i >= L::BUFS && !wait_or_stop(&tempty[b], (i / L::BUFS - 1) & 1, &stop)) break;
            if (!wait_or_stop(&full[s], (i / L::STAGES) & 1, &stop)) break;
            tc05::fence_after();
            const uint32_t at = tc05::smem_u32(smem + s * L::STAGE);
            const uint64_t da = desc_sw128(at), db = desc_sw128(at + L::A_ST);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_e4m3(tmem + b * L::COLS, da + 2 * k, db + 2 * k, idesc, k > 0);
            tc05::commit(&empty[s]);
            tc05::commit(&tfull[b]);
        }
        if (i < n_groups) {
            tc05::commit(drain);
            tc05::mbar_wait(drain, 0, WAIT_ITERS);
        }
    }

    // Sums: thread = (tile row, half of the columns).
    constexpr int HC = BN / 2;
    constexpr int CH = HC < 32 ? HC : 32;  // columns of one TMEM load
    const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * HC;
    float acc[HC];
    if (warp < EPI_WARPS) {
#pragma unroll
        for (int j = 0; j < HC; ++j) acc[j] = 0.f;
        // Scales of a group: a row's own times its columns' (SWAP: the rows' shared one times
        // each column's, which lane j holds for column j).
        const int xr = SWAP ? x0 / GK : min(x0 + row, a.x_rows - 1);
        const int yr = SWAP ? min(y0 + c0 + lane % HC, a.y_rows - 1) : min(y0 + c0, a.y_rows - 1) / GK;
        const float *xs = a.xs + xr * a.xs_row + g0 * a.xs_group;
        const float *ys = a.ys + yr * a.ys_row + g0 * a.ys_group;
        const uint32_t tbase = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
        constexpr int AHEAD = 4;  // groups whose scales are on the way
        float sx[AHEAD], sy[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            sx[i] = i < n_groups ? xs[i * a.xs_group] : 0.f;
            sy[i] = i < n_groups ? ys[i * a.ys_group] : 0.f;
        }
        bool ok = true;
        for (int i0 = 0; i0 < n_groups && ok; i0 += AHEAD)
#pragma unroll
            for (int ii = 0; ii < AHEAD; ++ii) {
                const int i = i0 + ii;
                if (i >= n_groups || !ok) break;
                const float s = sx[ii] * sy[ii];
                if (i + AHEAD < n_groups) {
                    sx[ii] = xs[(i + AHEAD) * a.xs_group];
                    sy[ii] = ys[(i + AHEAD) * a.ys_group];
                }
                const int b = i % L::BUFS;
                ok = wait_or_stop(&tfull[b], (i / L::BUFS) & 1, &stop);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                tc05::fence_after();
#pragma unroll
                for (int j0 = 0; j0 < HC; j0 += CH) {
                    uint32_t d[CH];
                    if constexpr (CH == 32) tc05::ld32(tbase + b * L::COLS + j0, d);
                    else if constexpr (CH == 16) tc05::ld16(tbase + b * L::COLS + j0, d);
                    else tc05::ld8(tbase + b * L::COLS + j0, d);
                    tc05::wait_ld_regs(d);
                    if (j0 + CH == HC) {
                        tc05::fence_before();
                        if (lane == 0) arrive(&tempty[b]);
                    }
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        const float f = SWAP ? __shfl_sync(~0u, s, j0 + j) : s;
                        acc[j0 + j] = fmaf(__uint_as_float(d[j]), f, acc[j0 + j]);
                    }
                }
            }
    }

    __syncwarp();  // the one-thread roles rejoin their warps
    const int cols_of = a.y_rows;
    if (split == 1) {
        if (warp < EPI_WARPS && x0 + row < a.x_rows) {
            if (SWAP) {
#pragma unroll
                for (int j = 0; j < HC; ++j) {
                    const int c = y0 + c0 + j;
                    if (c < cols_of) put_any(a.out, a.out_dtype, c * a.ldc + x0 + row, acc[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < HC; j += 8) {
                    const int c = y0 + c0 + j;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[j + e];
                    if (c < cols_of)
                        put8_any(a.out, a.out_dtype, (long long)(x0 + row) * a.ldc + c, a.vec, cols_of - c, v);
                }
            }
        }
        __syncthreads();
    } else {
        // Every copy and product of this CTA has completed (or its waits gave up and were
        // drained): the ring's memory takes the sums, column by column.
        __syncthreads();
        float *part = (float *)smem;
        if (warp < EPI_WARPS)
#pragma unroll
            for (int j = 0; j < HC; ++j) part[(c0 + j) * BM + row] = acc[j];
        cluster_sync();
        if (warp < EPI_WARPS) {
            const int per = BN / split, cb = rank * per;
            for (int j = tid >> 7; j < per; j += 2) {
                const int r = tid & 127, c = y0 + cb + j;
                const uint32_t at = tc05::smem_u32(part + (cb + j) * BM + r);
                float v = 0.f;
                for (int k = 0; k < split; ++k) v += ld_peer(at, k);
                if (x0 + r < a.x_rows && c < cols_of)
                    put_any(a.out, a.out_dtype,
                            SWAP ? (long long)c * a.ldc + x0 + r : (long long)(x0 + r) * a.ldc + c, v);
            }
        }
        cluster_sync();  // no CTA leaves while its sums may be read
    }
    if (tid == 0 && stop) atomicOr(a.err, HV_DECODE_STALLED);
    tc05::fence_before();
    __syncthreads();
    if (warp == EPI_WARPS) {
        tc05::fence_after();
        tc05::tmem_dealloc(tmem, L::TMEM);
    }
}

// ---- many tiles: persistent CTAs -------------------------------------------------
// 128 x 256 tiles, one CTA an SM that takes a tile after another.  The rings of operand stages
// and TMEM accumulators run on from tile to tile, so that the tensor core works through the
// output of the tile before.  An adding thread has 128 columns of a row: its sums take 128
// registers, so the copying and issuing warps give theirs up.  It keeps a 16-column TMEM load
// under way while it adds the one before, with packed pairs of multiply-adds.
constexpr int WIDE_BN = 256, WIDE_STAGES = 4, WIDE_BUFS = 2, WIDE_THREADS = 384, BAND = 16;
constexpr int WIDE_STAGE = (BM + WIDE_BN) * GK;
// Scales of SB groups at a time, a row's times its columns', for either half of the columns: two
// warps fetch and multiply them (loads in the adding warps made those wait: 711 us, 8192^3).
constexpr int SB = 8, SC_BYTES = 2 * SB * 2 * BM * 4;
constexpr int WIDE_BYTES = WIDE_STAGES * WIDE_STAGE + SC_BYTES + 256 + 1024;

__device__ __forceinline__ void fma2(uint64_t &acc, uint32_t lo, uint32_t hi, uint64_t f) {
    asm("{\n.reg .b64 t;\nmov.b64 t, {%1, %2};\nfma.rn.f32x2 %0, t, %3, %0;\n}\n" : "+l"(acc) : "r"(lo), "r"(hi), "l"(f));
}

// Tile `i` in bands of BAND tile rows, columns of a band one after another: the CTAs at work at
// one time share few rows and columns of the operands, which L2 then has.
__device__ __forceinline__ void tile_at(int i, int tiles_x, int tiles_y, int &tx, int &ty) {
    const int band = i / (BAND * tiles_y), in = i - band * BAND * tiles_y;
    const int h = min(BAND, tiles_x - band * BAND);
    ty = in / h;
    tx = band * BAND + in - ty * h;
}

__global__ void __launch_bounds__(WIDE_THREADS, 1)
    gemm_wide_kernel(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmy,
                     const __grid_constant__ GemmFp8Args a) {
    extern __shared__ uint8_t raw[];
    __shared__ uint32_t tslot;
    __shared__ volatile int stop;
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    float(*sc)[SB][2][BM] = (float(*)[SB][2][BM])(smem + WIDE_STAGES * WIDE_STAGE);
    uint64_t *full = (uint64_t *)(smem + WIDE_STAGES * WIDE_STAGE + SC_BYTES), *empty = full + WIDE_STAGES;
    uint64_t *tfull = empty + WIDE_STAGES, *tempty = tfull + WIDE_BUFS, *drain = tempty + WIDE_BUFS;
    uint64_t *sfull = drain + 1, *sempty = sfull + 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tiles_y = (a.y_rows + WIDE_BN - 1) / WIDE_BN, tiles = a.tiles_x * tiles_y;

    if (warp == 2) {
        tc05::tmem_alloc(&tslot, 512);
        tc05::tmem_relinquish();
    }
    if (tid == 0) {
        stop = 0;
        for (int i = 0; i < WIDE_STAGES; ++i) {
            tc05::mbar_init(&full[i], 1);
            tc05::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < WIDE_BUFS; ++i) {
            tc05::mbar_init(&tfull[i], 1);
            tc05::mbar_init(&tempty[i], EPI_WARPS);
        }
        tc05::mbar_init(drain, 1);
        for (int i = 0; i < 2; ++i) {
            tc05::mbar_init(&sfull[i], 64);
            tc05::mbar_init(&sempty[i], EPI_WARPS);
        }
        tc05::fence_mbar_init();
    }
    tc05::fence_before();
    __syncthreads();
    tc05::fence_after();
    griddep_wait();
    griddep_launch();
    const uint32_t tmem = tslot;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == 0 && lane == 0) {  // copies
            uint32_t n = 0;  // stages filled
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                int tx, ty;
                tile_at(t, a.tiles_x, tiles_y, tx, ty);
                for (int g = 0; g < a.groups; ++g, ++n) {
                    const uint32_t s = n % WIDE_STAGES;
                    if (n >= WIDE_STAGES && !wait_or_stop(&empty[s], (n / WIDE_STAGES - 1) & 1, &stop)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = tc05::smem_u32(smem + s * WIDE_STAGE);
                    expect_tx(&full[s], WIDE_STAGE);
                    tma_box(dst, &tmx, g * GK, tx * BM, &full[s]);
                    tma_box(dst + BM * GK, &tmy, g * GK, ty * WIDE_BN, &full[s]);
                }
            }
            if (!ok)  // what was issued has to land before shared memory goes
                for (uint32_t k = n > WIDE_STAGES ? n - WIDE_STAGES : 0; k < n; ++k)
                    tc05::mbar_wait(&full[k % WIDE_STAGES], (k / WIDE_STAGES) & 1, WAIT_ITERS);
        } else if (warp == 1 && lane == 0) {  // products
            constexpr uint32_t idesc = idesc_e4m3(BM, WIDE_BN);
            uint32_t n = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x)
                for (int g = 0; g < a.groups; ++g, ++n) {
                    const uint32_t s = n % WIDE_STAGES, b = n % WIDE_BUFS;
                    ok = (n < WIDE_BUFS || wait_or_stop(&tempty[b], (n / WIDE_BUFS - 1) & 1, &stop)) &&
                         wait_or_stop(&full[s], (n / WIDE_STAGES) & 1, &stop);
                    if (!ok) break;
                    tc05::fence_after();
                    const uint32_t at = tc05::smem_u32(smem + s * WIDE_STAGE);
                    const uint64_t da = desc_sw128(at), db = desc_sw128(at + BM * GK);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_e4m3(tmem + b * WIDE_BN, da + 2 * k, db + 2 * k, idesc, k > 0);
                    tc05::commit(&empty[s]);
                    tc05::commit(&tfull[b]);
                }
            if (!ok) {
                tc05::commit(drain);
                tc05::mbar_wait(drain, 0, WAIT_ITERS);
            }
        } else if (warp >= 2) {  // scales
            const int r = tid - 64;  // and r + 64
            int t = blockIdx.x, g = 0;
            const float *x0 = nullptr, *x1 = nullptr, *y0 = nullptr, *y1 = nullptr;
            for (uint32_t q = 0; t < tiles; ++q) {
                const int b = q & 1;
                if (q >= 2 && !wait_or_stop(&sempty[b], (q / 2 - 1) & 1, &stop)) break;
#pragma unroll
                for (int e0 = 0; e0 < SB; e0 += 4) {
                    float vx0[4], vx1[4], vy0[4], vy1[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (t >= tiles) break;
                        if (g == 0) {
                            int tx, ty;
                            tile_at(t, a.tiles_x, tiles_y, tx, ty);
                            x0 = a.xs + min(tx * BM + r, a.x_rows - 1) * a.xs_row;
                            x1 = a.xs + min(tx * BM + r + 64, a.x_rows - 1) * a.xs_row;
                            y0 = a.ys + min(ty * WIDE_BN, a.y_rows - 1) / GK * a.ys_row;
                            y1 = a.ys + min(ty * WIDE_BN + GK, a.y_rows - 1) / GK * a.ys_row;
                        }
                        vx0[e] = x0[g * a.xs_group];
                        vx1[e] = x1[g * a.xs_group];
                        vy0[e] = y0[g * a.ys_group];
                        vy1[e] = y1[g * a.ys_group];
                        if (++g == a.groups) {
                            g = 0;
                            t += gridDim.x;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[b][e0 + e][0][r] = vx0[e] * vy0[e];
                        sc[b][e0 + e][1][r] = vx0[e] * vy1[e];
                        sc[b][e0 + e][0][r + 64] = vx1[e] * vy0[e];
                        sc[b][e0 + e][1][r + 64] = vx1[e] * vy1[e];
                    }
                }
                arrive(&sfull[b]);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
        const int row = (warp & 3) * 32 + lane, c0 = ((warp - 4) >> 2) * 128;
        const uint32_t tbase = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
        const int half = (warp - 4) >> 2;
        uint64_t acc[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) acc[j] = 0;
        uint32_t n = 0;
        bool ok = true;
        for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            for (int g = 0; g < a.groups; ++g, ++n) {
                const uint32_t b = n % WIDE_BUFS, sb = n / SB;
                ok = n % SB || wait_or_stop(&sfull[sb & 1], (sb / 2) & 1, &stop);
                const float f = sc[sb & 1][n % SB][half][row];
                uint64_t s2;
                asm("mov.b64 %0, {%1, %1};\n" : "=l"(s2) : "f"(f));
                ok = ok && wait_or_stop(&tfull[b], (n / WIDE_BUFS) & 1, &stop);
                ok = __all_sync(~0u, ok);  // and every lane has its scale
                if (!ok) break;
                __syncwarp();
                if (n % SB == SB - 1 && lane == 0) arrive(&sempty[sb & 1]);
                tc05::fence_after();
                uint32_t d[2][16];
                tc05::ld16(tbase + b * WIDE_BN, d[0]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    tc05::wait_ld_regs(d[c & 1]);
                    if (c < 7) {
                        tc05::ld16(tbase + b * WIDE_BN + (c + 1) * 16, d[(c + 1) & 1]);
                    } else {
                        tc05::fence_before();
                        if (lane == 0) arrive(&tempty[b]);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) fma2(acc[c * 8 + j], d[c & 1][2 * j], d[c & 1][2 * j + 1], s2);
                }
            }
            if (!ok) break;
            int tx, ty;
            tile_at(t, a.tiles_x, tiles_y, tx, ty);
            const int m = tx * BM + row, col = ty * WIDE_BN + c0;
            const long long at = (long long)m * a.ldc + col;
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(v[2 * e]), "=f"(v[2 * e + 1]) : "l"(acc[j + e]));
                    acc[j + e] = 0;
                }
                if (m < a.x_rows && col + 2 * j < a.y_rows)
                    put8_any(a.out, a.out_dtype, at + 2 * j, a.vec, a.y_rows - col - 2 * j, v);
            }
        }
    }
    if (tid == 0 && stop) atomicOr(a.err, HV_DECODE_STALLED);
    tc05::fence_before();
    __syncthreads();
    if (warp == 2) {
        tc05::fence_after();
        tc05::tmem_dealloc(tmem, 512);
    }
}

PFN_cuTensorMapEncodeTiled encoder() {
    static PFN_cuTensorMapEncodeTiled encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return (PFN_cuTensorMapEncodeTiled)fn;
    }();
    return encode;
}

// [rows][k] bytes, `stride` apart, in boxes of 128 bytes x box_rows; what is past an edge reads as zero.
bool tensor_map(CUtensorMap *map, const void *base, int64_t rows, int k, int64_t stride, int box_rows) {
    const PFN_cuTensorMapEncodeTiled encode = encoder();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {GK, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Operand {
    const void *p;
    int64_t rows, stride;
    const float *scale;
    int64_t s_row, s_group;
};

template <int BN, bool SWAP>
int run(const Operand &x, const Operand &y, int k, GemmFp8Args a, int sms, cudaStream_t st) {
    using L = Lay<BN>;
    CUtensorMap tmx, tmy;
    if (!tensor_map(&tmx, x.p, x.rows, k, x.stride, BM) || !tensor_map(&tmy, y.p, y.rows, k, y.stride, BN))
        return fail(HV_ERR_CUDA, "gemm_fp8: cannot encode the operands' tensor maps");
    a.xs = x.scale, a.xs_row = x.s_row, a.xs_group = x.s_group;
    a.ys = y.scale, a.ys_row = y.s_row, a.ys_group = y.s_group;
    a.x_rows = (int)x.rows, a.y_rows = (int)y.rows;
    a.tiles_x = (int)((x.rows + BM - 1) / BM);
    const int64_t tiles = (int64_t)a.tiles_x * ((y.rows + BN - 1) / BN);
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sms && a.groups >= split * 2) split *= 2;
    if (tiles * split > INT32_MAX) return fail(HV_ERR_VALUE, "gemm_fp8: too many tiles");
    a.split = split;
    auto kernel = gemm_kernel<BN, SWAP>;
    static std::atomic<uint64_t> ready;
    cudaError_t e = allow_shared(kernel, ready);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(tiles * split));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = L::BYTES;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)split;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, kernel, tmx, tmy, a);
    }
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "gemm_fp8: %s", cudaGetErrorString(e));
    return HV_OK;
}

int run_wide(const Operand &x, const Operand &y, int k, GemmFp8Args a, int sms, cudaStream_t st) {
    CUtensorMap tmx, tmy;
    if (!tensor_map(&tmx, x.p, x.rows, k, x.stride, BM) || !tensor_map(&tmy, y.p, y.rows, k, y.stride, WIDE_BN))
        return fail(HV_ERR_CUDA, "gemm_fp8: cannot encode the operands' tensor maps");
    a.xs = x.scale, a.xs_row = x.s_row, a.xs_group = x.s_group;
    a.ys = y.scale, a.ys_row = y.s_row, a.ys_group = y.s_group;
    a.x_rows = (int)x.rows, a.y_rows = (int)y.rows;
    a.tiles_x = (int)((x.rows + BM - 1) / BM);
    const int64_t tiles = (int64_t)a.tiles_x * ((y.rows + WIDE_BN - 1) / WIDE_BN);
    if (tiles > INT32_MAX / 2) return fail(HV_ERR_VALUE, "gemm_fp8: too many tiles");
    static std::atomic<uint64_t> ready;
    cudaError_t e = allow_shared(gemm_wide_kernel, ready);
    if (e == cudaSuccess)
        e = launch_pdl(gemm_wide_kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(WIDE_THREADS), WIDE_BYTES, st,
                       tmx, tmy, a);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "gemm_fp8: %s", cudaGetErrorString(e));
    return HV_OK;
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_gemm_fp8(const hv_gemm_fp8_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (!dec::known_dtype(p->out_dtype)) return fail(HV_ERR_TYPE, "out_dtype must be HV_BF16, HV_F16 or HV_F32");
    const int64_t m = p->m, n = p->n, k = p->k, most = INT32_MAX - 512;
    if (m < 0 || n < 0 || m > most || n > most) return fail(HV_ERR_VALUE, "m or n outside [0, 2^31 - 512]");
    if (k < 1 || k > most) return fail(HV_ERR_VALUE, "k outside [1, 2^31 - 512]");
    if (m == 0 || n == 0) return HV_OK;
    if (!p->d_a || !p->d_a_scale || !p->d_b || !p->d_b_scale || !p->d_out) return fail(HV_ERR_VALUE, "null buffer");
    if (!dec::aligned(p->d_a, 16) || !dec::aligned(p->d_b, 16) || (m > 1 && p->a_stride % 16) ||
        (n > 1 && p->b_stride % 16))
        return fail(HV_ERR_VALUE, "operand rows must start on 16 bytes");
    const int64_t room = (k + 15) / 16 * 16;  // a one-row operand's stride is not used
    const int64_t sa = m > 1 ? p->a_stride : room, sb = n > 1 ? p->b_stride : room;
    if (sa < k || sb < k) return fail(HV_ERR_VALUE, "operand rows overlap");
    int *err = dec::error_word();
    const int sms = dec::sm_count();
    if (!err || !sms) return fail(HV_ERR_CUDA, "cannot read the device's properties");
    GemmFp8Args g{};
    g.out = p->d_out, g.ldc = p->out_stride, g.out_dtype = p->out_dtype, g.groups = (int)((k + GK - 1) / GK), g.err = err;
    g.vec = dec::aligned(p->d_out, 16) && (m == 1 || p->out_stride * dec::elem_size(p->out_dtype) % 16 == 0);
    const Operand a{p->d_a, m, sa, p->d_a_scale, p->a_scale_strides[0], p->a_scale_strides[1]};
    const Operand b{p->d_b, n, sb, p->d_b_scale, p->b_scale_strides[0], p->b_scale_strides[1]};
    const cudaStream_t st = (cudaStream_t)stream;
    const int kk = (int)k;
    if (m <= 16) return run<16, true>(b, a, kk, g, sms, st);
    if (m <= 32) return run<32, true>(b, a, kk, g, sms, st);
    if (m <= 64) return run<64, true>(b, a, kk, g, sms, st);
    // a 256-wide tile reads each operand byte for more products; a 128-wide one fills more SMs
    if (((m + 127) / 128) * ((n + 255) / 256) >= sms) return run_wide(a, b, kk, g, sms, st);
    return run<128, false>(a, b, kk, g, sms, st);
}
