// hv_decode_gemm.cu — e4m3 matrix product with a scale for each block of 128.
//
//   C[m][n] = sum_g as[m][g] * bs[n / 128][g] * sum_{k in group g} A[m][k] B[n][k],
//   g the groups of 128 along K; sums in 32 bits, one rounding to C's type.
//
// A CTA computes tiles of 128 rows x BN columns of the product of two K-major operands, X
// (rows) and Y (columns).  Its warps: one thread issues the TMA copies (128-byte swizzled boxes of
// one group) into a ring of stages; one issues tcgen05.mma kind::f8f6f4, four of K = 32 for a
// group, into one of several TMEM accumulators; two warps fetch scales; eight read each
// finished accumulator and add it, times its scales, to sums in their registers, since the
// tensor core itself cannot scale by 32-bit numbers.  They keep a TMEM load under way while
// they add the one before, with packed pairs of multiply-adds.
//
// Three shapes of work.  Many tiles: 128 x 256, one CTA an SM that takes a tile after another,
// its rings running on from tile to tile so that the tensor core works through the output of the
// tile before.  Fewer: 128 x 128, K split over the CTAs of a cluster, which join their sums
// through distributed shared memory in the order of their ranks.  Few tokens (SWAP): X = B,
// Y = A, so that the 128 rows that an MMA has anyway are weights; split as well, two CTAs an SM;
// the time is that of reading the weights once.
//
// Measured on one B200: 8192^3 550 to 590 us in bursts (up to 2.0 PFLOP/s; 630 to 665 us, at
// 1.5 GHz, when it runs on at the power limit), 4096^3 83 us.  Without the adds the wide form
// takes 455 us, with one MMA in four 325: its operands come at 70 bytes an SM clock.  Tiles of
// 256 x 256 over CTA pairs (cta_group::2) move a third less and took as long (536 us, 648 at the
// power limit), an accumulator's way to the other CTA and back being longer.  48 x 10240 x 4096
// 15.1 us (2.9 TB/s of weights: five to the first sums, six to stream, four to join; 16 bytes of its 80
// registers spill), 1 x 4096 x 4096 6.7 us, 1576 x 768 x 192 4.6 us.
//
// Every mbarrier wait is bounded: after a timeout the CTA waits for what it has in flight,
// releases its TMEM and, when all of its roles are through, sets the device's error word.
#include <cudaTypedefs.h>

#include <algorithm>

#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr int BM = 128, GK = 128;  // rows of a tile; a group of K, in elements and bytes
constexpr int EPI_WARPS = 8, THREADS = 128 + EPI_WARPS * 32;
constexpr int SB = 8;      // groups whose scales are fetched together
constexpr int BAND = 16;   // tile rows of a band
constexpr int AHEAD = 16;  // groups that are prefetched into L2

struct GemmFp8Args {
    const float *xs, *ys;  // scales of the row and column operands
    long long xs_row, xs_group, ys_row, ys_group;
    void *out;
    long long ldc;
    int x_rows, y_rows, groups, tiles_x, tiles_y, split, out_dtype, vec;
    uint32_t skip;  // see skipped_copy
    int *err;
};

template <int BN, bool SWAP>
struct Lay {
    static constexpr int A_ST = BM * GK, B_ST = BN * GK, STAGE = A_ST + B_ST;
    static constexpr int PER_SM = SWAP ? 2 : 1;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : BN == 64 ? 3 : BN == 32 ? 4 : 5;
    static constexpr int BUFS = BN == 256 ? 2 : 4;  // TMEM accumulators
    static constexpr int COLS = BN < 32 ? 32 : BN;  // TMEM columns of one
    static constexpr int TMEM = BUFS * COLS;
    // scales: of each column (SWAP: all rows share one), or of each row with either half of the columns
    static constexpr int SCALES = SWAP ? BN : 2 * BM;
    static constexpr int SC = STAGES * STAGE;  // [2][SB][SCALES] float
    static constexpr int OUT = SC + 2 * SB * SCALES * 4;  // 2 KB an adding warp (see store_rows)
    // SWAP: the cluster's sums of this CTA's share of the output's rows (a third of BN rounds up to two more in all)
    static constexpr int BARS = OUT + (SWAP ? (BN + 2) * BM * 4 : EPI_WARPS * 2048);
    static constexpr int BYTES = BARS + 256 + 1024;  // and room to align the ring to 1024
    static_assert(PER_SM * TMEM <= 512 && PER_SM * (BYTES + 1024) <= 228 * 1024, "resident CTAs");
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
// Bounded wait that also ends when another role of the CTA has given up.  (With the limit in a kernel
// argument 256 x 8192 x 8192 took 35.9 us, and 33.4 with a constant.)
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
template <typename T>
__device__ __forceinline__ void put4(T *p, bool vec, int n, float4 v) {
    alignas(16) T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 2) *(uint2 *)p = *(const uint2 *)e;
        else *(uint4 *)p = *(const uint4 *)e;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = e[i];
    }
}
__device__ __forceinline__ void put4_any(const GemmFp8Args &a, long long i, int n, float4 v) {
    if (a.out_dtype == HV_BF16) put4((__nv_bfloat16 *)a.out + i, a.vec, n, v);
    else if (a.out_dtype == HV_F16) put4((__half *)a.out + i, a.vec, n, v);
    else put4((float *)a.out + i, a.vec, n, v);
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ void st_peer(uint32_t saddr, uint32_t rank, float v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ float4 ld_peer(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ void split2(uint64_t pair, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(pair));
}

// A warp's 32 rows x 2 * N columns of sums to `out` (row 0 of the 32, column 0), of which `rows`
// and `cols` exist, through 2 KB of shared memory in pieces of 64 bytes a row: a store then
// writes 64 neighbouring bytes of eight rows (vec: rows lie on 16 bytes and end with a whole 16)
// or of one or two, and not 32 rows' 16 or 2.
template <typename T, int N>
__device__ __forceinline__ void store_rows(T *out, long long ldc, int rows, int cols, bool vec, uint4 *stage,
                                           const uint64_t (&acc)[N]) {
    constexpr int PER = 16 / sizeof(T);  // elements of 16 bytes
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int p = 0; p < 2 * N / (4 * PER); ++p) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            alignas(16) T e[PER];
#pragma unroll
            for (int i = 0; i < PER; i += 2) {
                float lo, hi;
                split2(acc[(p * 4 + u) * (PER / 2) + i / 2], lo, hi);
                e[i] = from_f32<T>(lo);
                e[i + 1] = from_f32<T>(hi);
            }
            stage[lane * 4 + (u ^ (lane >> 1 & 3))] = *(const uint4 *)e;
        }
        __syncwarp();
        if (vec) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2), u = lane & 3, c = (p * 4 + u) * PER;
                if (r < rows && c < cols) *(uint4 *)(out + r * ldc + c) = stage[r * 4 + (u ^ (r >> 1 & 3))];
            }
        } else {
            constexpr int ROW = 4 * PER, AT_ONCE = 32 / ROW;  // elements of a piece, rows of a store
            const int r0 = lane / ROW, e = lane % ROW, u = e / PER, c = p * ROW + e;
#pragma unroll 8
            for (int r = r0; r < 32; r += AT_ONCE)
                if (r < rows && c < cols)
                    out[r * ldc + c] = ((const T *)(stage + r * 4 + (u ^ (r >> 1 & 3))))[e % PER];
        }
        __syncwarp();
    }
}

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

// One tile after another (split = 1), or one tile a cluster of `split` CTAs next to one another.
template <int BN, bool SWAP>
__global__ void __launch_bounds__(THREADS, Lay<BN, SWAP>::PER_SM)
    gemm_kernel(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmy,
                const __grid_constant__ GemmFp8Args a) {
    using L = Lay<BN, SWAP>;
    extern __shared__ uint8_t raw[];
    __shared__ uint32_t tslot;
    __shared__ volatile int stop;
    uint8_t *smem = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    float(*sc)[SB][L::SCALES] = (float(*)[SB][L::SCALES])(smem + L::SC);
    uint64_t *full = (uint64_t *)(smem + L::BARS), *empty = full + L::STAGES;
    uint64_t *tfull = empty + L::STAGES, *tempty = tfull + L::BUFS, *sfull = tempty + L::BUFS, *sempty = sfull + 2;
    uint64_t *drain = sempty + 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tiles = a.tiles_x * a.tiles_y, split = a.split, rank = blockIdx.x % split;
    const int first = blockIdx.x / split, step = gridDim.x / split;  // tiles of this CTA
    const int g0 = (int)((long long)a.groups * rank / split), g1 = (int)((long long)a.groups * (rank + 1) / split);

    if (warp == 2) {
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
        for (int i = 0; i < 2; ++i) {
            tc05::mbar_init(&sfull[i], 64);
            tc05::mbar_init(&sempty[i], EPI_WARPS);
        }
        tc05::mbar_init(drain, 1);
        tc05::fence_mbar_init();
    }
    if (SWAP && warp == 0 && lane == 0 && first < tiles) {
        // The first stretch of the weights on its way into L2 while the kernel ahead in the stream
        // still runs: a prefetch returns nothing, so it may come before that one's stores (1 x
        // 4096 x 4096 among weights that L2 does not hold: 8.6 us a call without, 8.05 with).
        int tx, ty;
        tile_at(first, a.tiles_x, a.tiles_y, tx, ty);
        for (int g = g0; g < min(g1, g0 + AHEAD); ++g)
            asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(
                             reinterpret_cast<uint64_t>(&tmx)),
                         "r"(g * GK), "r"(tx * BM)
                         : "memory");
    }
    __syncwarp();
    tc05::fence_before();
    __syncthreads();
    tc05::fence_after();
    if (SWAP && split > 1)  // the others may write to this CTA's memory from now on
        asm volatile("barrier.cluster.arrive.relaxed.aligned;\n");
    griddep_wait();
    griddep_launch();
    const uint32_t tmem = tslot;

    // Sums of an adding thread: one row, half of the columns, in pairs.
    constexpr int HC = BN / 2, CW = HC < 16 ? HC : 16;  // CW: columns of one TMEM load
    const int row = (warp & 3) * 32 + lane, half = warp >= 8, c0 = half * HC;
    uint64_t acc[HC / 2];

    if (warp < 4) {
        if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        if (warp == 0 && lane == 0) {  // copies
            uint32_t n = 0;            // stages filled
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                int tx, ty;
                tile_at(t, a.tiles_x, a.tiles_y, tx, ty);
                for (int g = g0; g < g1; ++g, ++n) {
                    const uint32_t s = n % L::STAGES;
                    if (n >= L::STAGES && !wait_or_stop(&empty[s], (n / L::STAGES - 1) & 1, &stop)) {
                        ok = false;
                        break;
                    }
                    if (n == a.skip) continue;
                    const uint32_t dst = tc05::smem_u32(smem + s * L::STAGE);
                    expect_tx(&full[s], L::STAGE);
                    tma_box(dst, &tmx, g * GK, tx * BM, &full[s]);
                    tma_box(dst + L::A_ST, &tmy, g * GK, ty * BN, &full[s]);
                }
            }
            // What was issued has landed before shared memory goes, whichever role gives up.
            for (uint32_t k = n > L::STAGES ? n - L::STAGES : 0; k < n; ++k)
                if (k != a.skip) tc05::mbar_wait(&full[k % L::STAGES], (k / L::STAGES) & 1, DRAIN_ITERS);
        } else if (warp == 1 && lane == 0) {  // products
            constexpr uint32_t idesc = idesc_e4m3(BM, BN);
            uint32_t n = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step)
                for (int g = g0; g < g1; ++g, ++n) {
                    const uint32_t s = n % L::STAGES, b = n % L::BUFS;
                    ok = (n < L::BUFS || wait_or_stop(&tempty[b], (n / L::BUFS - 1) & 1, &stop)) &&
                         wait_or_stop(&full[s], (n / L::STAGES) & 1, &stop);
                    if (!ok) break;
                    tc05::fence_after();
                    const uint32_t at = tc05::smem_u32(smem + s * L::STAGE);
                    const uint64_t da = desc_sw128(at), db = desc_sw128(at + L::A_ST);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_e4m3(tmem + b * L::COLS, da + 2 * k, db + 2 * k, idesc, k > 0);
                    tc05::commit(&empty[s]);
                    tc05::commit(&tfull[b]);
                }
            tc05::commit(drain);  // and what was issued has read it, and written tensor memory
            tc05::mbar_wait(drain, 0, DRAIN_ITERS);
        } else if (warp >= 2) {  // scales (their loads in the adding warps made those wait: 711 us, 8192^3)
            const int r = tid - 64;  // row r and r + 64, or column r
            int t = first, g = g0;
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
                        if (g == g0) {
                            int tx, ty;
                            tile_at(t, a.tiles_x, a.tiles_y, tx, ty);
                            if (SWAP) {
                                x0 = a.xs + tx * a.xs_row;  // BM rows are a block
                                y0 = a.ys + min(ty * BN + r, a.y_rows - 1) * a.ys_row;
                            } else {
                                x0 = a.xs + min(tx * BM + r, a.x_rows - 1) * a.xs_row;
                                x1 = a.xs + min(tx * BM + r + 64, a.x_rows - 1) * a.xs_row;
                                y0 = a.ys + min(ty * BN, a.y_rows - 1) / GK * a.ys_row;
                                y1 = a.ys + min(ty * BN + HC, a.y_rows - 1) / GK * a.ys_row;
                            }
                        }
                        vx0[e] = x0[g * a.xs_group];
                        vy0[e] = y0[g * a.ys_group];
                        if (!SWAP) {
                            vx1[e] = x1[g * a.xs_group];
                            vy1[e] = y1[g * a.ys_group];
                        }
                        if (++g == g1) {
                            g = g0;
                            t += step;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float *to = sc[b][e0 + e];
                        if (SWAP) {
                            if (r < BN) to[r] = vx0[e] * vy0[e];
                        } else {
                            to[r] = vx0[e] * vy0[e];
                            to[r + 64] = vx1[e] * vy0[e];
                            to[BM + r] = vx0[e] * vy1[e];
                            to[BM + r + 64] = vx1[e] * vy1[e];
                        }
                    }
                }
                arrive(&sfull[b]);
            }
        }
        __syncwarp();  // the one-thread roles rejoin their warps
    } else {
        if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n");
        const uint32_t tbase = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
#pragma unroll
        for (int j = 0; j < HC / 2; ++j) acc[j] = 0;
        uint32_t n = 0;
        bool ok = true;
        for (int t = first; t < tiles && ok; t += step) {
            for (int g = g0; g < g1; ++g, ++n) {
                const uint32_t b = n % L::BUFS, sb = n / SB;
                ok = n % SB || wait_or_stop(&sfull[sb & 1], (sb / 2) & 1, &stop);
                const float *f = sc[sb & 1][n % SB] + (SWAP ? c0 : half * BM + row);
                uint64_t s2 = 0;
                if (!SWAP) asm("mov.b64 %0, {%1, %1};\n" : "=l"(s2) : "f"(*f));
                ok = ok && wait_or_stop(&tfull[b], (n / L::BUFS) & 1, &stop);
                ok = __all_sync(~0u, ok);
                if (!ok) break;
                tc05::fence_after();
                uint32_t d[2][CW];
                auto ask = [&](int c) {
                    if constexpr (CW == 16) tc05::ld16(tbase + b * L::COLS + c * CW, d[c & 1]);
                    else tc05::ld8(tbase + b * L::COLS + c * CW, d[c & 1]);
                };
                ask(0);
#pragma unroll
                for (int c = 0; c < HC / CW; ++c) {
                    tc05::wait_ld_regs(d[c & 1]);
                    if (c + 1 < HC / CW) {
                        ask(c + 1);
                    } else {
                        tc05::fence_before();
                        if (lane == 0) arrive(&tempty[b]);
                    }
#pragma unroll
                    for (int j = 0; j < CW / 2; ++j)
                        fma2(acc[c * CW / 2 + j], d[c & 1][2 * j], d[c & 1][2 * j + 1],
                             SWAP ? ((const uint64_t *)f)[c * CW / 2 + j] : s2);
                }
                __syncwarp();  // every lane has its scales
                if (n % SB == SB - 1 && lane == 0) arrive(&sempty[sb & 1]);
            }
            if (!ok || split > 1) break;
            int tx, ty;
            tile_at(t, a.tiles_x, a.tiles_y, tx, ty);
            const int m = tx * BM + row, col = ty * BN + c0;
            if (SWAP) {
#pragma unroll
                for (int j = 0; j < HC / 2; ++j) {
                    float v[2];
                    split2(acc[j], v[0], v[1]);
                    acc[j] = 0;
                    if (m < a.x_rows && col + 2 * j < a.y_rows) put_any(a.out, a.out_dtype, (col + 2 * j) * a.ldc + m, v[0]);
                    if (m < a.x_rows && col + 2 * j + 1 < a.y_rows)
                        put_any(a.out, a.out_dtype, (col + 2 * j + 1) * a.ldc + m, v[1]);
                }
            } else {
                const int m0 = tx * BM + (warp & 3) * 32;
                const long long at = (long long)m0 * a.ldc + col;
                uint4 *stage = (uint4 *)(smem + L::OUT) + (warp - 4) * 128;
                const int rows = a.x_rows - m0, cols = a.y_rows - col;
                if (a.out_dtype == HV_BF16) store_rows((__nv_bfloat16 *)a.out + at, a.ldc, rows, cols, a.vec, stage, acc);
                else if (a.out_dtype == HV_F16) store_rows((__half *)a.out + at, a.ldc, rows, cols, a.vec, stage, acc);
                else store_rows((float *)a.out + at, a.ldc, rows, cols, a.vec, stage, acc);
#pragma unroll
                for (int j = 0; j < HC / 2; ++j) acc[j] = 0;
            }
        }
    }

    if (SWAP && split > 1) {
        // Each rank has a share of the output's rows (the tokens), and the others send it their sums
        // of those as they finish: one cluster barrier and no remote reads (1 x 4096 x 4096 7.3 ->
        // 6.9 us, 8 x 1024 x 16384 10.7 -> 10.2).
        int tx, ty;
        tile_at(first, a.tiles_x, a.tiles_y, tx, ty);
        const int cols = min(BN, a.y_rows - ty * BN), per = (cols + split - 1) / split;
        float *sums = (float *)(smem + L::OUT);  // [split][per][BM]
        __syncwarp();
        cluster_wait();  // every CTA has begun
        if (warp >= 4) {
            int owner = c0 / per, in = c0 - owner * per;
#pragma unroll
            for (int j = 0; j < HC / 2; ++j) {
                float v[2];
                split2(acc[j], v[0], v[1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (c0 + 2 * j + e < cols)
                        st_peer(tc05::smem_u32(sums + (rank * per + in) * BM + row), owner, v[e]);
                    if (++in == per) in = 0, ++owner;
                }
            }
        }
        cluster_sync();
        const int from = rank * per, share = min(per, cols - from);
        for (int i = tid; i < share * (BM / 4); i += THREADS) {
            const int p = i / (BM / 4), q = i % (BM / 4) * 4;
            float4 v = *(const float4 *)(sums + p * BM + q);
            for (int k = 1; k < split; ++k) {
                const float4 x = *(const float4 *)(sums + (k * per + p) * BM + q);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            put4_any(a, (ty * BN + from + p) * a.ldc + tx * BM + q, a.x_rows - tx * BM - q, v);
        }
    } else if (BN < 256 && split > 1) {
        // Every copy and product of this CTA has completed (or its waits gave up and were
        // drained): the ring's memory takes the sums.
        constexpr int LD = BN + 4;
        static_assert(BN == 256 || BM * LD * 4 <= L::SC, "the sums fit where the ring was");
        float *part = (float *)smem;
        __syncthreads();
        if (warp >= 4)
#pragma unroll
            for (int j = 0; j < HC / 2; j += 2) {
                float4 v;
                split2(acc[j], v.x, v.y);
                split2(acc[j + 1], v.z, v.w);
                *(float4 *)(part + row * LD + c0 + 2 * j) = v;
            }
        cluster_sync();
        int tx, ty;
        tile_at(first, a.tiles_x, a.tiles_y, tx, ty);
        // Each rank has a share of the output's rows, four neighbouring elements a thread.
        const int per = (BM + split - 1) / split, from = rank * per, share = min(per, BM - from);
#pragma unroll 2
        for (int i = tid; i < share * (BN / 4); i += THREADS) {
            const int p = from + i / (BN / 4), q = i % (BN / 4) * 4;
            const uint32_t at = tc05::smem_u32(part + p * LD + q);
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < split ? ld_peer(at, k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 1; k < 8; ++k) v[0].x += v[k].x, v[0].y += v[k].y, v[0].z += v[k].z, v[0].w += v[k].w;
            if (tx * BM + p < a.x_rows)
                put4_any(a, (tx * BM + p) * a.ldc + ty * BN + q, a.y_rows - ty * BN - q, v[0]);
        }
        cluster_sync();  // no CTA leaves while its sums may be read
    }
    __syncwarp();
    tc05::fence_before();
    __syncthreads();
    if (tid == 0 && stop) atomicOr(a.err, HV_DECODE_STALLED);  // every role has been through
    if (warp == 2) {
        tc05::fence_after();
        tc05::tmem_dealloc(tmem, L::TMEM);
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
cudaLaunchConfig_t config(unsigned grid, int split, cudaStream_t st, cudaLaunchAttribute (&attr)[2]) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Lay<BN, SWAP>::BYTES;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cfg;
}

// How many ways K is split: the most of 2, 3, 4 and 8 that leaves every cluster resident at once
// and a CTA two groups.  (A second wave of clusters costs more than it saves: 512 x 4096 x 4096
// took 19 us unsplit and 284 split eight ways.  Five or six shares of 1 x 4096 x 4096 took 7.5
// us, four 6.8; of 48 x 10240 x 4096 one took 20 us, two 17.6, three 15.8.)  How many clusters a
// device holds is asked once; the answer counts one CTA an SM for kernels with tensor memory, of
// which PER_SM fit.
template <int BN, bool SWAP>
int split_of(int64_t tiles, int groups) {
    static std::atomic<int> held[64][9];  // clusters of each size, plus one
    int dev = 0, best = 1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 1;
    for (int s = 2; s <= 8 && 2 * s <= groups && tiles * s <= 2 * 512; s = s == 2 ? 3 : s == 3 ? 4 : 2 * s) {
        int n = held[dev][s].load(std::memory_order_relaxed) - 1;
        if (n < 0) {
            cudaLaunchAttribute attr[2];
            const cudaLaunchConfig_t cfg = config<BN, SWAP>((unsigned)s, s, nullptr, attr);
            if (cudaOccupancyMaxActiveClusters(&n, gemm_kernel<BN, SWAP>, &cfg) != cudaSuccess) {
                (void)cudaGetLastError();
                n = 0;
            }
            held[dev][s].store(n + 1, std::memory_order_relaxed);
        }
        if (tiles <= n * Lay<BN, SWAP>::PER_SM) best = s;
    }
    return best;
}

template <int BN, bool SWAP>
int run(const Operand &x, const Operand &y, int k, GemmFp8Args a, int sms, cudaStream_t st) {
    CUtensorMap tmx, tmy;
    if (!tensor_map(&tmx, x.p, x.rows, k, x.stride, BM) || !tensor_map(&tmy, y.p, y.rows, k, y.stride, BN))
        return fail(HV_ERR_CUDA, "gemm_fp8: cannot encode the operands' tensor maps");
    a.xs = x.scale, a.xs_row = x.s_row, a.xs_group = x.s_group;
    a.ys = y.scale, a.ys_row = y.s_row, a.ys_group = y.s_group;
    a.x_rows = (int)x.rows, a.y_rows = (int)y.rows;
    a.tiles_x = (int)((x.rows + BM - 1) / BM), a.tiles_y = (int)((y.rows + BN - 1) / BN);
    const int64_t tiles = (int64_t)a.tiles_x * a.tiles_y;
    if (tiles > INT32_MAX / 16) return fail(HV_ERR_VALUE, "gemm_fp8: too many tiles");
    const auto kernel = gemm_kernel<BN, SWAP>;
    static std::atomic<uint64_t> ready;
    cudaError_t e = allow_shared(kernel, ready);
    if (e == cudaSuccess) {
        a.split = BN == 256 ? 1 : split_of<BN, SWAP>(tiles, a.groups);
        const int64_t grid = a.split > 1 ? tiles * a.split : std::min<int64_t>(tiles, sms * Lay<BN, SWAP>::PER_SM);
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t cfg = config<BN, SWAP>((unsigned)grid, a.split, st, attr);
        e = cudaLaunchKernelEx(&cfg, kernel, tmx, tmy, a);
    }
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
    g.skip = dec::skipped_copy();
    // 16-byte stores: rows start on 16 bytes and are whole groups of them
    const int es = dec::elem_size(p->out_dtype);
    g.vec = dec::aligned(p->d_out, 16) && n * es % 16 == 0 && (m == 1 || p->out_stride * es % 16 == 0);
    const Operand a{p->d_a, m, sa, p->d_a_scale, p->a_scale_strides[0], p->a_scale_strides[1]};
    const Operand b{p->d_b, n, sb, p->d_b_scale, p->b_scale_strides[0], p->b_scale_strides[1]};
    const cudaStream_t st = (cudaStream_t)stream;
    const int kk = (int)k;
    if (m <= 16) return run<16, true>(b, a, kk, g, sms, st);
    if (m <= 32) return run<32, true>(b, a, kk, g, sms, st);
    if (m <= 64) return run<64, true>(b, a, kk, g, sms, st);
    // A 256-wide tile's group takes about the time of 1.5 of a 128-wide one's, which may split K.
    const int64_t tm = (m + BM - 1) / BM, t128 = tm * ((n + 127) / 128), t256 = tm * ((n + 255) / 256);
    const int64_t waves128 = (t128 + sms - 1) / sms, waves256 = (t256 + sms - 1) / sms;
    if (3 * waves256 <= 2 * waves128) return run<256, false>(a, b, kk, g, sms, st);
    return run<128, false>(a, b, kk, g, sms, st);
}
