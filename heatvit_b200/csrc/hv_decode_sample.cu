// hv_decode_sample.cu — a token for each row of logits, from one given uniform number a row.
//
//   w_i = exp((z_i - max z) / T);  kept: of the tokens ordered by z (equal ones by index) the first
//   top_k, of those the ones with w >= min_p, of those the shortest prefix whose weights reach top_p
//   of their sum.  Token: the first i, in the vocabulary's order, with sum_{j <= i, kept} w_j > u total.
//
// Every set that is kept is "all above a cut": a logit and, for those equal to it, the last index.
// So the work is passes over the row: its maximum; for top_k and top_p a search for the cut; and the
// sums of the kept weights, warp by warp in the vocabulary's order, in which the token is found.  A
// cluster of CTAs takes a row and holds it in shared memory, so that HBM is read once.
//
// Weights are whole numbers, round(w 2^s) with s = 45 for rows of up to 2^17 tokens: their sums are
// exact in 64 bits in whatever order they are added, so that a border between two tokens lies at one
// place for every pass, and the same bits come again.  w itself is taken in 64 bits (2^-35 of it off at
// most): in 32 the sum of a flat row of 131072 would be off by enough to move one draw in a hundred.
// That exponential is eleven operations in 64 bits, of which an SM has 64 a clock: 42 of the 201 us of 1024 x 65536 uncut.
// Reading, the maximum and the meetings take 118 (a greedy call, which weighs nothing).  (A table of roots of two saves
// three of the eleven and its reads collide in shared memory: 272 us with it when it took 225 without.)
//
// The search: the logits of the interval that holds the cut are counted in NB bins; bounds of the
// bins' weights give a narrower interval; a pass with exact sums checks it.  When it holds CAP logits
// or fewer these are sorted and the cut is read off; when it holds one value, by its count.  An
// interval that the bins do not narrow is halved by its bit patterns, so that the search ends.
//
// Measured on one B200, in a graph: 1024 x 65536 of float32 201 us uncut (1.3 TB/s),
// 118 greedy, which weighs nothing; 256 x 131072 of bfloat16 with top_p 0.95 219 to 379, the more the flatter; 48 x 50021 of float32 15.5 uncut, 32 with top_k 50, 64 with top_p
// 0.95; 1 x 1000 3.7 greedy, 6 uncut, 20 with a search, whose steps wait for one another.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>

#include "hv_decode.cuh"

namespace hv {
namespace {

using namespace dec;
namespace cg = cooperative_groups;

constexpr int THREADS = 512, WARPS = THREADS / 32, NB = 1024, CAP = THREADS, MAX_CLUSTER = 8;
constexpr int HELD_BYTES = 200 * 1024;  // of a row's slice in shared memory, at most
typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    long long *tokens;
    float *logprobs;
    long long stride;
    int vocab, slice, shift, wide, k;  // slice: logits of a CTA, a multiple of a warp's chunk
    float t, p, min;
    int *err;
};

// Numbers as integers of their order.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.f);  // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The next number up, and down (the key of -0 stands between those of 0 and its neighbour below).
__device__ __forceinline__ float after(float z) { return of_key(key_of(z) + 1); }
__device__ __forceinline__ float ahead_of(float z) {
    const uint32_t k = key_of(z) - 1;
    return of_key(k == 0x7fffffffu ? k - 1 : k);
}

// round(2^((z - m) c) 2^shift) of a logit that is not so low that this is under a half: 2^x as 2^(n/2) 2^r, n/2 the
// nearest half, by a polynomial of degree 6 fitted to 2^r on [-1/4, 1/4] (1.5e-11 = 2^-36 off at most).
struct Weigh {
    static constexpr u64 ZERO = 0x4330000000000000ull;  // 2^52: a number that it is added to has an integer in its low bits
    double m, c;
    float top;
    int shift;
    __device__ __forceinline__ u64 raw(float z) const {  // with the bits of ZERO, of a finite largest logit
        const double d = (double)z - m;
        constexpr double MAGIC = 6755399441055744.0 / 2;  // 1.5 * 2^52: a sum with it has halves as its last bit
        const double y = fma(d, c, MAGIC), r = fma(d, c, MAGIC - y);
        const int n = __double2loint(y);
        double p = fma(r, 0.00015391449075562332, 0.0013350080299276343);
        p = fma(p, r, 0.009618148088079028);
        p = fma(p, r, 0.055504057958650016);
        p = fma(p, r, 0.24022650652566854);
        p = fma(p, r, 0.6931471809395268);
        p = fma(p, r, 1.0);
        const double t = __hiloint2double((n & 1 ? 0x3ff6a09e : 0x3ff00000) + (((n >> 1) + shift) << 20), n & 1 ? 0x667f3bcd : 0);
        return (u64)__double_as_longlong(fma(p, t, 4503599627370496.0));
    }
    __device__ __forceinline__ u64 operator()(float z) const {
        if (top == CUDART_INF_F) return z == top ? 1ull << shift : 0;
        return raw(z) - ZERO;
    }
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// The row's kept logits so far: above `z`, or equal to it and not past index `i`.
struct Cut {
    float z;
    int i;
    __device__ __forceinline__ bool keeps(float v, int at) const { return v > z || (v == z && at <= i); }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// What a pass finds: sums and counts, and the keys of the extremes, of the whole row after meet().
struct Found {
    u64 above, in;
    uint32_t over, n, least, most;  // over and n: how many are in the sums
    __device__ __forceinline__ void add(const Found &o) {
        above += o.above, in += o.in, over += o.over, n += o.n;
        least = min(least, o.least), most = max(most, o.most);
    }
    __device__ __forceinline__ void over_lanes() {
        above = warp_sum(above), in = warp_sum(in);
        over = __reduce_add_sync(~0u, over), n = __reduce_add_sync(~0u, n);
        least = __reduce_min_sync(~0u, least), most = __reduce_max_sync(~0u, most);
    }
};

struct Shared {
    uint32_t hist[NB];
    u64 cand[CAP];  // inverted key, index: ascending is the order
    u64 sums[WARPS];
    Found parts[WARPS], of_rank[2][MAX_CLUSTER];
    uint32_t n;
    Cut cut;
    double bounds[WARPS][2];
    float lo, hi;
    int at, first_b, last_b;
};

// A row's slice as the cluster's CTA has it, and what the CTAs tell one another.
template <typename T, bool HELD>
struct Row {
    static constexpr int VEC = 16 / sizeof(T), CHUNK = 32 * VEC;
    const T *global;  // the row
    const T *held;    // the slice, ended with -inf to whole chunks
    Shared &sh;
    cg::cluster_group cluster;
    int first, end, wide, rank, ranks;
    uint32_t turn;

    __device__ __forceinline__ void sync() const {  // of the row's CTAs
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    }
    // Chunks of this warp: [c0, c1) of CHUNK neighbours each.
    __device__ __forceinline__ void chunks(int &c0, int &c1) const {
        const int all = (end - first + CHUNK - 1) / CHUNK, per = (all + WARPS - 1) / WARPS, w = threadIdx.x >> 5;
        c0 = min(all, w * per), c1 = min(all, c0 + per);
    }
    // This lane's VEC logits of a chunk.
    __device__ __forceinline__ void get(int chunk, float (&z)[VEC]) const {
        const int at = chunk * CHUNK + (threadIdx.x & 31) * VEC;
        alignas(16) T e[VEC];
        if (HELD) {
            *(uint4 *)e = *(const uint4 *)(held + at);
        } else if (wide && first + at + VEC <= end) {
            *(uint4 *)e = *(const uint4 *)(global + first + at);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) e[j] = first + at + j < end ? global[first + at + j] : from_f32<T>(-CUDART_INF_F);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[j] = to_f32(e[j]);
    }
    // f(VEC logits, index of the first) for the slice, warp by warp in its order; the whole warp calls it together.
    template <typename F>
    __device__ __forceinline__ void each_vec(F f) const {
        int c0, c1;
        chunks(c0, c1);
        for (int c = c0; c < c1; ++c) {
            float z[VEC];
            get(c, z);
            f(z, first + c * CHUNK + (int)(threadIdx.x & 31) * VEC);
        }
    }
    // f(logit, index) for the logits from l to h; a lane goes through its own.
    template <typename F>
    __device__ __forceinline__ void each_with(float l, float h, F f) const {
        each_vec([&](const float (&z)[VEC], int at) {
            uint32_t some = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) some |= (uint32_t)(z[j] >= l && z[j] <= h) << j;
#pragma unroll 1
            for (; some; some &= some - 1) {
                const int i = at + __ffs(some) - 1;
                f(to_f32(HELD ? held[i - first] : global[i]), i);
            }
            __syncwarp();
        });
    }
    // The sum of a warp's, then of every warp's and CTA's, findings.
    __device__ __forceinline__ Found meet(Found f) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        f.over_lanes();
        __syncthreads();
        if (lane == 0) sh.parts[warp] = f;
        __syncthreads();
        const int b = turn++ & 1;
        if (warp == 0) {
            f = lane < WARPS ? sh.parts[lane] : Found{0, 0, 0, 0, ~0u, 0};
            f.over_lanes();
            if (lane < ranks) cluster.map_shared_rank(&sh, lane)->of_rank[b][rank] = f;
        }
        sync();
        f = sh.of_rank[b][0];
        for (int r = 1; r < ranks; ++r) f.add(sh.of_rank[b][r]);
        return f;
    }
    // (What is read of another CTA's memory, and written to it, is so ahead of a meeting: a CTA may leave after its last.)
    // After meet(): what the CTAs ahead of this one found.
    __device__ __forceinline__ Found ahead() const {
        Found f{0, 0, 0, 0, ~0u, 0};
        for (int r = 0; r < rank; ++r) f.add(sh.of_rank[(turn & 1) ^ 1][r]);
        return f;
    }

    // And what the warps ahead of this one did.
    __device__ __forceinline__ Found warps_ahead() const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        Found f = lane < warp ? sh.parts[lane] : Found{0, 0, 0, 0, ~0u, 0};
        f.over_lanes();
        return f;
    }

    // Of the kept logits from l to hi: the sum and number of those above h, and of the others, with their extremes.
    template <typename W>
    __device__ __forceinline__ Found look(const Cut &cut, float l, float h, float hi, W weigh) {
        Found f{0, 0, 0, 0, ~0u, 0};
        float least = CUDART_INF_F, most = -CUDART_INF_F;
        each_with(fmaxf(l, cut.z), hi, [&](float z, int i) {
            if (!cut.keeps(z, i)) return;
            const u64 w = weigh(z);
            if (z > h) {
                f.above += w, ++f.over;
            } else {
                f.in += w, ++f.n;
                least = fminf(least, z), most = fmaxf(most, z);
            }
        });
        f.least = key_of(least), f.most = key_of(most);
        return meet(f);
    }
    // The sum and number of the kept logits, or of those that `cut` keeps and `but` does not.
    template <typename W>
    __device__ __forceinline__ Found sum(const Cut &cut, const Cut *but, W weigh) {
        Found f{0, 0, 0, 0, ~0u, 0};
        each_with(cut.z, but ? but->z : CUDART_INF_F, [&](float z, int i) {
            if (cut.keeps(z, i) && !(but && but->keeps(z, i))) f.in += weigh(z), ++f.n;
        });
        return meet(f);
    }
    // The sum of all weights, given a logit that weighs nothing and stands for all below it: no branches, no choices.
    __device__ __forceinline__ Found sum_all(const Weigh &weigh, float nothing) {
        Found f{0, 0, 0, 0, ~0u, 0};
        uint32_t n = 0;
        each_vec([&](const float (&z)[VEC], int) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) f.in += weigh.raw(fmaxf(z[j], nothing));
            n += VEC;
        });
        f.in -= n * Weigh::ZERO;
        return meet(f);
    }

    // The index of the r-th (from 1) of the kept logits equal to z, in the row's order.
    __device__ __forceinline__ int nth_equal(const Cut &cut, float z, u64 r) {
        const int lane = threadIdx.x & 31;
        Found f{0, 0, 0, 0, ~0u, 0};
        each_with(z, z, [&](float v, int i) { f.n += cut.keeps(v, i); });
        const uint32_t mine = __reduce_add_sync(~0u, f.n);
        meet(f);
        u64 before = ahead().n + warps_ahead().n;
        if (before < r && before + mine >= r) {  // in this warp's chunks
            int c0, c1;
            chunks(c0, c1);
            for (int c = c0; c < c1; ++c) {
                float v[VEC];
                get(c, v);
                const int at = first + c * CHUNK + lane * VEC;
                uint32_t n = 0;
#pragma unroll
                for (int j = 0; j < VEC; ++j) n += v[j] == z && cut.keeps(v[j], at + j);
                uint32_t incl = n;
                for (int o = 1; o < 32; o *= 2) {
                    const uint32_t x = __shfl_up_sync(~0u, incl, o);
                    if (lane >= o) incl += x;
                }
                const unsigned hit = __ballot_sync(~0u, before + incl >= r);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        u64 k = before + incl - n;
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            if (v[j] == z && cut.keeps(v[j], at + j) && ++k == r)
                                for (int q = 0; q < ranks; ++q) cluster.map_shared_rank(&sh, q)->at = at + j;
                    }
                    break;
                }
                before += __shfl_sync(~0u, incl, 31);
            }
        }
        sync();
        return sh.at;
    }

    // Counts of the kept logits of [lo, hi] in NB bins from the top, in rank 0, which then sets l and h everywhere: between
    // them lies, by bounds of the bins' weights, what brings `above` to `target`.  bound(z, up): a bound of a weight.
    template <typename B>
    __device__ __forceinline__ void narrow(const Cut &cut, float lo, float hi, u64 above, u64 target, B bound, float &l, float &h, uint32_t &number) {
        const int tid = threadIdx.x, lane = tid & 31;
        for (int i = tid; i < NB; i += THREADS) sh.hist[i] = 0;
        const float s = (float)NB / (hi - lo);
        sync();
        each_with(lo, hi, [&](float z, int i) {
            // the nearest integer to (hi - z) s - 1/2, by an addition whose last bit it is (NaN, of an infinite interval: the
            // first bin)
            const int b = __float_as_int(fmaxf(fmaf(hi - z, s, 8388607.5f), 8388608.f)) - 0x4b000000;
            if (cut.keeps(z, i)) atomicAdd(&sh.hist[min(NB - 1, b)], 1u);
        });
        __syncthreads();
        if (rank) {
            uint32_t *to = cluster.map_shared_rank(&sh, 0)->hist;
            for (int i = tid; i < NB; i += THREADS)
                if (sh.hist[i]) atomicAdd(to + i, sh.hist[i]);
        }
        sync();
        if (rank == 0) {
            // Bounds of the sums down to each bin, neighbouring bins a thread; the first bin that may reach the target and
            // the first that must.
            constexpr int PER = NB / THREADS;
            const int warp = tid >> 5;
            double most[PER], least[PER], m0 = 0, l0 = 0;
            uint32_t count[PER], all = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int b = tid * PER + i;
                count[i] = sh.hist[b];
                most[i] = count[i] ? count[i] * bound(fminf(hi, hi - (b - 0.05f) / s), true) : 0.0;
                least[i] = count[i] ? count[i] * bound(fmaxf(lo, hi - (b + 1.05f) / s), false) : 0.0;
                m0 += most[i], l0 += least[i], all += count[i];
            }
            const double m_own = m0, l_own = l0;
            all = __reduce_add_sync(~0u, all);
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(~0u, m0, o), w = __shfl_up_sync(~0u, l0, o);
                if (lane >= o) m0 += v, l0 += w;
            }
            if (tid == 0) sh.first_b = sh.last_b = NB;
            if (lane == 31) sh.bounds[warp][0] = m0, sh.bounds[warp][1] = l0, sh.parts[warp].n = all;
            __syncthreads();
            all = 0;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) m0 += sh.bounds[w][0], l0 += sh.bounds[w][1];
                all += sh.parts[w].n;
            }
            m0 += (double)above - m_own, l0 += (double)above - l_own;  // ahead of this thread's bins
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                m0 += most[i], l0 += least[i];
                if (count[i] && m0 >= (double)target * (1 - 1e-9)) atomicMin(&sh.first_b, tid * PER + i);
                if (count[i] && l0 >= (double)target * (1 + 1e-9)) atomicMin(&sh.last_b, tid * PER + i);
            }
            __syncthreads();
            const int first_b = sh.first_b, last_b = sh.last_b;
            l = last_b >= NB ? lo : fmaxf(lo, hi - (last_b + 1.05f) / s);
            h = first_b >= NB ? hi : fminf(hi, hi - (first_b - 0.05f) / s);
            if (tid < ranks) {
                Shared *to = cluster.map_shared_rank(&sh, tid);
                to->lo = l, to->hi = h, to->n = all;
            }
        }
        sync();
        l = sh.lo, h = sh.hi, number = sh.n;
        if (!(l <= h)) l = lo, h = hi;
    }

    // The cut at which the weights of the kept logits, added in their order, first reach `target` (from 1 up to their
    // sum).  It lies in [lo, hi], with none above, and `number` of them at most.  kept: how many the cut keeps, or up to
    // CAP fewer.
    template <typename W, typename B>
    __device__ __forceinline__ Cut search(const Cut &cut, float lo, float hi, uint32_t number, u64 target, W weigh, B bound,
                                          uint32_t &kept) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        u64 above = 0;  // the sum of those above hi
        kept = 0;       // their number, for now
        bool halve = false;
        for (;;) {
            if (lo == hi) {  // one value
                const u64 w = weigh(lo), r = (target - above + w - 1) / w;
                kept += (uint32_t)r;
                return {lo, r >= number ? cut.z == lo ? cut.i : INT32_MAX : nth_equal(cut, lo, r)};
            }
            if (number <= CAP) {
                if (tid == 0) sh.n = 0, sh.cut = cut;  // (what was kept, unless a candidate says less)
                sync();
                Shared *to = cluster.map_shared_rank(&sh, 0);
                each_with(lo, hi, [&](float z, int i) {
                    if (cut.keeps(z, i)) to->cand[atomicAdd(&to->n, 1u)] = (u64)~key_of(z) << 32 | (uint32_t)i;
                });
                sync();
                if (rank == 0) {
                    number = sh.n;
                    int size = 32;
                    while (size < (int)number) size *= 2;
                    u64 mine = tid < (int)number ? sh.cand[tid] : ~0ull;
                    for (int k = 2; k <= size; k *= 2)  // bitonic, a candidate a thread
                        for (int j = k / 2; j; j /= 2) {
                            u64 its;
                            if (j >= 32) {
                                __syncthreads();
                                sh.cand[tid] = mine;
                                __syncthreads();
                                its = sh.cand[tid ^ j];
                            } else {
                                its = __shfl_xor_sync(~0u, mine, j);
                            }
                            if ((its < mine) == (!(tid & j) == !(tid & k))) mine = its;
                        }
                    // sums in order
                    const float z = of_key(~(uint32_t)(mine >> 32));
                    const u64 own = tid < (int)number ? weigh(z) : 0;
                    u64 s = own;
                    for (int o = 1; o < 32; o *= 2) {
                        const u64 v = __shfl_up_sync(~0u, s, o);
                        if (lane >= o) s += v;
                    }
                    if (lane == 31) sh.sums[warp] = s;
                    __syncthreads();
                    for (int w = 0; w < warp; ++w) s += sh.sums[w];
                    s += above;
                    if (tid < (int)number && s >= target && s - own < target)
                        for (int q = 0; q < ranks; ++q) cluster.map_shared_rank(&sh, q)->cut = {z, (int)(uint32_t)mine};
                }
                sync();
                return sh.cut;
            }
            const uint32_t kl = key_of(lo), kh = key_of(hi);
            float l, h;
            if (halve) {
                l = of_key(kl + (kh - kl) / 2 + ((kh - kl) & 1)), h = hi;
            } else {
                narrow(cut, lo, hi, above, target, bound, l, h, number);
            }
            halve = !halve && key_of(h) - key_of(l) >= (kh - kl) / 2;
            const Found f = look(cut, l, h, hi, weigh);
            if (above + f.above < target && target <= above + f.above + f.in) {
                lo = of_key(f.least), hi = of_key(f.most), above += f.above, kept += f.over, number = f.n;
                continue;
            }
            if (above + f.above >= target) lo = after(h);  // above what was tried
            else hi = ahead_of(l), above += f.above + f.in, kept += f.over + f.n;
            const Found g = look(cut, lo, hi, hi, [](float) -> u64 { return 0; });
            lo = of_key(g.least), hi = of_key(g.most), number = g.n;
        }
    }
};

// ceil(p sum) and floor(u sum), exactly, of numbers in [0, 1).
__device__ __forceinline__ u64 part_of(float p, u64 sum, bool up) {
    const u64 f = (u64)((double)p * 18446744073709551616.0);
    return __umul64hi(f, sum) + (up && f * sum != 0);
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    griddep_wait();
    griddep_launch();
    extern __shared__ __align__(16) uint8_t dyn[];
    Shared &sh = *(Shared *)dyn;
    T *held = (T *)(dyn + (sizeof(Shared) + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    // A CTA's memory may be written by another once it has begun: said here, waited for ahead of the first meeting.
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release;\n" ::: "memory");
    const long long r = blockIdx.x / ranks;
    const int first = (int)min((long long)a.vocab, (long long)rank * a.slice), end = (int)min((long long)a.vocab, first + (long long)a.slice);
    Row<T, HELD> row{(const T *)a.logits + r * a.stride, held, sh, cluster, first, end, a.wide, rank, ranks, 0};
    constexpr int VEC = Row<T, HELD>::VEC, CHUNK = Row<T, HELD>::CHUNK;
    // Settings: asked for ahead of the logits.
    const float temp = a.temperature ? a.temperature[r] : a.t, u = a.uniform[r];
    const float top_p = a.top_p ? a.top_p[r] : a.p, min_p = a.min_p ? a.min_p[r] : a.min;
    const int top_k = a.top_k ? a.top_k[r] : a.k;

    // The largest logit; a NaN stays one.
    float top = -CUDART_INF_F;
    auto larger = [&](float z) { top = max_nan(top, z); };
    if (HELD) {
        const int n = end - first, full = (n + CHUNK - 1) / CHUNK * CHUNK;
        if (a.wide) {
            const uint4 *from = (const uint4 *)(row.global + first);
            const int whole = n / VEC;
            constexpr int U = 8;  // loads of a thread under way
            for (int v0 = tid; v0 < whole; v0 += U * THREADS) {
                uint4 x[U];
#pragma unroll
                for (int q = 0; q < U; ++q)
                    if (v0 + q * THREADS < whole) x[q] = __ldcs(from + v0 + q * THREADS);
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int v = v0 + q * THREADS;
                    if (v >= whole) break;
                    ((uint4 *)held)[v] = x[q];
                    alignas(16) T e[VEC];
                    *(uint4 *)e = x[q];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) larger(to_f32(e[j]));
                }
            }
            for (int i = whole * VEC + tid; i < n; i += THREADS) {
                held[i] = row.global[first + i];
                larger(to_f32(held[i]));
            }
        } else {
#pragma unroll 8
            for (int i = tid; i < n; i += THREADS) {
                const T e = row.global[first + i];
                held[i] = e;
                larger(to_f32(e));
            }
        }
        for (int i = n + tid; i < full; i += THREADS) held[i] = from_f32<T>(-CUDART_INF_F);
    } else {
        row.each_vec([&](const float (&z)[VEC], int) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) larger(z[j]);  // (-inf past the slice's end)
        });
    }
    Found f{0, 0, 0, 0, ~0u, top == top ? key_of(top) : ~0u};
    if (ranks > 1) asm volatile("barrier.cluster.wait.acquire;\n" ::: "memory");
    f = row.meet(f);
    const float m = of_key(f.most);
    const bool none = f.most == ~0u || m == -CUDART_INF_F;
    if (none || !(temp > 0.f)) {
        const int at = none ? 0 : row.nth_equal({m, INT32_MAX}, m, 1);
        if (rank == 0 && tid == 0) {
            if (none) atomicOr(a.err, HV_DECODE_BAD_LOGITS);
            a.tokens[r] = at;
            if (a.logprobs) a.logprobs[r] = none ? CUDART_NAN_F : 0.f;
        }
        return;
    }
    const Weigh weigh{(double)m, 1.4426950408889634 / (double)temp, m, a.shift};

    // Logits that weigh nothing are never drawn: the lowest that may, and with min_p the lowest that is kept.  (The sum of
    // all weights has those below as well, so they must be zeros in it: half a unit, less far more than the 2^-35 that a
    // weight may be off.)
    Cut cut{-CUDART_MAX_NORMAL_F, INT32_MAX};
    const double lowest = (double)m - (a.shift + 1 + 1e-9) / weigh.c;
    if (lowest > cut.z) cut.z = fminf(__double2float_ru(lowest), m);
    const float live = cut.z, nothing = fmaxf(__double2float_rd((double)m - (a.shift + 2) / weigh.c), -CUDART_MAX_NORMAL_F);
    if (min_p > 0.f) {
        const double least = (double)m + (double)temp * log((double)min_p);
        if (least == least) cut.z = fmaxf(cut.z, fminf(__double2float_ru(least), m));  // (inf * log(1) keeps all)
    }
    if (top_k > 0 && top_k < a.vocab) {
        const auto one = [](float) -> u64 { return 1; };
        const Found all = row.sum(cut, nullptr, one);
        uint32_t kept;
        if (all.in > (u64)top_k)
            cut = row.search(cut, cut.z, m, all.n, (u64)top_k, one, [](float, bool) { return 1.0; }, kept);
    }
    // The kept weights, a sum for each warp's chunks, and their total.
    // (2^-900 is still a number in 64 bits)
    const bool whole = cut.z == live && cut.i == INT32_MAX && m < CUDART_INF_F && ((double)nothing - weigh.m) * weigh.c > -900.0 &&
                       weigh(nothing) == 0;
    const Found all = whole ? row.sum_all(weigh, nothing) : row.sum(cut, nullptr, weigh);
    const uint32_t number = whole ? (uint32_t)a.vocab : all.n;
    u64 mine = sh.parts[warp].in, before = row.ahead().in + row.warps_ahead().in, total = all.in;
    if (top_p < 1.f && number > 1) {
        const u64 target = max(1ull, part_of(fmaxf(top_p, 0.f), total, true));
        const Cut was = cut;
        uint32_t kept;
        // Logits that all together could not make up the rest of the sum are under the cut.  A logit counts for at most half a
        // unit more than it weighs, which takes half a unit from what each has to weigh; where that leaves nothing (a
        // logarithm of -inf or NaN) the search has no floor.
        const double rest = ((1.0 - fmax(0.0, (double)top_p)) * (double)total / number - 0.5) / (double)(1ull << a.shift);
        const float floor = __double2float_rd((double)m + (double)temp * log(rest) * (1 + 1e-6) - 1e-6 * (double)temp);
        cut = row.search(was, floor == floor ? fminf(fmaxf(was.z, floor), m) : was.z, m, number, target, weigh, [&](float z, bool up) {
            const double w = (double)exp2f((float)(((double)z - weigh.m) * weigh.c)) * (double)(1ull << a.shift);
            return up ? w * (1 + 1e-5) + 1 : fmax(0.0, w * (1 - 1e-5) - 1);
        }, kept);
        // The sums again: of what is left, or less what is not, whichever is fewer logits.
        const bool less = kept > number / 2;
        const Found f = less ? row.sum(was, &cut, weigh) : row.sum(cut, nullptr, weigh);
        const u64 own = sh.parts[warp].in;
        const u64 ahead = row.ahead().in + row.warps_ahead().in;
        total = less ? total - f.in : f.in;
        before = less ? before - ahead : ahead;
        mine = less ? mine - own : own;
    }

    const u64 target = u >= 1.f ? total - 1 : u > 0.f ? part_of(u, total, false) : 0;
    if (before <= target && target < before + mine) {
        int c0, c1;
        row.chunks(c0, c1);
        for (int c = c0; c < c1; ++c) {
            float z[VEC];
            row.get(c, z);
            const int at = first + c * CHUNK + lane * VEC;
            u64 own = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) own += cut.keeps(z[j], at + j) ? weigh(z[j]) : 0;
            u64 s = own;
            for (int o = 1; o < 32; o *= 2) {
                const u64 v = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += v;
            }
            const unsigned hit = __ballot_sync(~0u, before + s > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    u64 k = before + s - own;
                    bool found = false;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        if (found || !cut.keeps(z[j], at + j)) continue;
                        k += weigh(z[j]);
                        if (k <= target) continue;
                        found = true;
                        a.tokens[r] = at + j;
                        if (a.logprobs)
                            a.logprobs[r] = (float)((z[j] == m ? 0.0 : ((double)z[j] - weigh.m) / (double)temp) -
                                                    log((double)total / (double)(1ull << a.shift)));
                    }
                }
                break;
            }
            before += __shfl_sync(~0u, s, 31);
        }
    }
}

template <typename T, bool HELD>
int launch(const SampleArgs &a, int rows, int ranks, cudaStream_t st) {
    static std::atomic<uint64_t> ready;
    const auto kernel = sample_kernel<T, HELD>;
    cudaError_t e = allow_shared(kernel, ready);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)rows * ranks);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = (sizeof(Shared) + 15) / 16 * 16 + (HELD ? (size_t)a.slice * sizeof(T) : 0);
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)ranks;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "sample_tokens: %s", cudaGetErrorString(e));
    return HV_OK;
}

template <typename T>
int launch(SampleArgs a, int rows, int sms, cudaStream_t st) {
    constexpr int CHUNK = 32 * 16 / sizeof(T);
    // CTAs of a row: until every SM has one and a slice is 64 KB, while slices have 4096 logits or more.  (48 x 50021 of
    // float32 over 2, 4, 8: 33, 29, 45 us with top_k = 50; 256 x 131072 of bfloat16 177, 149, 225.)
    int ranks = 1;
    while (ranks < MAX_CLUSTER && a.vocab / (2 * ranks) >= 4096 &&
           ((long long)rows * ranks < sms || (long long)a.vocab * sizeof(T) > 64ll * 1024 * ranks))
        ranks *= 2;
    if ((long long)rows * ranks > INT32_MAX) return fail(HV_ERR_VALUE, "too many rows for one call");
    a.slice = ((a.vocab + ranks - 1) / ranks + CHUNK - 1) / CHUNK * CHUNK;
    return (long long)a.slice * sizeof(T) <= HELD_BYTES ? launch<T, true>(a, rows, ranks, st) : launch<T, false>(a, rows, ranks, st);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_sample_tokens(const hv_sample_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (!dec::known_dtype(p->dtype)) return fail(HV_ERR_TYPE, "dtype must be HV_BF16, HV_F16 or HV_F32");
    if (p->rows < 0) return fail(HV_ERR_VALUE, "negative row count");
    if (p->vocab < 1 || p->vocab > (1 << 30)) return fail(HV_ERR_VALUE, "vocab must be in [1, 2^30]");
    if (p->rows == 0) return HV_OK;
    if (!p->d_logits || !p->d_uniform || !p->d_tokens) return fail(HV_ERR_VALUE, "null buffer");
    int *err = dec::error_word();
    const int sms = dec::sm_count();
    if (!err || !sms) return fail(HV_ERR_CUDA, "cannot read the device's properties");
    SampleArgs a{};
    a.logits = p->d_logits, a.uniform = p->d_uniform, a.temperature = p->d_temperature, a.top_p = p->d_top_p;
    a.min_p = p->d_min_p, a.top_k = p->d_top_k, a.tokens = (long long *)p->d_tokens, a.logprobs = p->d_logprobs;
    a.stride = p->row_stride, a.vocab = p->vocab, a.k = p->top_k, a.t = p->temperature, a.p = p->top_p, a.min = p->min_p;
    int bits = 0;
    while ((1ll << bits) < p->vocab) ++bits;
    a.shift = bits <= 17 ? 45 : 62 - bits;  // sums stay under 2^63
    a.wide = dec::aligned(p->d_logits, 16) && p->row_stride * dec::elem_size(p->dtype) % 16 == 0;
    a.err = err;
    const cudaStream_t st = (cudaStream_t)stream;
    return p->dtype == HV_BF16 ? launch<__nv_bfloat16>(a, p->rows, sms, st)
           : p->dtype == HV_F16 ? launch<__half>(a, p->rows, sms, st)
                                : launch<float>(a, p->rows, sms, st);
}
