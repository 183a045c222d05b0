// hv_decode_sample.cu — a token for each row of logits, from one given uniform number a row.
//
//   w_i = exp((z_i - max z) / T);  kept: of the tokens ordered by z (equal ones by index) the first
//   top_k, of those the ones with w >= min_p, of those the shortest prefix whose weights reach top_p
//   of their sum.  Token: the first i, in the vocabulary's order, with sum_{j <= i, kept} w_j > u total.
//
// Every set that is kept is "all above a cut": a logit and, for those equal to it, the last index.
// So the work is passes over the row: its maximum; for top_k and top_p a search for the cut; and the
// sums of the kept weights, warp by warp in the vocabulary's order, in which the token is found.
//
// Weights are whole numbers, round(w 2^s) with s = 45 for rows of up to 2^17 tokens: their sums are
// exact in 64 bits in whatever order they are added, so that a border between two tokens lies at one
// place for every pass, and the same bits come again.  w itself is taken in 64 bits (2^-39 of it off at
// most): in 32 the sum of a flat row of 131072 would be off by enough to move one draw in a hundred.
//
// The search: the logits of the interval that holds the cut are counted in NB bins; bounds of the
// bins' weights give a narrower interval; a pass with exact sums checks it.  When it holds CAP logits
// or fewer these are sorted and the cut is read off; when it holds one value, by its count.  An
// interval that the bins do not narrow is halved by its bit patterns, so that the search ends.
#include <math_constants.h>

#include "hv_decode.cuh"

namespace hv {
namespace {

using namespace dec;

constexpr int THREADS = 1024, WARPS = THREADS / 32, NB = 1024, CAP = 1024, VEC = 8;
typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    long long *tokens;
    float *logprobs;
    long long stride;
    int vocab, shift, wide, k;
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

// round(2^((z - m) c) 2^shift): 2^x as a power of two, a 32nd root of one from a table, and the series
// of 2^r, |r| <= 1/64, to r^4 (2^-39 off).
struct Weigh {
    const double *table;
    double m, c;
    float top;
    int shift;
    __device__ __forceinline__ u64 operator()(float z) const {
        if (z == top) return 1ull << shift;
        const double x = ((double)z - m) * c;
        if (!(x > -(double)(shift + 1))) return 0;
        constexpr double MAGIC = 6755399441055744.0 / 32;  // 1.5 * 2^52: its sum with x has 32nds as its last bit
        const double y = x + MAGIC, r = x - (y - MAGIC);
        const int n = __double2loint(y);
        double p = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);  // ln(2)^4 / 4!, ln(2)^3 / 3!
        p = fma(p, r, 0.2402265069591007);
        p = fma(p, r, 0.6931471805599453);
        p = fma(p, r, 1.0);
        p *= table[n & 31];
        p = __hiloint2double(__double2hiint(p) + (((n >> 5) + shift) << 20), __double2loint(p));
        return (u64)__double_as_longlong(p + 4503599627370496.0) & 0xfffffffffffffull;  // 2^52: p's integer in the low bits
    }
};

struct Shared {
    double table[32];
    uint32_t hist[NB];
    u64 cand[CAP];  // inverted key, index: ascending is the order
    u64 sums[WARPS][3];
    uint32_t words[WARPS][4];
    u64 sum[3];
    uint32_t word[4];
    float lo, hi;
    uint32_t n;
    int at;
};

// The row's kept logits so far: above `z`, or equal to it and not past index `i`.
struct Cut {
    float z;
    int i;
    __device__ __forceinline__ bool keeps(float v, int at) const { return v > z || (v == z && at <= i); }
};

// Calls f(logit, index) for the row's elements of this thread, in chunks of 32 * VEC neighbours a
// warp; each warp has a stretch of the row.
template <typename T, typename F>
__device__ __forceinline__ void each(const T *row, int vocab, bool wide, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seg = (vocab + WARPS * 32 * VEC - 1) / (WARPS * 32 * VEC) * (32 * VEC);
    const long long end = min((long long)vocab, (long long)(warp + 1) * seg);
    for (long long i = (long long)warp * seg + lane * VEC; i < end; i += 32 * VEC) {
        if (wide && i + VEC <= end) {
            alignas(16) T e[VEC];
#pragma unroll
            for (int q = 0; q < VEC * (int)sizeof(T) / 16; ++q) ((uint4 *)e)[q] = ((const uint4 *)(row + i))[q];
#pragma unroll
            for (int j = 0; j < VEC; ++j) f(to_f32(e[j]), (int)i + j);
        } else {
            for (int j = 0; j < VEC && i + j < end; ++j) f(to_f32(row[i + j]), (int)i + j);
        }
    }
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
    for (int o = 16; o; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// What a pass finds of the interval [lo, hi], in all threads.
struct Found {
    u64 above, in;  // weights (or counts) above it and in it
    uint32_t n, least, most;  // how many are in it, and the keys of the extremes of those
};

template <typename T, typename W>
__device__ __forceinline__ Found look(Shared &sh, const T *row, const SampleArgs &a, const Cut &cut, float lo, float hi, W weigh) {
    u64 above = 0, in = 0;
    uint32_t n = 0, least = ~0u, most = 0;
    each(row, a.vocab, a.wide, [&](float z, int i) {
        if (z < lo || !cut.keeps(z, i)) return;
        const u64 w = weigh(z);
        if (z > hi) {
            above += w;
        } else {
            in += w;
            ++n;
            least = min(least, key_of(z));
            most = max(most, key_of(z));
        }
    });
    above = warp_sum(above), in = warp_sum(in);
    n = __reduce_add_sync(~0u, n), least = __reduce_min_sync(~0u, least), most = __reduce_max_sync(~0u, most);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) {
        sh.sums[warp][0] = above, sh.sums[warp][1] = in;
        sh.words[warp][0] = n, sh.words[warp][1] = least, sh.words[warp][2] = most;
    }
    __syncthreads();
    if (warp == 0) {
        above = warp_sum(sh.sums[lane][0]), in = warp_sum(sh.sums[lane][1]);
        n = __reduce_add_sync(~0u, sh.words[lane][0]), least = __reduce_min_sync(~0u, sh.words[lane][1]);
        most = __reduce_max_sync(~0u, sh.words[lane][2]);
        if (lane == 0) sh.sum[0] = above, sh.sum[1] = in, sh.word[0] = n, sh.word[1] = least, sh.word[2] = most;
    }
    __syncthreads();
    return {sh.sum[0], sh.sum[1], sh.word[0], sh.word[1], sh.word[2]};
}

// The index of the r-th (from 1) of the kept logits equal to z, in the row's order.
template <typename T>
__device__ __forceinline__ int nth_equal(Shared &sh, const T *row, const SampleArgs &a, const Cut &cut, float z, u64 r) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t n = 0;
    each(row, a.vocab, a.wide, [&](float v, int i) { n += v == z && cut.keeps(v, i); });
    const uint32_t total = __reduce_add_sync(~0u, n);
    __syncthreads();
    if (lane == 0) sh.words[warp][0] = total;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < warp; ++w) before += sh.words[w][0];
    if (before < r && before + total >= r) {  // in this warp's stretch
        const int seg = (a.vocab + WARPS * 32 * VEC - 1) / (WARPS * 32 * VEC) * (32 * VEC);
        const int end = min(a.vocab, (warp + 1) * seg);
        for (int i0 = warp * seg; i0 < end; i0 += 32) {
            const int i = i0 + lane;
            const float v = i < end ? to_f32(row[i]) : 0.f;
            unsigned m = __ballot_sync(~0u, i < end && v == z && cut.keeps(v, i));
            if (before + __popc(m) >= r) {
                for (u64 k = before + 1; k < r; ++k) m &= m - 1;
                if (lane == 0) sh.at = i0 + __ffs(m) - 1;
                break;
            }
            before += __popc(m);
        }
    }
    __syncthreads();
    return sh.at;
}

// The cut at which the weights of the kept logits, added in their order, first reach `target` (from 1 up to their
// sum), given that it lies in [lo, hi].  bound(z, up): a bound of a logit's weight, in double.
template <typename T, typename W, typename B>
__device__ __forceinline__ Cut search(Shared &sh, const T *row, const SampleArgs &a, const Cut &cut, float lo, float hi, u64 target,
                                      W weigh, B bound) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float l = lo, h = hi;  // what is tried: an interval in [lo, hi]
    bool halve = false;
    for (;;) {
        const Found f = look(sh, row, a, cut, l, h, weigh);
        if (f.above >= target) {  // above what was tried
            lo = of_key(key_of(h) + 1);
        } else if (f.above + f.in < target) {  // below
            hi = of_key(key_of(l) - 1);
        } else if (f.least == f.most) {  // one value
            const float z = of_key(f.least);
            const u64 w = weigh(z), r = (target - f.above + w - 1) / w;
            return {z, r >= f.n ? cut.z == z ? cut.i : INT32_MAX : nth_equal(sh, row, a, cut, z, r)};
        } else if (f.n <= CAP) {
            if (tid == 0) sh.n = 0;
            __syncthreads();
            each(row, a.vocab, a.wide, [&](float z, int i) {
                if (z >= l && z <= h && cut.keeps(z, i)) sh.cand[atomicAdd(&sh.n, 1u)] = (u64)~key_of(z) << 32 | (uint32_t)i;
            });
            int size = 32;
            while (size < (int)f.n) size *= 2;
            if (tid >= (int)f.n && tid < size) sh.cand[tid] = ~0ull;
            __syncthreads();
            for (int k = 2; k <= size; k *= 2)  // bitonic
                for (int j = k / 2; j; j /= 2) {
                    const int x = tid ^ j;
                    if (tid < size && x > tid) {
                        const u64 p = sh.cand[tid], q = sh.cand[x];
                        if ((p > q) == !(tid & k)) sh.cand[tid] = q, sh.cand[x] = p;
                    }
                    __syncthreads();
                }
            // sums in order: a candidate a thread
            const u64 mine = tid < (int)f.n ? sh.cand[tid] : 0;
            const float z = of_key(~(uint32_t)(mine >> 32));
            u64 s = tid < (int)f.n ? weigh(z) : 0;
            const u64 own = s;
            for (int o = 1; o < 32; o *= 2) {
                const u64 v = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += v;
            }
            if (lane == 31) sh.sums[warp][0] = s;
            __syncthreads();
            for (int w = 0; w < warp; ++w) s += sh.sums[w][0];
            s += f.above;
            if (tid < (int)f.n && s >= target && s - own < target) sh.lo = z, sh.at = (int)(uint32_t)mine;
            __syncthreads();
            return {sh.lo, sh.at};
        } else {
            lo = of_key(f.least), hi = of_key(f.most);
        }
        const uint32_t kl = key_of(lo), kh = key_of(hi);
        if (halve) {
            halve = false;
            l = of_key(kl + (kh - kl) / 2 + ((kh - kl) & 1)), h = hi;
            continue;
        }
        // Bins of [lo, hi] from the top; the weights above it are known where it was looked at, and looked at again here.
        halve = true;
        __syncthreads();
        for (int i = tid; i < NB; i += THREADS) sh.hist[i] = 0;
        const float s = (float)NB / (hi - lo);
        __syncthreads();
        u64 above = 0;
        each(row, a.vocab, a.wide, [&](float z, int i) {
            if (z < lo || !cut.keeps(z, i)) return;
            if (z > hi) above += weigh(z);
            else atomicAdd(&sh.hist[min(NB - 1, (int)((hi - z) * s))], 1u);
        });
        above = warp_sum(above);
        if (lane == 0) sh.sums[warp][0] = above;
        __syncthreads();
        if (warp == 0) {
            above = warp_sum(sh.sums[lane][0]);
            // bounds of the sums down to each bin, 32 bins a lane
            double most = 0, least = 0;
            for (int i = 0; i < NB / 32; ++i) {
                const int b = lane * (NB / 32) + i;
                most += sh.hist[b] * bound(fminf(hi, hi - (b - 0.05f) / s), true);
                least += sh.hist[b] * bound(fmaxf(lo, hi - (b + 1.05f) / s), false);
            }
            double m0 = most, l0 = least;
            for (int o = 1; o < 32; o *= 2) {
                const double v = __shfl_up_sync(~0u, m0, o), w = __shfl_up_sync(~0u, l0, o);
                if (lane >= o) m0 += v, l0 += w;
            }
            m0 += (double)above - most, l0 += (double)above - least;  // ahead of this lane's bins
            int first = NB, last = NB;  // the first bin that may reach the target, the first that must
            for (int i = 0; i < NB / 32; ++i) {
                const int b = lane * (NB / 32) + i;
                m0 += sh.hist[b] * bound(fminf(hi, hi - (b - 0.05f) / s), true);
                l0 += sh.hist[b] * bound(fmaxf(lo, hi - (b + 1.05f) / s), false);
                if (m0 >= (double)target * (1 - 1e-9) && first == NB) first = b;
                if (l0 >= (double)target * (1 + 1e-9) && last == NB) last = b;
            }
            first = __reduce_min_sync(~0u, first), last = __reduce_min_sync(~0u, last);
            if (lane == 0) {
                sh.hi = first >= NB ? hi : fminf(hi, hi - (first - 0.05f) / s);
                sh.lo = last >= NB ? lo : fmaxf(lo, hi - (last + 1.05f) / s);
            }
        }
        __syncthreads();
        l = sh.lo, h = sh.hi;
        if (!(l <= h)) l = lo, h = hi;
        if (key_of(h) - key_of(l) < (kh - kl) / 2) halve = false;
    }
}

// ceil(p sum) and floor(u sum), exactly, of numbers in [0, 1).
__device__ __forceinline__ u64 part_of(float p, u64 sum, bool up) {
    const u64 f = (u64)((double)p * 18446744073709551616.0);
    return __umul64hi(f, sum) + (up && f * sum != 0);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const __grid_constant__ SampleArgs a) {
    griddep_wait();
    griddep_launch();
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long r = blockIdx.x;
    const T *row = (const T *)a.logits + r * a.stride;
    if (tid < 32) sh.table[tid] = exp2(tid / 32.0);

    // The largest logit and the first index of it; a NaN shows as one above all.
    u64 best = 0;
    each(row, a.vocab, a.wide, [&](float z, int i) {
        const u64 v = (u64)(z == z ? key_of(z) : ~0u) << 32 | ~(uint32_t)i;
        best = max(best, v);
    });
    for (int o = 16; o; o /= 2) best = max(best, __shfl_xor_sync(~0u, best, o));
    if (lane == 0) sh.sums[warp][0] = best;
    __syncthreads();
    best = sh.sums[0][0];
    for (int w = 1; w < WARPS; ++w) best = max(best, sh.sums[w][0]);
    __syncthreads();
    const uint32_t top_key = (uint32_t)(best >> 32);
    const float m = of_key(top_key);
    if (top_key == ~0u || m == -CUDART_INF_F) {
        if (tid == 0) {
            atomicOr(a.err, HV_DECODE_BAD_LOGITS);
            a.tokens[r] = 0;
            if (a.logprobs) a.logprobs[r] = CUDART_NAN_F;
        }
        return;
    }
    const float temp = a.temperature ? a.temperature[r] : a.t;
    if (!(temp > 0.f)) {
        if (tid == 0) {
            a.tokens[r] = (uint32_t)~best;
            if (a.logprobs) a.logprobs[r] = 0.f;
        }
        return;
    }
    const float top_p = a.top_p ? a.top_p[r] : a.p, min_p = a.min_p ? a.min_p[r] : a.min;
    const int top_k = a.top_k ? a.top_k[r] : a.k;
    const Weigh weigh{sh.table, (double)m, 1.4426950408889634 / (double)temp, m, a.shift};

    // Logits that weigh nothing are never drawn: the lowest that may, and with min_p the lowest that is kept.
    Cut cut{-CUDART_MAX_NORMAL_F, INT32_MAX};
    const double lowest = (double)m - (a.shift + 2) / weigh.c;
    if (lowest > cut.z) cut.z = fminf(__double2float_rd(lowest), m);
    if (min_p > 0.f) {
        const double least = (double)m + (double)temp * log((double)min_p);
        if (least == least) cut.z = fmaxf(cut.z, fminf(__double2float_ru(least), m));  // (inf * log(1) keeps all)
    }

    if (top_k > 0 && top_k < a.vocab) {
        const auto one = [](float) -> u64 { return 1; };
        const Found all = look(sh, row, a, cut, cut.z, m, one);
        if (all.in > (u64)top_k)
            cut = search(sh, row, a, cut, of_key(all.least), m, (u64)top_k, one, [](float, bool) { return 1.0; });
    }
    Found kept = look(sh, row, a, cut, cut.z, m, weigh);
    if (top_p < 1.f && kept.n > 1) {
        const u64 target = max(1ull, part_of(fmaxf(top_p, 0.f), kept.in, true));
        cut = search(sh, row, a, cut, of_key(kept.least), m, target, weigh, [&](float z, bool up) {
            const double w = exp2(((double)z - weigh.m) * weigh.c) * (double)(1ull << a.shift);
            return up ? w * (1 + 1e-9) + 1 : fmax(0.0, w * (1 - 1e-9) - 1);
        });
    }

    // The kept weights, a sum for each warp's stretch of the row, and the token.
    u64 mine = 0;
    each(row, a.vocab, a.wide, [&](float z, int i) {
        if (cut.keeps(z, i)) mine += weigh(z);
    });
    mine = warp_sum(mine);
    __syncthreads();
    if (lane == 0) sh.sums[warp][0] = mine;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? sh.sums[w][0] : 0;
        total += sh.sums[w][0];
    }
    const float u = a.uniform[r];
    const u64 target = u >= 1.f ? total - 1 : u > 0.f ? part_of(u, total, false) : 0;
    if (before <= target && target < before + mine) {
        const int seg = (a.vocab + WARPS * 32 * VEC - 1) / (WARPS * 32 * VEC) * (32 * VEC);
        const int end = min(a.vocab, (warp + 1) * seg);
        for (int i0 = warp * seg; i0 < end; i0 += 32) {
            const int i = i0 + lane;
            const float z = i < end ? to_f32(row[i]) : 0.f;
            const u64 w = i < end && cut.keeps(z, i) ? weigh(z) : 0;
            u64 s = w;
            for (int o = 1; o < 32; o *= 2) {
                const u64 v = __shfl_up_sync(~0u, s, o);
                if (lane >= o) s += v;
            }
            const unsigned hit = __ballot_sync(~0u, before + s > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.tokens[r] = i;
                    if (a.logprobs)
                        a.logprobs[r] = (float)(((double)z == weigh.m ? 0.0 : ((double)z - weigh.m) / (double)temp) -
                                                log((double)total / (double)(1ull << a.shift)));
                }
                break;
            }
            before += __shfl_sync(~0u, s, 31);
        }
    }
}

template <typename T>
int launch(const SampleArgs &a, int rows, cudaStream_t st) {
    const cudaError_t e = launch_pdl(sample_kernel<T>, dim3((unsigned)rows), dim3(THREADS), 0, st, a);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "sample_tokens: %s", cudaGetErrorString(e));
    return HV_OK;
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
    if (!err) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
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
    return p->dtype == HV_BF16 ? launch<__nv_bfloat16>(a, p->rows, st)
           : p->dtype == HV_F16 ? launch<__half>(a, p->rows, st)
                                : launch<float>(a, p->rows, st);
}
