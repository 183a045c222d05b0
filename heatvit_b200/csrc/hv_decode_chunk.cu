// hv_decode_chunk.cu — attention of a chunk of new tokens of each sequence over a paged cache.
//
//   out[t, h] = sum_j softmax_j(scale * q[t, h] . K[j, h / group]) V[j, h / group],  j < seen(t),
//   seen(t) = lens - n + i + 1 for the i-th of a sequence's n new tokens (causal), or lens;
//   a row that sees nothing gives zeros (and a log-sum-exp of -inf).
//
// Bound by the tensor cores beside the softmax, and then by power, for long prompts (4 d multiply-adds a pair of tokens and
// head, at 128 x 128 x 128 in 520 clocks); with heads of 64 by the softmax, whose exponentials (one a pair and head, 16 a clock
// and SM) are a third of it and reads of tensor memory, maxima, conversions and sums the rest; and where few tokens see a
// long cache by HBM for a while, in a long run by power, since the rows of a tile that nobody has are worked on as well.
//
// Rows are (token, query head of a key head's group), so that a tile of 128 rows shares its keys
// whatever the group is.  One CTA an SM: 4 warps copy keys and values into a ring of tiles, by TMA in boxes of slots where
// pages are a multiple of eight tokens, else (and where a sequence ends) with cp.async, zeros past the end; one warp
// issues tcgen05.mma kind::f16; a row tile has two softmax warpgroups, a row in each of their threads and half of a
// step's 128 keys in each.  They read the scores from TMEM, keep the running maximum and sum, and write the weights to
// TMEM, where the second product takes them as its A operand; the sums stay in TMEM.
//
// Heads of up to 128 dimensions have two row tiles in flight (NT), whose products and weights take
// turns: two tiles of rows against the same keys, or, where an item has no more than 128
// rows, the same rows against the even and the odd key tiles, joined at the end.  Wider heads have one.
//
// Work: an item is a tile of NT * 128 rows of one sequence and key head; its key tiles are steps.  The
// steps of all items are laid end to end and every CTA takes an equal share of that line, so that
// ragged and causal batches are even and one long sequence uses every SM.  An item inside a share
// is written straight out; one that is cut leaves parts (unnormalised sums, maximum, sum of weights, in 32
// bits) in the workspace, and the CTA that finishes last joins them in the order of the shares.
//
// Measured on one B200 (calls in a long run): 8192 new tokens over 16384 (32 heads of 128 over 8, bf16) 3.08 to 3.13 ms at the
// power limit (1.7 GHz), 2.73 to 2.83 in bursts (972 to 1007 TFLOP/s); 16 x 6 tokens over 32768 482 us, likewise (991 W, 1.48 GHz),
// 382 to 410 in bursts (5.2 to 5.6 TB/s of cache); 24 prompts of up to 4001 tokens (24 heads of 64 over 6, fp16) 1.11 ms, short of that
// limit; 3 x 1499 of heads of 256 130 us with pages of 24 (boxes of 8 slots), 117 with pages of 16, 64 and 256, 202 with pages of one
// (cp.async): 18 steps an SM, of which the products are 1.1 us each, the ring (five slots, four a step) holding little ahead; 4 x 5 tokens
// over 300 24 us, latency; 3 tokens each of 256, 1024 and 4096 sequences 56, 154 and 608 us, as one warp of each CTA goes through them.  The operands
// of the products in uniform registers (the whole warp goes through the loop, one lane issues) took a 128^3 from 950 clocks
// to 520.  TMA, the second softmax warpgroup and the line's length in closed form came in together and were not timed
// apart: the first of these calls from 3.64 to 3.19 ms, the second from 580 to 506 us.
//
// A row's maximum moves only when it is passed by 2^SOFT, so that the sums are rarely rescaled.  The weights go
// into the second product rounded to the cache's type, and their sum is that of the rounded numbers: weights that are
// alike, and so rounded alike, cancel.  (As two numbers each, as attention of one token has them, they would
// take the tensor cores half as long again.)
//
// The second product multiplies masked values by zero, which a NaN or an infinity survives.  Slots past a
// sequence's end are zeros in shared memory; where a row does not see a token that others see, the warpgroup looks
// through the value tile, and one that holds such a number is added by its threads, each taking what its row sees.
// An infinite value that a row does see is its output's, unless the weight rounds to zero (fp16: under 2^-34 of the row's
// largest; bf16: under 2^-120), which makes a NaN of it.
#include <cudaTypedefs.h>
#include <math_constants.h>

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "hv_chunk_order.cuh"
#include "hv_decode.cuh"
#include "hv_tc05.cuh"

namespace hv {
namespace {

using namespace dec;

// A running maximum before the first score, finite so that a score of -inf weighs exp2(-inf) = 0 and not NaN.
constexpr float LOWEST = -3.402823466e38f;
// A row's largest weight is 2^TOP when its maximum moves, and 2^(TOP + SOFT) before it moves again.  bf16 weights stay at 1
// and below, so that sums of large values overflow no sooner than those of exact weights; fp16 ones begin at 2^9, so
// that those of a long tail keep their bits (normal numbers from 2^-14 to 2^15).
constexpr float SOFT = 6.f;
template <typename T>
constexpr float TOP = -SOFT;
template <>
constexpr float TOP<__half> = 9.f;
constexpr int BK = 128;       // keys of a step
constexpr int MIN_SHARE = 2;  // steps
constexpr int ITEM = 3;       // steps' time that an item takes beside its steps: its rows of q, the join and its output
constexpr int MAX_GRID = 512;
constexpr int LAG = 2;        // copies of a producer that are under way ahead of the one that is waited for

struct ChunkArgs {
    const void *q, *kc, *vc;
    void *out;
    float *lse;
    const int32_t *pages, *lens, *starts;
    long long q_tok, q_head, o_tok, o_head, lse_tok, lse_head;
    long long kc_page, kc_slot, kc_head, vc_page, vc_slot, vc_head, pages_stride;
    int tokens, seqs, heads, kv_heads, group, num_pages, page, page_shift, max_pages, causal, q_vec, o_vec, negate;
    float scale_log2;   // not negative: `negate` has the sign
    uint32_t skip;      // see skipped_copy
    float *parts;       // [grid][2][D / 4][R][4], then [grid][2][4][128][2]
    uint32_t *counts;   // [4][MAX_GRID], zero between calls
    int box;            // rows of a TMA box of the cache; 0: none
    int q_box;          // q by TMA
    int tp_shift;       // log2 of a row tile's tokens, where that is a whole power of two, or -1
    int *err;
};

// a / b, of numbers that nearly always fit in 32 bits.
__device__ __forceinline__ long long ratio(long long a, long long b) {
    return (unsigned long long)(a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

template <int D>
struct Lay {
    static constexpr chunk::Order ORDER = chunk::order_of(D);
    static constexpr int DP = chunk::padded_dim(D);  // dimensions in shared memory: 128-byte blocks of 64
    static constexpr int NT = ORDER.row_tiles, R = 128 * NT;
    static constexpr int PARTS = ORDER.parts, SLOT = BK / PARTS;  // keys of a ring slot
    static constexpr int SLOT_BYTES = SLOT * DP * 2, Q_TILE = 128 * DP * 2, Q_BYTES = NT * Q_TILE;
    static constexpr int STAGES = ORDER.stages;
    static constexpr int STAT = Q_BYTES + STAGES * SLOT_BYTES;  // [4][128] float: what the softmax warpgroups tell one another
    static constexpr int BARS = STAT + 2048, MISC = BARS + 336, BYTES = MISC + 160;
    // A row tile has two softmax warpgroups, with 64 keys of a step each; then four copying warps, then the products'.
    static constexpr int GROUPS = 2 * NT, SOFT_WARPS = 4 * GROUPS, MMA_WARP = SOFT_WARPS + 4, WARPS = SOFT_WARPS + 8, THREADS = WARPS * 32;
    // Registers of a thread at launch, and of the roles from then on (shares of what the block was launched with).
    static constexpr int REGS = NT == 2 ? 80 : 128, COPY_REGS = NT == 2 ? 56 : 72, MMA_REGS = NT == 2 ? 40 : 56;
    static constexpr int SOFT_REGS = NT == 2 ? 96 : 192;
    static_assert(128 * (COPY_REGS + MMA_REGS + GROUPS * SOFT_REGS) <= REGS * THREADS, "registers");
    // TMEM columns: scores, sums, weights.  APART: the weights have columns of their own, so that the next scores are
    // under way while they are made; with two row tiles of 128 dimensions they have to take the scores' place.
    static constexpr bool APART = ORDER.apart;
    // Heads of 256: the ring is so short that the slot of a step's last values may still await the step before's.
    static constexpr bool POLL_AFTER_SUMS = !ORDER.values_may_be_polled(false, 12);
    static_assert(ORDER.values_may_be_polled(POLL_AFTER_SUMS, 12), "a poll that may end on an older fill");
    __host__ __device__ static constexpr int s_col(int w) { return w * BK; }
    __host__ __device__ static constexpr int o_col(int w) { return 256 + w * DP; }
    __host__ __device__ static constexpr int p_col(int w, int h) {  // of the first and the last 64 keys
        return NT == 1 ? BK + h * 32 : APART ? 384 + w * 64 + h * 32 : w * BK + h * 64;
    }
    static constexpr int PART = R * D, CH = D / 8;  // numbers of a part; 16-byte pieces of a row
    static_assert(BYTES <= 227 * 1024 - 512, "shared memory");
    static_assert(o_col(NT) <= (APART && NT == 2 ? 384 : 512), "tensor memory");
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float exp2_(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void arrive(uint64_t *mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(tc05::smem_u32(mbar)) : "memory");
}
// One poll of phase `parity` of `bar`, for up to `ns` (the thread sleeps meanwhile).
__device__ __forceinline__ bool poll(uint64_t *bar, uint32_t parity, uint32_t ns) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(tc05::smem_u32(bar)), "r"(parity), "r"(ns)
        : "memory");
    return done;
}
// Bounded wait that also ends when another role of the CTA has given up.
__device__ __forceinline__ bool wait_or_stop(uint64_t *bar, uint32_t parity, volatile int *stop) {
    for (uint32_t i = 0; i < WAIT_ITERS; ++i) {
        if (poll(bar, parity, 2000)) return true;
        if (*stop) return false;
    }
    *stop = 1;
    return false;
}
// A 128-byte swizzled operand's descriptor: its high word, and its low one for an address.  K-major: atoms of eight rows
// of 128 bytes, 1024 apart; MN-major: the same atoms of eight k of 64 elements, the blocks of 64 along N `lbo` bytes apart.
// Steps within an operand are added to the low word, in 16 bytes.
constexpr uint32_t DESC_HI = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
// kind::f16, f32 accumulator.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn_major) {
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
// Issued by the one lane for which `leads`; the whole warp comes here, so that operands stay in uniform registers.
__device__ __forceinline__ void mma_ss(uint32_t leads, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 x, y;\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\n"
        "mov.b64 x, {%1, %4};\nmov.b64 y, {%2, %4};\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(DESC_HI), "r"(acc), "r"(leads)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leads, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p, q;\n.reg .b64 y;\nsetp.ne.b32 p, %5, 0;\nsetp.ne.b32 q, %6, 0;\n"
        "mov.b64 y, {%2, %4};\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(DESC_HI), "r"(acc), "r"(leads)
        : "memory");
}
__device__ __forceinline__ uint32_t elected() {
    uint32_t r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t *)&v;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *(uint32_t *)&v;
}
__device__ __forceinline__ float2 unpack(uint32_t v, __nv_bfloat16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t v, __half) { return __half22float2(*(const __half2 *)&v); }
// The largest magnitude's bits from which on numbers are infinite or NaN, twice.
__device__ __forceinline__ uint32_t infinite(__nv_bfloat16) { return 0x7f807f80u; }
__device__ __forceinline__ uint32_t infinite(__half) { return 0x7c007c00u; }
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void split2(uint64_t pair, float &lo, float &hi) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(pair));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A sequence's rows of q and cached tokens, brought into range (what is not is reported once, by `tell`).
struct Seq {
    int s0, n, len;
    __device__ __forceinline__ void set(const ChunkArgs &a, int b, bool tell) {
        const int r0 = a.starts[b], r1 = a.starts[b + 1], l = a.lens[b];
        s0 = min(max(r0, 0), a.tokens);
        const int s1 = min(max(r1, 0), a.tokens);
        n = max(s1 - s0, 0);
        const long long cap = min((long long)a.max_pages * a.page, (long long)HV_ATTENTION_MAX_LENGTH);
        len = (int)min((long long)max(l, 0), cap);
        if (tell) {
            if (s0 != r0 || s1 != r1 || s1 < s0) atomicOr(a.err, HV_DECODE_BAD_START);
            if (l > cap) atomicOr(a.err, HV_DECODE_BAD_LENGTH);
        }
    }
    // Tokens that the i-th new one sees.
    __device__ __forceinline__ int seen(const ChunkArgs &a, int i) const {
        return a.causal ? min(max(len - n + i + 1, 0), len) : len;
    }
    __device__ __forceinline__ int row_tiles(const ChunkArgs &a, int R) const {
        return (int)(((long long)n * a.group + R - 1) / R);
    }
    // Steps of a row tile: one at least, so that rows which see nothing are written.
    __device__ __forceinline__ int steps(const ChunkArgs &a, int R, int qt) const {
        if (!a.causal) return max(1, (len + BK - 1) / BK);
        const int last = (int)min((long long)(qt + 1) * R, (long long)n * a.group) - 1;
        return max(1, (seen(a, last / a.group) + BK - 1) / BK);
    }
};

// Steps [t0, t1) of the item (sequence b, key head h, row tile qt), of `steps` in all, as a share cuts them.  On the line an
// item has ITEM further places ahead of its steps: what it costs beside them.
template <int R>
struct Segment {
    Seq seq;
    int b, h, qt, qts, steps, t0, t1, x0, x1;  // x0, x1: its places of the line
    long long item, left;  // the line's index of the item's first place; places of the share from x0 on
    __device__ __forceinline__ void clip() {
        x1 = (int)min((long long)steps + ITEM, x0 + left);
        t0 = max(0, x0 - ITEM), t1 = max(0, x1 - ITEM);
    }
    __device__ __forceinline__ bool next(const ChunkArgs &a) {
        do {
            left -= x1 - x0;
            if (left <= 0) return false;
            item += steps + ITEM;
            x0 = 0;
            if (++qt == qts) {
                qt = 0;
                if (++h == a.kv_heads) {
                    h = 0;
                    do {
                        seq.set(a, ++b, false);  // only called where a further step exists
                        qts = seq.row_tiles(a, R);
                    } while (qts == 0);
                }
            }
            steps = seq.steps(a, R, qt);
            clip();
        } while (t0 == t1);
        return true;
    }
    // The shares that have its first and its last step.
    __device__ __forceinline__ int first_share(long long share) const { return (int)ratio(item + ITEM, share); }
    __device__ __forceinline__ int last_share(long long share) const { return (int)ratio(item + ITEM + steps - 1, share); }
    __device__ __forceinline__ int rows(const ChunkArgs &a) const {
        return (int)min((long long)R, (long long)seq.n * a.group - (long long)qt * R);
    }
};

// What a row's sums are multiplied by, and its log-sum-exp; a row that sees nothing has zeros.
__device__ __forceinline__ float row_factor(int seen, float l) { return seen > 0 ? 1.f / l : 0.f; }
__device__ __forceinline__ float row_lse(int seen, float m, float l) {
    return seen > 0 ? (m + log2f(l)) * 0.69314718055994531f : -CUDART_INF_F;
}

__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(Lay<D>::THREADS, 1)
    chunk_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                 const __grid_constant__ CUtensorMap tmq) {
    using L = Lay<D>;
    constexpr int NT = L::NT, R = L::R, DP = L::DP, SLOT = L::SLOT, PARTS = L::PARTS, STAGES = L::STAGES;
    extern __shared__ __align__(1024) uint8_t smem[];  // (with no static shared memory ahead of it)
    uint8_t *ring = smem + L::Q_BYTES;
    float *told = (float *)(smem + L::STAT);  // [softmax warpgroup][row]
    uint64_t *full = (uint64_t *)(smem + L::BARS), *empty = full + STAGES, *qfull = empty + STAGES, *qempty = qfull + 1;
    uint64_t *sfull = qempty + 1, *sfree = sfull + 2, *pready = sfree + 2, *odone = pready + 2, *tbar = odone + 2, *gbar = tbar + 2;
    uint64_t *both = gbar + 4, *drain = both + 1, *pair_bar = drain + 1;  // tbar: a row tile's warps, gbar: a warpgroup's
    static_assert((2 * STAGES + 26) * 8 <= 336, "barriers");
    long long *line = (long long *)(smem + L::MISC);  // whether this CTA has work (>= 0), a share of the line
    uint32_t *tslot = (uint32_t *)(line + 2);
    volatile int *stop = (volatile int *)(tslot + 1);
    volatile int *by_hand = stop + 1;        // [2]: this step's values are added by the warpgroup
    volatile int *last_flag = by_hand + 2;   // [2]
    Segment<R> *start = (Segment<R> *)(last_flag + 2);
    static_assert(sizeof(Segment<R>) <= 160 - 40 && L::MISC % 8 == 0, "the first segment");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == L::MMA_WARP) {
        tc05::tmem_alloc(tslot, 512);
        tc05::tmem_relinquish();
    }
    if (tid == 0) {
        *stop = tc05::smem_u32(smem) % 1024 != 0;  // operands would lie elsewhere than their descriptors say
        for (int i = 0; i < STAGES; ++i) {
            tc05::mbar_init(&full[i], 4);
            tc05::mbar_init(&empty[i], 1);
        }
        tc05::mbar_init(qfull, 4);
        tc05::mbar_init(qempty, 1);
        for (int i = 0; i < 2; ++i) {
            by_hand[i] = 0;
            tc05::mbar_init(&sfull[i], 1);
            tc05::mbar_init(&sfree[i], 8);
            tc05::mbar_init(&pready[i], 8);
            tc05::mbar_init(&odone[i], 1);
            tc05::mbar_init(&tbar[i], 8);
        }
        for (int i = 0; i < 4; ++i) tc05::mbar_init(&gbar[i], 4);
        for (int i = 0; i < 8; ++i) tc05::mbar_init(&pair_bar[i], 2);
        tc05::mbar_init(both, 16);
        tc05::mbar_init(drain, 1);
        tc05::fence_mbar_init();
    }
    griddep_wait();
    griddep_launch();

    // The line's length, this CTA's share of it, and the sequence of the share's first step.
    if (warp == 0) {
        // steps of each lane's sequence, for one key head
        Seq s{0, 0, 0};  // this lane's of the last 32 sequences
        auto steps_of = [&](int b, bool tell) {
            s = {0, 0, 0};
            if (b < a.seqs) s.set(a, b, tell);
            const int qts = s.n ? s.row_tiles(a, R) : 0;
            long long sum = 0;
            if (!a.causal) {
                sum = qts ? (long long)qts * s.steps(a, R, 0) : 0;
            } else {
                // Row tiles of tp whole tokens, of which the i-th sees off + i tp: the sum of ceil((off + i tp) / 128), in
                // closed form where one of tp and 128 is a multiple of the other.
                const int off = s.len - s.n, shift = a.tp_shift;
                const bool closed = shift >= 0 && off >= 0;
                if (qts && closed) {
                    const int full = s.n >> shift;
                    if (shift >= 7) {
                        sum = (long long)full * ((off + BK - 1) / BK) + ((long long)full * (full + 1) / 2 << (shift - 7));
                    } else {
                        const int m = 7 - shift;  // (off + 127 + i tp) / 128 = ((off + 127) / tp + i) / 2^m
                        auto down = [&](uint32_t k) {  // 0 / 2^m + 1 / 2^m + ... + k / 2^m, rounded down each
                            const long long q = k >> m;
                            return ((q * (q - 1) / 2) << m) + q * (long long)((k & ((1u << m) - 1)) + 1);
                        };
                        const uint32_t x = (uint32_t)(off + BK - 1) >> shift;
                        sum = down(x + full) - down(x);
                    }
                    if (full << shift < s.n) sum += s.steps(a, R, qts - 1);
                }
                unsigned many = __ballot_sync(~0u, qts && !closed);  // the others by the whole warp
                while (many) {
                    const int l = __ffs(many) - 1;
                    many &= many - 1;
                    const Seq o{0, __shfl_sync(~0u, s.n, l), __shfl_sync(~0u, s.len, l)};
                    const int its = __shfl_sync(~0u, qts, l);
                    long long part = 0;
                    for (int qt = lane; qt < its; qt += 32) part += o.steps(a, R, qt);
                    for (int x = 16; x; x /= 2) part += __shfl_xor_sync(~0u, part, x);
                    if (lane == l) sum += part;
                }
            }
            return sum + (long long)qts * ITEM;
        };
        long long total = 0, held = 0;
        for (int b0 = 0; b0 < a.seqs; b0 += 32) {
            held = steps_of(b0 + lane, blockIdx.x == 0);
            long long sum = held;
            for (int x = 16; x; x /= 2) sum += __shfl_xor_sync(~0u, sum, x);
            total += sum;
        }
        total *= a.kv_heads;
        const long long share = max((long long)(ITEM + MIN_SHARE), ratio(total + gridDim.x - 1, gridDim.x)), first = share * blockIdx.x;
        long long before = 0, per = 0;  // steps of the sequences ahead, and of the one that is found, for one key head
        int found = -1;
        Seq its{0, 0, 0};
        for (int b0 = 0; b0 < a.seqs && found < 0 && first < total; b0 += 32) {
            const long long n = a.seqs <= 32 ? held : steps_of(b0 + lane, false);
            long long incl = n;
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(~0u, incl, o);
                if (lane >= o) incl += v;
            }
            const unsigned m = __ballot_sync(~0u, (before + incl) * a.kv_heads > first);
            if (m) {
                const int l = __ffs(m) - 1;
                found = b0 + l;
                before += __shfl_sync(~0u, incl - n, l);
                per = __shfl_sync(~0u, n, l);
                its = {__shfl_sync(~0u, s.s0, l), __shfl_sync(~0u, s.n, l), __shfl_sync(~0u, s.len, l)};
            } else {
                before += __shfl_sync(~0u, incl, 31);
            }
        }
        if (found >= 0) {  // its first step: the key head, and the row tile within it
            Segment<R> seg;
            seg.b = found;
            seg.seq = its;
            seg.qts = seg.seq.row_tiles(a, R);
            seg.left = min(share, total - first);
            long long in = first - before * a.kv_heads;
            seg.h = (int)ratio(in, per);
            in -= seg.h * per;
            seg.qt = 0;
            if (!a.causal) {
                const int n = seg.seq.steps(a, R, 0) + ITEM;
                seg.qt = (int)ratio(in, n);
                in -= (long long)seg.qt * n;
            } else {
                for (; seg.qt < seg.qts; seg.qt += 32) {  // 32 row tiles at a time
                    const int qt = seg.qt + lane, n = qt < seg.qts ? seg.seq.steps(a, R, qt) + ITEM : 0;
                    long long incl = n;
                    for (int o = 1; o < 32; o <<= 1) {
                        const long long v = __shfl_up_sync(~0u, incl, o);
                        if (lane >= o) incl += v;
                    }
                    const unsigned m = __ballot_sync(~0u, incl > in);
                    if (m) {
                        const int l = __ffs(m) - 1;
                        in -= __shfl_sync(~0u, incl - n, l);
                        seg.qt += l;
                        break;
                    }
                    in -= __shfl_sync(~0u, incl, 31);
                }
            }
            seg.steps = seg.seq.steps(a, R, seg.qt);
            seg.x0 = (int)in;
            seg.item = first - in;
            seg.clip();
            if (seg.t0 == seg.t1 && !seg.next(a)) found = -1;
            if (lane == 0) *start = seg;
        }
        if (lane == 0) line[0] = found, line[1] = share;
    }
    __syncwarp();
    tc05::fence_before();
    __syncthreads();
    tc05::fence_after();
    const uint32_t tmem = *tslot;
    const long long share = line[1];
    const bool works = line[0] >= 0 && !*stop;
    Segment<R> seg;
    if (works) seg = *start;
    __syncwarp();
    constexpr bool APART = L::APART;
    constexpr chunk::Order ORDER = L::ORDER;

    if (warp >= L::SOFT_WARPS && warp < L::MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(L::COPY_REGS));
        const int w = warp - L::SOFT_WARPS;
        uint32_t fills = 0, qn = 0, waiting = 0;  // slots filled, items, copies by cp.async not yet reported
        uint64_t *pend[LAG + 1];
        bool ok = works;
        auto report = [&](uint64_t *bar) {
            tc05::fence_proxy_async();
            __syncwarp();
            if (lane == 0) arrive(bar);
        };
        auto flush = [&]() {
            if (!waiting) return;
            asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
            for (int i = 0; i <= LAG; ++i)
                if (i < (int)waiting) report(pend[i]);
            waiting = 0;
        };
        auto issued = [&](uint64_t *bar) {
            asm volatile("cp.async.commit_group;\n" ::: "memory");
#pragma unroll
            for (int i = 0; i <= LAG; ++i)
                if (i == (int)waiting) pend[i] = bar;
            if (++waiting > LAG) {
                asm volatile("cp.async.wait_group %0;\n" ::"n"(LAG) : "memory");
                report(pend[0]);
#pragma unroll
                for (int i = 0; i < LAG; ++i) pend[i] = pend[i + 1];
                --waiting;
            }
        };
        // Before a wait for room all that is on its way is reported, since room may depend on it.
        auto room = [&](uint64_t *bar, uint32_t parity) {
            if (__all_sync(~0u, tc05::mbar_wait(bar, parity, 1))) return true;
            flush();
            return (bool)__all_sync(~0u, wait_or_stop(bar, parity, stop));
        };
        auto expect = [&](uint64_t *bar, uint32_t bytes, bool arrives) {
            if (arrives)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(tc05::smem_u32(bar)), "r"(bytes) : "memory");
            else
                asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(tc05::smem_u32(bar)), "r"(bytes) : "memory");
        };
        constexpr int RW = SLOT / 4, N = RW * L::CH / 32;  // rows of a warp in a slot, accesses of a lane
        constexpr int NB = DP / 64;                         // blocks of 64 dimensions
        const int nb = a.box ? RW / a.box : 0;              // boxes of a warp's rows
        const int my_box = lane / NB, box_shift = __ffs(a.box) - 1;
        const T *kc = (const T *)a.kc, *vc = (const T *)a.vc;
        if (ok) do {
                const int n = seg.t1 - seg.t0, rows = seg.rows(a), head = seg.h;
                const bool alt = NT == 2 && rows <= 128;
                const int lead = ORDER.lead_of(alt);
                const long long table = seg.b * a.pages_stride;
                auto page_at = [&](int t) { return a.pages[table + (a.page_shift >= 0 ? t >> a.page_shift : t / a.page)]; };
                // Pages.  With boxes a lane holds one of a window of `steps` steps' boxes, so that loads are far ahead; else
                // that of its own row in the step whose values come next and two further ones.
                const int per_step = a.box ? PARTS * nb : 32, steps = 32 / per_step, step_shift = __ffs(steps) - 1;
                auto window = [&](int g) {
                    const int j = g * steps + lane / per_step, e = lane % per_step;
                    const int p = e / (a.box ? nb : 1), box = e - p * nb;
                    const int t = (seg.t0 + min(j, n - 1)) * BK + p * SLOT + w * RW + (box << box_shift);
                    return j < n && t < seg.seq.len ? page_at(t) : INT32_MIN;
                };
                struct Pages {
                    int of[PARTS];
                };
                auto own_pages = [&](int j) {
                    Pages r;
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        const int t = (seg.t0 + min(j, n - 1)) * BK + p * SLOT + w * RW + lane;
                        r.of[p] = lane < RW && j < n && t < seg.seq.len ? page_at(t) : INT32_MIN;
                    }
                    return r;
                };
                int now = 0, next = 0, at_window = 0;
                Pages p0 = {}, p1 = {}, p2 = {};
                if (a.box) now = window(0), next = window(1);
                else p0 = own_pages(0), p1 = own_pages(1), p2 = own_pages(2);
                // Keys or values of step j: by TMA the boxes that are live as a whole, row by row with cp.async what is not.
                auto fill = [&](int j, const Pages &own, bool keys) {
                    for (int p = 0; p < PARTS; ++p) {
                        const uint32_t s = fills % STAGES, dst = tc05::smem_u32(ring + s * L::SLOT_BYTES) + w * RW * 128;
                        const int t0 = (seg.t0 + j) * BK + p * SLOT + w * RW;
                        const int t = t0 + (a.box ? my_box << box_shift : lane);  // of this lane's box, or row
                        int page = PARTS == 1 || p == 0 ? own.of[0] : own.of[PARTS - 1];
                        if (a.box) {
                            const int from = (j & (steps - 1)) * per_step + p * nb + min(my_box, nb - 1);
                            page = __shfl_sync(~0u, j >> step_shift == at_window ? now : next, from);
                        }
                        bool good = (a.box ? my_box < nb : lane < RW) && t < seg.seq.len;
                        if (good && (page < 0 || page >= a.num_pages)) {
                            atomicOr(a.err, HV_DECODE_BAD_PAGE);
                            good = false;
                        }
                        const int slot = a.page_shift >= 0 ? t & (a.page - 1) : t % a.page;
                        const unsigned boxes = __ballot_sync(~0u, a.box && good && t + a.box <= seg.seq.len);
                        const bool all = a.box && __popc(boxes) == nb * NB;
                        if (fills >= STAGES && !room(&empty[s], (fills / STAGES - 1) & 1)) return false;
                        if (fills++ == a.skip) continue;
                        if (boxes) {
                            if (lane == 0) expect(&full[s], __popc(boxes) * a.box * 128, all);
                            __syncwarp();
                            if (boxes >> lane & 1)
                                asm volatile(
                                    "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
                                    "[%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst + lane % NB * (SLOT * 128) + (my_box << box_shift) * 128),
                                    "l"(reinterpret_cast<uint64_t>(keys ? &tmk : &tmv)), "r"(lane % NB * 64), "r"(slot), "r"(head),
                                    "r"(page), "r"(tc05::smem_u32(&full[s]))
                                    : "memory");
                            __syncwarp();
                        }
                        if (all) continue;
                        const int of = a.box ? (lane >> box_shift) * NB & 31 : lane;  // the lane that knows row `lane`
                        const int its = __shfl_sync(~0u, good ? page : -1, of), its_slot = __shfl_sync(~0u, slot, of);
                        const int at = a.box ? its_slot + (lane & (a.box - 1)) : its_slot;
                        long long off = -1;
                        if (lane < RW && its >= 0 && t0 + lane < seg.seq.len)
                            off = keys ? its * a.kc_page + at * a.kc_slot + head * a.kc_head : its * a.vc_page + at * a.vc_slot + head * a.vc_head;
#pragma unroll 4
                        for (int i = 0; i < N; ++i) {
                            const int c = i * 32 + lane, row = c / L::CH, col = c % L::CH;
                            const long long o = __shfl_sync(~0u, off, row);
                            if (a.box && boxes >> ((row >> box_shift) * NB) & 1) continue;
                            cp16(dst + (col >> 3) * (SLOT * 128) + row * 128 + (((col ^ row) & 7) << 4), (keys ? kc : vc) + (o < 0 ? 0 : o + col * 8),
                                 o < 0 ? 0 : 16);
                        }
                        issued(&full[s]);
                        if (a.box) flush();  // (the others are not reported behind it)
                    }
                    return true;
                };
                ok = fill(0, p0, true) && (!alt || n == 1 || fill(1, p1, true));
                if (!ok) break;
                // rows of q
                if (qn && !room(qempty, (qn - 1) & 1)) { ok = false; break; }
                const int tiles = NT == 2 && !alt ? 2 : 1;
                if (a.q_box) {  // [tokens][group][64] boxes; what is past the sequence is in no row that is written
                    if (w == 0) {
                        if (lane == 0) expect(qfull, tiles * L::Q_TILE, true);
                        __syncwarp();
                        if (lane < tiles * NB)
                            asm volatile(
                                "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
                                "[%5];\n" ::"r"(tc05::smem_u32(smem) + lane / NB * L::Q_TILE + lane % NB * (128 * 128)),
                                "l"(reinterpret_cast<uint64_t>(&tmq)), "r"(lane % NB * 64), "r"(head * a.group),
                                "r"(seg.seq.s0 + seg.qt * (R / a.group) + lane / NB * (128 / a.group)), "r"(tc05::smem_u32(qfull))
                                : "memory");
                        __syncwarp();
                    } else if (lane == 0) {
                        arrive(qfull);
                    }
                } else {
                    const T *q = (const T *)a.q + (long long)seg.seq.s0 * a.q_tok;
                    const long long r0 = (long long)seg.qt * R;
#pragma unroll 1
                    for (int g = w * 32; g < tiles * 128; g += 128) {
                        const int r = g + lane;
                        long long off = -1;
                        if (r < rows) {
                            const int at = (int)(r0 + r), tok = at / a.group;
                            off = tok * a.q_tok + (head * a.group + at - tok * a.group) * a.q_head;
                        }
                        const uint32_t dst = tc05::smem_u32(smem) + (g >> 7) * L::Q_TILE + (g & 127) * 128;
#pragma unroll 2
                        for (int i = 0; i < L::CH; ++i) {
                            const int c = i * 32 + lane, row = c / L::CH, col = c % L::CH;
                            const long long o = __shfl_sync(~0u, off, row);
                            const uint32_t to = dst + (col >> 3) * (128 * 128) + row * 128 + (((col ^ row) & 7) << 4);
                            if (a.q_vec) {
                                cp16(to, q + (o < 0 ? 0 : o + col * 8), o < 0 ? 0 : 16);
                            } else {
                                alignas(16) T e[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) e[k] = o < 0 ? from_f32<T>(0.f) : q[o + col * 8 + k];
                                const uint4 v = *(const uint4 *)e;
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                             : "memory");
                            }
                        }
                    }
                    issued(qfull);
                }
                ++qn;
                for (int j = 0; j < n && ok; ++j) {
                    Pages p3 = {};
                    if (!a.box) {
                        p3 = own_pages(j + 3);
                    } else if (j >> step_shift != at_window) {
                        at_window = j >> step_shift;
                        now = next;
                        next = window(at_window + 1);
                    }
                    if (!APART) ok = fill(j, p0, false);
                    if (ok && j + lead < n) ok = fill(j + lead, alt ? p2 : p1, true);
                    if (APART && ok) ok = fill(j, p0, false);
                    p0 = p1, p1 = p2, p2 = p3;
                }
                flush();
            } while (ok && seg.next(a));
        flush();
        if (a.box)  // what was issued has landed before shared memory goes, whichever role gives up
            for (uint32_t k = fills > STAGES ? fills - STAGES : 0; k < fills; ++k)
                if (k != a.skip)
                    for (uint32_t i = 0; i < DRAIN_ITERS && !poll(&full[k % STAGES], (k / STAGES) & 1, 2000); ++i)
                        if (*stop && i > 1000) break;
        if (a.q_box && qn)
            for (uint32_t i = 0; i < DRAIN_ITERS && !poll(qfull, (qn - 1) & 1, 2000); ++i)
                if (*stop && i > 1000) break;
        __syncwarp();
    } else if (warp >= L::MMA_WARP) {  // the products: one warp of its warpgroup
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(L::MMA_REGS));
        if (warp == L::MMA_WARP) {
            const uint32_t leads = elected();
            auto commit = [&](uint64_t *bar) {
                if (leads) tc05::commit(bar);
                __syncwarp();
            };
            constexpr uint32_t qk = idesc_f16<T>(128, SLOT, false), pv = idesc_f16<T>(128, DP, true);
            const uint32_t qk_idesc = qk | (a.negate ? 1u << 13 : 0);
            const uint32_t qs = tc05::smem_u32(smem), rs = tc05::smem_u32(ring);
            uint32_t base = 0, qn = 0, pn = 0, sn = 0, scored = 0;  // pn, sn: phase bits of either row tile's weights and scores
            bool ok = works;
            auto wait_all = [&](uint64_t *bar, uint32_t parity) { return (bool)__all_sync(~0u, wait_or_stop(bar, parity, stop)); };
            auto tile_full = [&](uint32_t f) {
                bool r = true;
#pragma unroll
                for (int p = 0; p < PARTS; ++p) r = r && wait_all(&full[(f + p) % STAGES], ((f + p) / STAGES) & 1);
                return r;
            };
            auto release = [&](uint32_t f) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p) commit(&empty[(f + p) % STAGES]);
            };
            // scores of row tile w: rows of q tile t against the keys of ring fill f
            auto scores = [&](int w, int t, uint32_t f) {
                if (APART) {  // the scores before have been read
                    if ((scored >> w & 1) && !wait_all(&sfree[w], sn >> w & 1 ^ 1)) return false;
                    sn ^= 1u << w;
                    scored |= 1u << w;
                }
                if (!tile_full(f)) return false;
                tc05::fence_after();
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    const uint32_t x = desc_lo(qs + t * L::Q_TILE, 16), y = desc_lo(rs + (f + p) % STAGES * L::SLOT_BYTES, 16);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_ss(leads, tmem + w * BK + p * SLOT, x + (k >> 2) * 1024 + (k & 3) * 2, y + (k >> 2) * (SLOT * 8) + (k & 3) * 2,
                               qk_idesc, k > 0);
                }
                commit(&sfull[w]);
                return true;
            };
            // sums of row tile w: its weights times the values of ring fill f
            auto sums = [&](int w, uint32_t f, bool add) {
                if (!tile_full(f) || !wait_all(&pready[w], pn >> w & 1)) return false;
                tc05::fence_after();
                if (!by_hand[w]) {
                    const uint32_t to = tmem + (w ? L::o_col(1) : L::o_col(0));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // halves of the keys
                        const uint32_t x = tmem + (w ? L::p_col(1, h) : L::p_col(0, h));
                        const uint32_t y = desc_lo(rs + (f + h * (PARTS - 1)) % STAGES * L::SLOT_BYTES, SLOT * 128) + (PARTS == 1 ? h * 512 : 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_ts(leads, to, x + k * 8, y + k * 128, pv, add || h || k);
                    }
                }
                pn ^= 1u << w;
                commit(&odone[w]);
                return true;
            };
            if (ok) do {
                    // Units: either row tile in turn against each step's keys, or the one against the steps in turn.
                    const int n = seg.t1 - seg.t0;
                    const bool alt = NT == 2 && seg.rows(a) <= 128, pair = NT == 2 && !alt;
                    const int lead = ORDER.lead_of(alt), all = pair ? 2 * n : n;
                    ok = wait_all(qfull, qn++ & 1);
                    // the scores of unit i, and the sums of unit i - NT behind them (APART) or ahead of them
                    for (int i = 0; i < all + NT && ok; ++i) {
#pragma unroll 1
                        for (int e = 0; e < 2 && ok; ++e) {
                            if ((e == 0) == APART) {
                                if (i >= all) continue;
                                const uint32_t f = base + ORDER.k_fill(pair ? i >> 1 : i, lead);
                                ok = scores(NT == 2 ? i & 1 : 0, pair ? i & 1 : 0, f);
                                if (!ok) break;
                                if (!pair || i & 1) release(f);
                                if (i + 1 == all) commit(qempty);
                            } else {
                                const int u = i - NT;
                                if (u < 0) continue;
                                const uint32_t f = base + ORDER.v_fill(pair ? u >> 1 : u, n, lead);
                                ok = sums(NT == 2 ? u & 1 : 0, f, u >= NT);
                                if (ok && (!pair || u & 1)) release(f);
                            }
                        }
                    }
                    base += 2 * n * PARTS;
                } while (ok && seg.next(a));
            commit(drain);  // what was issued has read shared memory and written tensor memory
            tc05::mbar_wait(drain, 0, DRAIN_ITERS);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(L::SOFT_REGS));
        // A warpgroup: half `h` of the keys of row tile `w`, a row in each thread.
        const int wg = warp >> 2, w = wg >> 1, h = wg & 1, row = tid & 127;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t otm = lanes + (w ? L::o_col(1) : L::o_col(0)), stm = lanes + w * BK + h * 64;
        const uint32_t ptm = lanes + (w ? (h ? L::p_col(1, 1) : L::p_col(1, 0)) : (h ? L::p_col(0, 1) : L::p_col(0, 0)));
        const float c = a.scale_log2;
        uint32_t un = 0, tn = 0, gn = 0, bn = 0, base = 0;  // units of this row tile; turns of the barriers
        bool hand = false, ok = works;
        auto meet = [&](uint64_t *bar, uint32_t &turn) {  // the warps that share a barrier
            __syncwarp();
            if (lane == 0) arrive(bar);
            return (bool)__all_sync(~0u, wait_or_stop(bar, turn++ & 1, stop));
        };
        // The sums of the unit before, and its weights, are the tensor core's until this.
        auto before_done = [&]() {
            if (!APART || !un) return true;  // (else scores come after it)
            const bool r = __all_sync(~0u, wait_or_stop(&odone[w], (un - 1) & 1, stop));
            tc05::fence_after();
            return r;
        };
        bool counted = false;
        if (ok) do {
                const int n = seg.t1 - seg.t0, rows = seg.rows(a);
                const bool alt = NT == 2 && rows <= 128;
                const int r = (alt ? 0 : w * 128) + row;
                const bool exists = r < rows;
                const int at = (int)((long long)seg.qt * R + r), tok = at / a.group;
                const int seen = exists ? seg.seq.seen(a, tok) : seg.seq.len;
                const int first_seen = seg.seq.seen(a, (int)((long long)seg.qt * R + r - row) / a.group);  // the tile's first row
                counted = false;
                float m = LOWEST, l = 0.f;
                bool fresh = true;
                for (int j = alt ? w : 0; j < n; j += alt ? 2 : 1) {
                    ok = __all_sync(~0u, wait_or_stop(&sfull[w], un & 1, stop));
                    if (!ok) break;
                    tc05::fence_after();
                    const int k0 = (seg.t0 + j) * BK + h * 64, lim = seen - k0;  // of this half
                    // The scores are read twice, 32 at a time: in registers all would have the loops unrolled, and those
                    // outgrow the instruction cache.
                    const bool masked = __any_sync(~0u, lim < 64);
                    float top = -CUDART_INF_F;
                    if (!masked) {
                        uint32_t x[2][32];
                        float t = -CUDART_INF_F;
                        tc05::ld32(stm, x[0]);
                        tc05::ld32(stm + 32, x[1]);
                        tc05::wait_ld_regs(x[0]);
                        tc05::wait_ld_regs(x[1]);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            top = fmaxf(fmaxf(top, __uint_as_float(x[0][i])), __uint_as_float(x[0][i + 1]));
                            t = fmaxf(fmaxf(t, __uint_as_float(x[1][i])), __uint_as_float(x[1][i + 1]));
                        }
                        top = fmaxf(top, t);
                    } else {
#pragma unroll 1
                        for (int g = 0; g < 64; g += 16) {
                            uint32_t x[16];
                            __syncwarp();
                            tc05::ld16(stm + g, x);
                            tc05::wait_ld_regs(x);
#pragma unroll
                            for (int i = 0; i < 16; ++i) top = fmaxf(top, g + i < lim ? __uint_as_float(x[i]) : -CUDART_INF_F);
                        }
                    }
                    // the row's over both halves
                    told[wg * 128 + row] = top;
                    uint32_t turn = un;
                    ok = meet(&pair_bar[w * 4 + (warp & 3)], turn);
                    if (!ok) break;
                    top = fmaxf(top, told[(wg ^ 1) * 128 + row]) * c;
                    if (__any_sync(~0u, top > m + (TOP<T> + SOFT))) {
                        const float to = fmaxf(top - TOP<T>, m), f = exp2_(m - to);
                        m = to;
                        l *= f;
                        if (!fresh) {
                            ok = before_done();
                            if (!ok) break;
#pragma unroll 1
                            for (int k = h * (D / 2); k < (h + 1) * (D / 2); k += 16) {
                                uint32_t o[16];
                                __syncwarp();
                                tc05::ld16(otm + k, o);
                                tc05::wait_ld_regs(o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tc05::st16(otm + k, o);
                            }
                        }
                    }
                    if (hand) {  // the products' warp has read it
                        ok = before_done() && meet(&tbar[w], tn);
                        if (!ok) break;
                        if (row == 0 && h == 0) by_hand[w] = 0;
                        hand = false;
                        ok = meet(&tbar[w], tn);
                        if (!ok) break;
                    }
                    uint32_t vf = 0;
                    if (first_seen < seg.seq.len && first_seen < k0 - h * 64 + BK) {
                        // Values that some row of the tile does not see: any that are no numbers?
                        if (L::POLL_AFTER_SUMS) {
                            ok = before_done();
                            if (!ok) break;
                        }
                        vf = base + ORDER.v_fill(j, n, ORDER.lead_of(alt));
                        const uint32_t fp = vf + h * (PARTS - 1);
                        ok = __all_sync(~0u, wait_or_stop(&full[fp % STAGES], (fp / STAGES) & 1, stop));
                        if (!ok) break;
                        const uint4 *v = (const uint4 *)(ring + fp % STAGES * L::SLOT_BYTES) + (PARTS == 1 ? h * 512 : 0);
                        uint32_t top2 = 0;
#pragma unroll 2
                        for (int i = row; i < 64 * L::CH; i += 128) {
                            const uint4 u = v[(i / 64 >> 3) * (SLOT * 8) + i % 64 * 8 + (((i / 64) ^ i) & 7)];
                            top2 = __vmaxu2(top2, u.x & 0x7fff7fffu), top2 = __vmaxu2(top2, u.y & 0x7fff7fffu);
                            top2 = __vmaxu2(top2, u.z & 0x7fff7fffu), top2 = __vmaxu2(top2, u.w & 0x7fff7fffu);
                        }
                        const bool bad = __vmaxu2(top2, infinite(T()) - 0x00010001u) != infinite(T()) - 0x00010001u;
                        if (__any_sync(~0u, bad) && lane == 0) by_hand[w] = 1;
                        ok = meet(&tbar[w], tn);
                        if (!ok) break;
                        hand = by_hand[w];
                    }
                    ok = before_done();
                    if (!ok) break;
                    const uint64_t c2 = two(c, c), m2 = two(-m, -m);
                    uint64_t sum2 = 0;
                    auto put = [&](uint32_t v) {
                        const float2 p = unpack(v, T());
                        sum2 = add2(sum2, two(p.x, p.y));
                    };
                    auto read = [&]() {  // the scores are
                        if (APART) {
                            tc05::fence_before();
                            __syncwarp();
                            if (lane == 0) arrive(&sfree[w]);
                        }
                    };
                    if (!masked) {
#pragma unroll 1
                        for (int g = 0; g < 2; ++g) {
                            uint32_t x[32], v[16];
                            __syncwarp();
                            tc05::ld32(stm + g * 32, x);
                            tc05::wait_ld_regs(x);
                            if (g) read();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const uint64_t y = fma2(two(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), c2, m2);
                                float lo, hi;
                                split2(y, lo, hi);
                                v[i] = pack(exp2_(lo), exp2_(hi), T());
                                put(v[i]);
                            }
                            __syncwarp();
                            tc05::st16(ptm + g * 16, v);  // (over scores that have been read)
                        }
                    } else {
#pragma unroll 1
                        for (int g = 0; g < 64; g += 16) {
                            uint32_t x[16];
                            __syncwarp();
                            tc05::ld16(stm + g, x);
                            tc05::wait_ld_regs(x);
                            if (g == 48) read();
                            uint32_t v[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float lo = exp2_(fmaf(__uint_as_float(x[2 * i]), c, -m));
                                const float hi = exp2_(fmaf(__uint_as_float(x[2 * i + 1]), c, -m));
                                v[i] = pack(g + 2 * i < lim ? lo : 0.f, g + 2 * i + 1 < lim ? hi : 0.f, T());
                                put(v[i]);
                            }
                            __syncwarp();
                            st8(ptm + g / 2, v);
                        }
                    }
                    tc05::wait_st();
                    float lo, hi;
                    split2(sum2, lo, hi);
                    l += lo + hi;
                    if (hand) {
                        // The weights times the values of ring fill vf, for the keys that a row sees alone: this half's
                        // dimensions, of all keys.
                        tc05::fence_before();
                        ok = meet(&tbar[w], tn);
                        if (!ok) break;
                        tc05::fence_after();
                        const int most = seen - (k0 - h * 64);
#pragma unroll 1
                        for (int k = h * (D / 2); k < (h + 1) * (D / 2); k += 8) {
                            uint32_t o[8];
                            __syncwarp();
                            if (fresh) {
#pragma unroll
                                for (int i = 0; i < 8; ++i) o[i] = 0;
                            } else {
                                tc05::ld8(otm + k, o);
                                tc05::wait_ld_regs(o);
                            }
#pragma unroll 1
                            for (int key = 0; key < BK; key += 8) {
                                const int half = key >> 6;
                                uint32_t v[4];
                                __syncwarp();
                                tc05::ld4(lanes + (w ? (half ? L::p_col(1, 1) : L::p_col(1, 0)) : (half ? L::p_col(0, 1) : L::p_col(0, 0))) + (key & 63) / 2, v);
                                tc05::wait_ld_regs(v);
                                const uint8_t *at_slot = ring + (vf + key / SLOT) % STAGES * L::SLOT_BYTES + (k >> 6) * (SLOT * 128) +
                                                         key % SLOT * 128;
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float2 p2 = unpack(v[i / 2], T());
                                    const float wt = i & 1 ? p2.y : p2.x;
                                    const uint4 u = *(const uint4 *)(at_slot + i * 128 + ((((k & 63) >> 3) ^ i) << 4));
                                    const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
                                    if (key + i < most)
#pragma unroll
                                        for (int e = 0; e < 4; ++e) {
                                            const float2 y = unpack(uu[e], T());
                                            o[e * 2] = __float_as_uint(fmaf(wt, y.x, __uint_as_float(o[e * 2])));
                                            o[e * 2 + 1] = __float_as_uint(fmaf(wt, y.y, __uint_as_float(o[e * 2 + 1])));
                                        }
                                }
                            }
                            __syncwarp();
                            st8(otm + k, o);
                        }
                        tc05::wait_st();
                    }
                    fresh = false;
                    ++un;
                    tc05::fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(&pready[w]);
                }
                if (!ok) break;
                // The row tile's sums are done; the row's weights over both halves, and, where the tiles had the even and the
                // odd steps of the same rows, over both tiles.
                const bool some = alt ? n > w : true;
                if (some) {
                    ok = __all_sync(~0u, wait_or_stop(&odone[w], (un - 1) & 1, stop));
                    if (!ok) break;
                }
                auto everyone = [&]() { return alt ? meet(both, bn) : meet(&tbar[w], tn); };
                told[wg * 128 + row] = l;
                tc05::fence_before();
                ok = everyone();
                if (!ok) break;
                tc05::fence_after();
                l += told[(wg ^ 1) * 128 + row];
                float mine = 1.f, its = 0.f;  // what the sums of this row tile, and of the other, are multiplied by
                if (alt) {
                    const float other = told[(wg ^ 2) * 128 + row] + told[(wg ^ 3) * 128 + row];
                    ok = meet(both, bn);
                    if (!ok) break;
                    told[wg * 128 + row] = m;
                    ok = meet(both, bn);
                    if (!ok) break;
                    const float M = fmaxf(m, told[(wg ^ 2) * 128 + row]);
                    mine = exp2_(m - M), its = exp2_(told[(wg ^ 2) * 128 + row] - M);
                    l = l * mine + other * its;
                    m = M;
                }
                const bool two_tiles = alt && n > 1, other_alone = alt && !some;
                constexpr int QUARTER = D / 4;
                const int col0 = alt ? wg * QUARTER : h * (D / 2), col1 = col0 + (alt ? QUARTER : D / 2);  // this warpgroup's
                const uint32_t its_otm = lanes + (w ? L::o_col(0) : L::o_col(1));
                auto columns = [&](int col, float (&v)[8]) {
                    uint32_t o[8];
                    __syncwarp();  // rows that do not exist store nothing: the warp's lanes meet again
                    tc05::ld8(other_alone ? its_otm + col : otm + col, o);
                    tc05::wait_ld_regs(o);
                    const float f = other_alone ? its : mine;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(o[i]) * f;
                    if (two_tiles) {
                        tc05::ld8(its_otm + col, o);
                        tc05::wait_ld_regs(o);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = fmaf(__uint_as_float(o[i]), its, v[i]);
                    }
                };
                T *out = (T *)a.out;
                float *lse = a.lse;
                if (exists) {
                    const long long tk = seg.seq.s0 + tok;
                    const int hd = seg.h * a.group + at - tok * a.group;
                    out += tk * a.o_tok + hd * a.o_head;
                    if (lse) lse += tk * a.lse_tok + hd * a.lse_head;
                }
                const int c_first = seg.first_share(share), c_last = seg.last_share(share);
                if (c_first == c_last) {
                    const float inv = row_factor(seen, l);
#pragma unroll 1
                    for (int col = col0; col < col1; col += 8) {
                        float v[8];
                        columns(col, v);
                        alignas(16) T e[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(seen > 0 ? v[i] * inv : 0.f);
                        if (!exists) continue;
                        if (a.o_vec) {
                            *(uint4 *)(out + col) = *(const uint4 *)e;
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) out[col + i] = e[i];
                        }
                    }
                    if (exists && lse && col0 == 0) *lse = row_lse(seen, m, l);
                } else {
                    // A share leaves its second slot to the item that starts in it, its first to one that started before.
                    auto slot = [&](int k) { return 2ll * k + (k == c_first); };
                    const int tile0 = alt ? 0 : w * 128;  // rows of this warpgroup
                    float4 *po = (float4 *)a.parts;       // a slot: [D / 4][R]
                    float2 *pst = (float2 *)(a.parts + 2ll * gridDim.x * L::PART) + wg * 128;  // a slot: [4][128]
                    const long long own = slot(blockIdx.x);
#pragma unroll 1
                    for (int col = col0; col < col1; col += 8) {
                        float v[8];
                        columns(col, v);
                        if (exists)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                __stcg(po + own * (L::PART / 4) + (long long)(col / 4 + i) * R + tile0 + row,
                                       make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
                    }
                    if (exists) __stcg(pst + own * 512 + row, make_float2(m, l));
                    const int k_parts = c_last - c_first + 1;
                    ok = meet(&gbar[wg], gn);
                    if (!ok) break;
                    if (row == 0) {
                        __threadfence();
                        last_flag[wg] = atomicInc(a.counts + wg * MAX_GRID + c_first, k_parts - 1) == (uint32_t)k_parts - 1;
                        __threadfence();
                    }
                    counted = true;
                    ok = meet(&gbar[wg], gn);
                    if (!ok) break;
                    if (last_flag[wg]) {
                        // a row's maximum and sum over the parts; then each part's weight in the place of its maximum
                        if (exists) {
                            float M = LOWEST, S = 0.f;
#pragma unroll 4
                            for (int k = 0; k < k_parts; ++k) M = fmaxf(M, __ldcg(pst + slot(c_first + k) * 512 + row).x);
#pragma unroll 4
                            for (int k = 0; k < k_parts; ++k) {
                                const float2 v = __ldcg(pst + slot(c_first + k) * 512 + row);
                                S += exp2_(v.x - M) * v.y;
                            }
                            const float inv = row_factor(seen, S);
#pragma unroll 1
                            for (int k = 0; k < k_parts; ++k) {
                                float2 *p = pst + slot(c_first + k) * 512 + row;
                                __stcg(p, make_float2(seen > 0 ? exp2_(__ldcg(p).x - M) : 0.f, inv));
                            }
                            if (lse && col0 == 0) *lse = row_lse(seen, M, S);
                        }
                        __threadfence_block();
                        ok = meet(&gbar[wg], gn);
                        if (!ok) break;
                        const int nr = min(128, rows - tile0), n4 = nr * (col1 - col0) / 4;
#pragma unroll 1
                        for (int i = row; i < n4; i += 128) {
                            const int rr = i % nr, c4 = col0 / 4 + i / nr;
                            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                            float inv = 0.f;
#pragma unroll 4
                            for (int k = 0; k < k_parts; ++k) {
                                const long long sl = slot(c_first + k);
                                const float2 wv = __ldcg(pst + sl * 512 + rr);
                                const float4 v = __ldcg(po + sl * (L::PART / 4) + (long long)c4 * R + tile0 + rr);
                                inv = wv.y;
                                acc.x = fmaf(wv.x, v.x, acc.x), acc.y = fmaf(wv.x, v.y, acc.y);
                                acc.z = fmaf(wv.x, v.z, acc.z), acc.w = fmaf(wv.x, v.w, acc.w);
                            }
                            const int at2 = (int)((long long)seg.qt * R + tile0 + rr), tk = at2 / a.group;
                            T *o = (T *)a.out + (seg.seq.s0 + (long long)tk) * a.o_tok +
                                   (seg.h * a.group + at2 - tk * a.group) * a.o_head + c4 * 4;
                            const bool sees = seg.seq.seen(a, tk) > 0;
                            alignas(8) T e[4] = {from_f32<T>(sees ? acc.x * inv : 0.f), from_f32<T>(sees ? acc.y * inv : 0.f),
                                                 from_f32<T>(sees ? acc.z * inv : 0.f), from_f32<T>(sees ? acc.w * inv : 0.f)};
                            if (a.o_vec) {
                                *(uint2 *)o = *(const uint2 *)e;
                            } else {
#pragma unroll
                                for (int q = 0; q < 4; ++q) o[q] = e[q];
                            }
                        }
                    }
                }
                // What the others have of this warpgroup (in `told`, and its sums) has been read.
                tc05::fence_before();
                ok = everyone();
                if (!ok) break;
                tc05::fence_after();
                base += 2 * n * PARTS;
                if (!seg.next(a)) break;
            } while (true);
        if (!ok && works && row == 0) {
            // Gave up: the counters of the cut items of this share are counted on, so that they end at zero.
            do {
                const int c_first = seg.first_share(share), c_last = seg.last_share(share);
                if (c_first != c_last && !counted) atomicInc(a.counts + wg * MAX_GRID + c_first, c_last - c_first);
                counted = false;
            } while (seg.next(a));
        }
        tc05::fence_before();
    }
    __syncwarp();
    __syncthreads();
    if (tid == 0 && *stop) atomicOr(a.err, HV_DECODE_STALLED);  // every role has been through
    if (warp == L::MMA_WARP) {
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

// A cache in boxes of `rows` slots x 64 dimensions of one head of a page; false where its strides do not allow that.
template <typename T, int D>
bool tensor_map(CUtensorMap *map, const void *base, const ChunkArgs &a, long long page, long long slot, long long head, int rows) {
    const PFN_cuTensorMapEncodeTiled encode = encoder();
    if (!encode || !base || !a.num_pages) return false;
    const cuuint64_t dims[4] = {D, (cuuint64_t)a.page, (cuuint64_t)a.kv_heads, (cuuint64_t)a.num_pages};
    const long long strides[3] = {slot, head, page};
    cuuint64_t bytes[3];
    for (int i = 0; i < 3; ++i) {
        if (dims[i + 1] > 1 && (strides[i] < D || strides[i] >= 1ll << 38)) return false;
        bytes[i] = dims[i + 1] > 1 ? (cuuint64_t)strides[i] * 2 : 512;
    }
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 4, const_cast<void *>(base), dims, bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q in boxes of the heads of a group x as many tokens as make 128 rows; false where they do not.
template <typename T, int D>
bool q_map(CUtensorMap *map, const ChunkArgs &a) {
    const PFN_cuTensorMapEncodeTiled encode = encoder();
    if (!encode || a.group > 128 || 128 % a.group) return false;
    const cuuint64_t dims[3] = {D, (cuuint64_t)a.heads, (cuuint64_t)a.tokens};
    const long long strides[2] = {a.q_head, a.q_tok};
    cuuint64_t bytes[2];
    for (int i = 0; i < 2; ++i) {
        if (dims[i + 1] > 1 && (strides[i] < D || strides[i] >= 1ll << 38)) return false;
        bytes[i] = dims[i + 1] > 1 ? (cuuint64_t)strides[i] * 2 : 512;
    }
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(128 / a.group)}, estr[3] = {1, 1, 1};
    const CUtensorMapDataType type =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode(map, type, 3, const_cast<void *>(a.q), dims, bytes, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch(ChunkArgs a, int grid, cudaStream_t st) {
    using L = Lay<D>;
    // Pages of a multiple of eight tokens come by TMA, in boxes of as many as a page and a copying warp's rows share.
    CUtensorMap tmk = {}, tmv = {};
    for (a.box = L::SLOT / 4; a.page % a.box; a.box /= 2) {}
    if (a.box < 8 || !tensor_map<T, D>(&tmk, a.kc, a, a.kc_page, a.kc_slot, a.kc_head, a.box) ||
        !tensor_map<T, D>(&tmv, a.vc, a, a.vc_page, a.vc_slot, a.vc_head, a.box))
        a.box = 0;
    CUtensorMap tmq = {};
    a.q_box = a.q_vec && q_map<T, D>(&tmq, a);
    static std::atomic<uint64_t> ready;
    static std::atomic<int> regs;
    cudaError_t e = allow_shared(chunk_kernel<T, D>, ready);
    if (e != cudaSuccess) return e;
    if (!regs.load(std::memory_order_relaxed)) {  // what the warps' shares are taken from
        cudaFuncAttributes f;
        e = cudaFuncGetAttributes(&f, chunk_kernel<T, D>);
        if (e != cudaSuccess) return e;
        if (f.numRegs != L::REGS) return cudaErrorInvalidConfiguration;
        regs.store(f.numRegs, std::memory_order_relaxed);
    }
    return launch_pdl(chunk_kernel<T, D>, dim3((unsigned)grid), dim3(L::THREADS), L::BYTES, st, a, tmk, tmv, tmq);
}

template <typename T>
cudaError_t by_dim(const ChunkArgs &a, int dim, int grid, cudaStream_t st) {
    switch (dim) {
        case 32: return launch<T, 32>(a, grid, st);
        case 64: return launch<T, 64>(a, grid, st);
        case 96: return launch<T, 96>(a, grid, st);
        case 128: return launch<T, 128>(a, grid, st);
        case 192: return launch<T, 192>(a, grid, st);
        default: return launch<T, 256>(a, grid, st);
    }
}

bool known_dim(int d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

int wave() {
    const int sms = sm_count();
    return sms < MAX_GRID ? sms : MAX_GRID;
}

static_assert(4 * MAX_GRID * 4 <= HV_ATTENTION_COUNTER_BYTES, "the counters that the caller zeroes");
static_assert(HV_ATTENTION_MAX_LENGTH + (long long)BK <= INT32_MAX, "token numbers of a last step are ints");

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_paged_chunk_attention_workspace(int dim, int64_t *bytes) {
    if (!bytes) return fail(HV_ERR_VALUE, "null argument");
    if (!known_dim(dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    const int grid = wave(), rows = dim <= 128 ? 256 : 128;
    if (!grid) return fail(HV_ERR_CUDA, "cannot read the device's SM count");
    *bytes = HV_ATTENTION_COUNTER_BYTES + 2ll * grid * (rows * dim + 1024) * 4;
    return HV_OK;
}

extern "C" int hv_paged_chunk_attention(const hv_chunk_args *p, void *stream) {
    if (!p) return fail(HV_ERR_VALUE, "null argument");
    if (p->dtype != HV_BF16 && p->dtype != HV_F16) return fail(HV_ERR_TYPE, "dtype must be HV_BF16 or HV_F16");
    if (p->tokens < 0 || p->seqs < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads)
        return fail(HV_ERR_VALUE, "heads must be a positive multiple of kv_heads");
    if (!known_dim(p->dim)) return fail(HV_ERR_VALUE, "dim must be 32, 64, 96, 128, 192 or 256");
    if (p->page_size < 1 || p->num_pages < 0 || p->max_pages < 0) return fail(HV_ERR_VALUE, "bad cache geometry");
    if ((double)p->tokens * (p->heads / p->kv_heads) > HV_ATTENTION_MAX_LENGTH)
        return fail(HV_ERR_VALUE, "too many rows for one call");
    if (p->seqs == 0 || p->tokens == 0) return HV_OK;
    if (!p->d_q || !p->d_out || !p->d_lens || !p->d_starts || (p->max_pages && !p->d_page_table) ||
        (p->num_pages && (!p->d_k_cache || !p->d_v_cache)))
        return fail(HV_ERR_VALUE, "null buffer");
    int64_t need = 0;
    const int rc = hv_paged_chunk_attention_workspace(p->dim, &need);
    if (rc) return rc;
    if (!p->d_workspace || p->workspace_bytes < need)
        return fail(HV_ERR_VALUE, "the workspace has %lld bytes of %lld", (long long)p->workspace_bytes, (long long)need);
    if (!dec::aligned(p->d_workspace, 256)) return fail(HV_ERR_VALUE, "the workspace must be 256-byte aligned");
    bool ok = dec::aligned(p->d_k_cache, 16) && dec::aligned(p->d_v_cache, 16);
    for (int i = 0; i < 3; ++i) ok = ok && p->k_cache_strides[i] % 8 == 0 && p->v_cache_strides[i] % 8 == 0;
    if (!ok) return fail(HV_ERR_VALUE, "cache rows must start on 16 bytes");
    int *err = dec::error_word();
    if (!err) return fail(HV_ERR_CUDA, "cannot resolve the device error word");
    ChunkArgs a{};
    a.q = p->d_q, a.kc = p->d_k_cache, a.vc = p->d_v_cache, a.out = p->d_out, a.lse = p->d_lse;
    a.pages = p->d_page_table, a.lens = p->d_lens, a.starts = p->d_starts;
    a.q_tok = p->q_strides[0], a.q_head = p->q_strides[1], a.o_tok = p->out_strides[0], a.o_head = p->out_strides[1];
    a.lse_tok = p->lse_strides[0], a.lse_head = p->lse_strides[1];
    a.kc_page = p->k_cache_strides[0], a.kc_slot = p->k_cache_strides[1], a.kc_head = p->k_cache_strides[2];
    a.vc_page = p->v_cache_strides[0], a.vc_slot = p->v_cache_strides[1], a.vc_head = p->v_cache_strides[2];
    a.pages_stride = p->page_table_stride;
    a.tokens = p->tokens, a.seqs = p->seqs, a.heads = p->heads, a.kv_heads = p->kv_heads, a.group = p->heads / p->kv_heads;
    a.num_pages = p->num_pages, a.page = p->page_size, a.max_pages = p->max_pages, a.causal = p->causal;
    a.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
    a.q_vec = dec::aligned(a.q, 16) && a.q_tok % 8 == 0 && a.q_head % 8 == 0;
    a.o_vec = dec::aligned(a.out, 16) && a.o_tok % 8 == 0 && a.o_head % 8 == 0;
    // A score is taken times a scale above zero, with q negated for one below, so that the largest stays the
    // largest and -inf that; for zero the least normal number gives the weights of 0.  A NaN stays one.
    a.tp_shift = -1;
    for (int i = 0, rows = p->dim <= 128 ? 256 : 128; rows >> i; ++i)
        if (rows >> i == rows / a.group && rows % a.group == 0) a.tp_shift = __builtin_ctz(rows / a.group);
    a.negate = p->scale < 0;
    a.scale_log2 = fabsf(p->scale) * 1.4426950408889634f;
    if (a.scale_log2 < FLT_MIN) a.scale_log2 = FLT_MIN;
    a.skip = dec::skipped_copy();
    a.counts = (uint32_t *)p->d_workspace;
    a.parts = (float *)((char *)p->d_workspace + HV_ATTENTION_COUNTER_BYTES);
    a.err = err;
    const int grid = wave();
    const cudaError_t e = p->dtype == HV_BF16 ? by_dim<__nv_bfloat16>(a, p->dim, grid, (cudaStream_t)stream)
                                              : by_dim<__half>(a, p->dim, grid, (cudaStream_t)stream);
    if (e != cudaSuccess) return fail(HV_ERR_CUDA, "paged_chunk_attention: %s", cudaGetErrorString(e));
    return HV_OK;
}
