// prompt_attn.hip -- attention of packed prompts: every sequence's queries over
// its own keys, causal or not, grouped heads, one pass with a running maximum
// and sum.
//
// out_i = sum_{j <= i + Lk - Lq} softmax_j(scale <q_i, k_j>) v_j  (all j < Lk
// without the mask); a row that sees no key is 0.
//
// Both products are computed transposed, so that nothing crosses lanes between
// them.  S^T = K Q^T on 32x32 tiles: lane (q = lane % 32, h = lane / 32) ends
// with the scores of its query row against keys 8 (r / 4) + 4 h + r % 4, r < 16.
// O^T = V^T P^T takes P^T as the operand whose lane holds one query row and any
// keys of its half, as long as V^T's lanes hold the same ones: the softmax's
// results go in as they are, V is read from LDS in that key order.  Maxima and
// sums are a query row's, a lane's own: one exchange between the halves per
// tile.
//
// A workgroup's four waves (two pairs where a tile's keys are split) take HW query
// heads of one kv head, the largest power of two up to four (two) that divides the
// heads per kv head, by 4 / HW (2 / HW) blocks of 32 rows: K and V are staged once
// for all of them, and with four heads the causal diagonal cuts through 32 rows
// instead of 128.
//
// Bound by the matrix instructions where rows are long, and by exponentials with
// narrow heads: a score costs 4 D operations there and one exp2 at a quarter of the
// vector rate, about as long as its products at D = 64.  Measured, one pass, causal,
// 32 / 8 heads of 128 but where said: 16384 bf16 tokens of one sequence 2.10 to 2.34
// ms by the card's clock, 940 to 1050 TFLOP/s (a large bf16 matrix product of the
// library runs at 1200); 8192 of eight 0.11 to 0.12 ms, 0.155 with 16 / 8 heads of 256;
// 4999 fp16 tokens of five sequences, 16 heads of 64, 30 us; 2048 fp32 of two 130 to 140
// us, 412 with 16 / 8 heads of 256; 150 bf16 of three 7.6 us, of which a launch with
// nothing to do is half.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace ojx {

namespace {
constexpr int kKeys = 64;                        // keys per tile
constexpr int kFlags = 16;                       // bytes of LDS behind the tiles: an int per wave
// Workgroups up to which half as many rows go to each and the keys of a tile to two
// waves: as many as are resident at once (three, two or one to a CU by head dim).
// Below it the longest rows' way through their keys sets the time (1500 tokens of
// 8 / 2 heads of 128: 98 workgroups, 35.0 -> 26.8 us; 3000 of 16 of 64: 416, 43.9 ->
// 36.0), above it the splits' own cost (2048 tokens of 32 / 8 heads of 128: 536, 54.4
// -> 57.7; 4096 of 16 / 2 of 256: 524, 190 -> 284).
constexpr long split_below(int DP) { return 256 * (DP <= 64 ? 3 : DP <= 128 ? 2 : 1); }
// A weight is 2^(score scale - max), the product not rounded.  From 2^24 on the maximum
// is rounded by more than 1, and a weight could pass its type's range, or all of them
// be 0: scores past this are rounded as their maximum is (rounded_score).
constexpr float kFar = 0x1p20f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct PromptParams {
    const void *q, *k, *v;
    long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;     // token and head strides, elements
    void *out;                                   // [Nq][Hq][D]
    float *lse;                                  // [Nq][Hq] or null
    const int *cu_q, *cu_k;                      // [B + 1]
    int B, Nq, Nk, Hq, Hkv, D;
    int hw, causal, zero_rest;                   // log2 of the heads per workgroup
    float scale2;                                // scale x log2(e)
};

struct Bf16 {
    typedef __hip_bfloat16 T;
    typedef bf16x8_t V8;
    static constexpr int kInf = 0x7f80;          // an infinity's bits
    static constexpr float kBias = 0.f;
    static __device__ __forceinline__ f32x16_t mma(V8 a, V8 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ __bf16 from(float f) { return (__bf16)f; }
};
struct F16 {
    typedef __half T;
    typedef f16x8_t V8;
    static constexpr int kInf = 0x7c00;
    // Weights times 2^7: the largest, 2^8 above 1 (raise_max), still fit, and those
    // that fp16's subnormals round to 0 are below 2^-32, not 2^-25, of a row's largest
    static constexpr float kBias = 7.f;
    static __device__ __forceinline__ f32x16_t mma(V8 a, V8 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ _Float16 from(float f) { return (_Float16)f; }
};

// Entry b of cumulative lengths, clamped to the n rows there are, whatever it holds.
__device__ __forceinline__ int cu_at(const int *cu, int b, int n) { return min(max(cu[b], 0), n); }

// 16-byte unit `u` of row `row` in a K tile, and 32-byte unit of a V tile: XOR
// swizzles under which the 16 rows of a K read, and the 8 rows of a transposed V
// read, spread over all the banks.
template <int ROWB>
__device__ __forceinline__ int k_unit(int row, int u) {
    return ROWB >= 256 ? u ^ (row & 15) : u ^ (row >> 1 & 7);
}
template <int ROWB>
__device__ __forceinline__ int v_unit(int row, int u) {
    return ROWB >= 256 ? u ^ (row & 7) : u ^ (row >> 1 & 3);
}

// max and sum of a lane's value and the other half's: v_permlane32_swap of a register
// with itself leaves the low half's in the first result, the high half's in the second.
__device__ __forceinline__ float halves_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Waits for the loads so far.  Without it before a loop the compiler waits inside
// it, for the loop's own loads too, before the first use of what was loaded
// before it.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0) alone

// The key that accumulator register r of a lane's half h stands for.
__device__ __forceinline__ constexpr int key_of(int r) { return 8 * (r / 4) + r % 4; }

// a *= f in accumulation registers.  Written as a product the compiler copies all of
// the kernel's accumulators to vector registers and back on every tile, also where
// none is rescaled.  The waits that it would put between matrix instructions and these
// reads and writes stand in the block: 24 states before (the longest needs 19), 4 after.
__device__ __forceinline__ void scale_acc(f32x16_t &a, float f) {
    float e[16], t;
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = a[i];
    asm volatile(
        "s_nop 15\n\ts_nop 7\n\t"
        "v_accvgpr_read_b32 %16, %0\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %0, %16\n\t"
        "v_accvgpr_read_b32 %16, %1\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %1, %16\n\t"
        "v_accvgpr_read_b32 %16, %2\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %2, %16\n\t"
        "v_accvgpr_read_b32 %16, %3\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %3, %16\n\t"
        "v_accvgpr_read_b32 %16, %4\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %4, %16\n\t"
        "v_accvgpr_read_b32 %16, %5\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %5, %16\n\t"
        "v_accvgpr_read_b32 %16, %6\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %6, %16\n\t"
        "v_accvgpr_read_b32 %16, %7\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %7, %16\n\t"
        "v_accvgpr_read_b32 %16, %8\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %8, %16\n\t"
        "v_accvgpr_read_b32 %16, %9\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %9, %16\n\t"
        "v_accvgpr_read_b32 %16, %10\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %10, %16\n\t"
        "v_accvgpr_read_b32 %16, %11\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %11, %16\n\t"
        "v_accvgpr_read_b32 %16, %12\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %12, %16\n\t"
        "v_accvgpr_read_b32 %16, %13\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %13, %16\n\t"
        "v_accvgpr_read_b32 %16, %14\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %14, %16\n\t"
        "v_accvgpr_read_b32 %16, %15\n\tv_mul_f32 %16, %16, %17\n\tv_accvgpr_write_b32 %15, %16\n\t"
        "s_nop 3"
        : "+a"(e[0]), "+a"(e[1]), "+a"(e[2]), "+a"(e[3]), "+a"(e[4]), "+a"(e[5]), "+a"(e[6]), "+a"(e[7]), "+a"(e[8]), "+a"(e[9]), "+a"(e[10]), "+a"(e[11]), "+a"(e[12]), "+a"(e[13]), "+a"(e[14]), "+a"(e[15]), "=&v"(t)
        : "v"(f));
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = e[i];
}

// Running maximum (log2) of one query row per lane with a tile's largest score t:
// rescales acc and l where the row's maximum grew by more than 2^8.
// Weights up to 2^8 above 1 lose nothing: they are rounded relative to their
// size and all sums are fp32.  A weight is 2^(score - ref), ref = m - bias.
//
// ACC: acc stays in accumulation registers.
template <bool ACC, int NT>
__device__ __forceinline__ void raise_max(float t, float bias, float &m, float &ref, float &l, f32x16_t (&acc)[NT]) {
    if (__any(t > m + 8.f)) {
        const float mn = fmaxf(m, t), rn = (mn == -INFINITY ? 0.f : mn) - bias;
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - rn);
        m = mn;
        ref = rn;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (ACC) scale_acc(acc[i], alpha);
            else acc[i] *= alpha;
    }
}

// A score as the maximum holds it: the product rounded before anything is subtracted.
__device__ __forceinline__ float rounded_score(float s, float scale2) {
    float x = s * scale2;
    asm volatile("" : "+v"(x));
    return x;
}

// The thread's number, for AGAIN hidden from the compiler: what it computes from it
// anew would else stay in registers all through the first time.
template <bool AGAIN>
__device__ __forceinline__ int own_thread() {
    int t = threadIdx.x;
    if (AGAIN) asm volatile("" : "+v"(t));
    return t;
}

enum { kDone, kOthersAgain, kAgain };

// The kernel's first argument, read once more, for the same reason (16-bit kernels of
// 65 to 128 dims: 29 scalar registers spilled without, 6 with; 8192 tokens of eight
// sequences, head_dim 80: 104.5 -> 100.8 us).
__device__ __forceinline__ PromptParams own_params() {
    typedef __attribute__((address_space(4))) const uint32_t word_t;
    word_t *a = (word_t *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    uint32_t w[sizeof(PromptParams) / 4];
#pragma unroll
    for (unsigned i = 0; i < sizeof(PromptParams) / 4; ++i) w[i] = a[i];
    PromptParams p;
    __builtin_memcpy(&p, w, sizeof(p));
    return p;
}

// Whether a wave of the workgroup has `mine` set.  flags: an int of LDS per wave.
__device__ __forceinline__ bool any_wave(int *flags, bool mine) {
    const bool wave = __any(mine);
    if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = wave;
    __syncthreads();
    return flags[0] | flags[1] | flags[2] | flags[3];
}

// Exact pieces as split3_bf16 makes them, of any value: one that rounds past bf16's
// range is cut to eight bits first, an infinity or NaN is the third piece alone.  That
// piece takes part in one product, with the other operand's first piece, which has its
// sign and is 0 only with it: the product is what the two values' own would be.
__device__ __forceinline__ void split3_any(const float (&v)[8], bf16x8_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(v[i]), a = u & 0x7fffffffu;
        const float f = a < 0x7f800000u ? v[i] : 0.f;
        const __bf16 h1 = (__bf16)(a < 0x7f7f8000u ? f : __uint_as_float(u & 0xffff0000u));
        const float r1 = f - (float)h1;
        const __bf16 h2 = (__bf16)r1;
        p[0][i] = a < 0x7f800000u ? h1 : (__bf16)0.f;
        p[1][i] = a < 0x7f800000u ? h2 : (__bf16)0.f;
        p[2][i] = a < 0x7f800000u ? (__bf16)(r1 - (float)h2) : (__bf16)v[i];
    }
}

// The infinities and NaN of a V operand, taken out of it: 1 for +inf, 2^7 for -inf,
// 2^14 for NaN in their places, which a product with ones for the keys that a row sees
// counts exactly (at most 64 keys), and what the counts add to an output.
template <typename E>
__device__ __forceinline__ typename E::V8 take_marks(typename E::V8 &v) {
    typedef short s16x8_t __attribute__((ext_vector_type(8)));
    s16x8_t z = __builtin_bit_cast(s16x8_t, v);
    typename E::V8 m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int a = z[i] & 0x7fff;
        m[i] = E::from(a < E::kInf ? 0.f : a > E::kInf ? 0x1p14f : z[i] < 0 ? 0x1p7f : 1.f);
        if (a >= E::kInf) z[i] = 0;
    }
    v = __builtin_bit_cast(typename E::V8, z);
    return m;
}
// Bit 15 or 31 of the result is set where one of v's values is an infinity or NaN.
template <typename E>
__device__ __forceinline__ uint32_t has_marks(const typename E::V8 &v) {
    constexpr uint32_t inf = E::kInf * 0x10001u, one = (0x8000u - E::kInf) * 0x10001u;
    const u32x4_t w = __builtin_bit_cast(u32x4_t, v);
    uint32_t x = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) x |= (w[i] & inf) + one;
    return x;
}
__device__ __forceinline__ float from_marks(float counts) {
    const int c = (int)counts;
    const float up = (c & 127) ? INFINITY : 0.f, down = (c >> 7 & 127) ? -INFINITY : 0.f;
    return c >> 14 ? NAN : up + down;
}

// Hides the keys past `lim` from the lane's row; k0 = the tile's first key.
template <int NB>
__device__ __forceinline__ void mask_tile(f32x16_t (&s)[NB], int lim, int k0, int h) {
    int rel = lim - k0 - 4 * h;
    asm volatile("" : "+v"(rel));                // keeps the selects behind the wave's branch
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        if (key_of(r) > rel) s[0][r] = -INFINITY;
        if (NB > 1 && 32 + key_of(r) > rel) s[NB - 1][r] = -INFINITY;
    }
}

// Ones for the keys of operand f (as the weights lie in it) that come before `rel` or at
// it, counted from the lane's first.
template <typename E>
__device__ __forceinline__ typename E::V8 seen_keys(int f, int rel) {
    typename E::V8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = E::from(32 * (f >> 1) + key_of(8 * (f & 1) + e) <= rel ? 1.f : 0.f);
    return x;
}
}  // namespace

// The rows and keys of a workgroup.
struct PromptBlock {
    int b, first, len, tile;     // sequence (-1 or B: rows of none), its rows, the tile in it
    int head0, k_first, Lk;
};

// Workgroups: slots x head groups, the head group fastest: consecutive
// workgroups go to different XCDs, so with 8 head groups (or a multiple) an XCD
// keeps the K and V of its own heads; the last rows of the batch, the longest
// tiles of a single causal sequence, start first.
// Sequence b takes the slots from s(b) = cu[b] / BM + b + 1 (its rows need at most
// the next sequence's slots less one), rows before the first sequence the slots
// from 0 and rows behind the last one those from s(B).
__device__ __forceinline__ bool prompt_block(const PromptParams &p, int slots, int bm_shift, PromptBlock &o) {
    const int hg = p.Hq >> p.hw, lane = threadIdx.x & 63;
    const int t = slots - 1 - (int)blockIdx.x / hg;
    o.head0 = (int)blockIdx.x % hg << p.hw;
    o.k_first = 0;
    int next, k_next = 0;
    if (p.B < 64) {              // both lists in one load each, the entries by lane
        const int i = min(lane, p.B), cq = cu_at(p.cu_q, i, p.Nq), ck = cu_at(p.cu_k, i, p.Nk);
        o.b = __popcll(__ballot(lane <= p.B && (cq >> bm_shift) + lane + 1 <= t)) - 1;
        o.first = o.b < 0 ? 0 : __builtin_amdgcn_readlane(cq, max(o.b, 0));
        next = o.b < p.B ? __builtin_amdgcn_readlane(cq, o.b + 1) : p.Nq;
        if (o.b >= 0 && o.b < p.B) {
            o.k_first = __builtin_amdgcn_readlane(ck, max(o.b, 0));
            k_next = __builtin_amdgcn_readlane(ck, o.b + 1);
        }
    } else {
        int count = 0;
        for (int i0 = 0; i0 <= p.B; i0 += 64) {
            const int i = min(i0 + lane, p.B);
            count += __popcll(__ballot(i0 + lane <= p.B && (cu_at(p.cu_q, i, p.Nq) >> bm_shift) + i + 1 <= t));
        }
        o.b = count - 1;
        o.first = o.b < 0 ? 0 : cu_at(p.cu_q, o.b, p.Nq);
        next = o.b < p.B ? cu_at(p.cu_q, o.b + 1, p.Nq) : p.Nq;
        if (o.b >= 0 && o.b < p.B) {
            o.k_first = cu_at(p.cu_k, o.b, p.Nk);
            k_next = cu_at(p.cu_k, o.b + 1, p.Nk);
        }
        next = __builtin_amdgcn_readfirstlane(next);
        k_next = __builtin_amdgcn_readfirstlane(k_next);
        o.first = __builtin_amdgcn_readfirstlane(o.first);
        o.k_first = __builtin_amdgcn_readfirstlane(o.k_first);
    }
    o.len = next - o.first;
    o.tile = t - (o.b < 0 ? 0 : (o.first >> bm_shift) + o.b + 1);
    o.Lk = max(k_next - o.k_first, 0);
    return o.tile >= 0 && (long)o.tile << bm_shift < o.len;   // whatever cu holds
}

// Rows of no sequence: zeros, where the caller wants them written.
template <typename T>
__device__ __forceinline__ void zero_rows(const PromptParams &p, const PromptBlock &o, int bm_shift) {
    if (!p.zero_rest) return;
    const int r0 = o.tile << bm_shift, n = min(1 << bm_shift, o.len - r0);
    const int heads = 1 << p.hw, per = heads * p.D;
    for (int x = threadIdx.x; x < n * per; x += blockDim.x) {
        const size_t row = (size_t)(o.first + r0 + x / per) * p.Hq + o.head0 + x % per / p.D;
        store_act(static_cast<T *>(p.out), row * p.D + x % p.D, 0.f);
        if (p.lse && x % p.D == 0) p.lse[row] = -INFINITY;
    }
}

// bf16 and fp16: v_mfma_f32_32x32x16, head dims up to DP (the dims past D are
// zeros in Q and K).  KS = 2: half the waves take the first 32 keys of every tile,
// the other half the last 32, and the pairs join their sums in LDS: twice the
// workgroups with half the work in a row, for grids too small to hide how long
// their longest rows take.
//
// AGAIN: with scores rounded as their maximum is, and V's infinities and NaN taken out
// of the product.  Returns what is left to do again: kAgain where the wave's rows are
// not written yet, kOthersAgain where other waves' are not.  mine: the wave's rows are
// to be written (the others of AGAIN help with the tiles).
template <typename E, int DP, int KS, bool AGAIN>
__device__ __forceinline__ int prompt_block_attn(const PromptParams &p, int slots, bool mine) {
    typedef typename E::T T;
    typedef typename E::V8 V8;
    constexpr int NW = 4, WR = NW / KS, NB = 2 / KS;  // waves of different rows, 32-key blocks of a wave
    constexpr int NT = 64 * NW, ROWB = 2 * DP, UPR = DP / 8, TILE = kKeys * ROWB;
    constexpr int CH = kKeys * UPR / NT;             // 16-byte units of a tile per thread
    extern __shared__ __align__(16) unsigned char sm[];   // [2 buffers][K tile, V tile], flags
    const int tid = own_thread<AGAIN>(), lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int wr = w % WR, kb = KS == 1 ? 0 : 32 * (w / WR);    // the wave's keys begin at kb
    const int bm_shift = 5 + __builtin_ctz(WR) - p.hw;
    PromptBlock o;
    if (!prompt_block(p, slots, bm_shift, o)) return kDone;
    if (o.b < 0 || o.b >= p.B) {
        zero_rows<T>(p, o, bm_shift);
        return kDone;
    }
    const int head = o.head0 + (wr & ((1 << p.hw) - 1)), kvh = o.head0 / (p.Hq / p.Hkv);
    const int Lq = o.len, Lk = o.Lk, off = Lk - Lq;
    const int tile0 = o.tile << bm_shift;                  // the workgroup's first row
    const int row0 = tile0 + 32 * (wr >> p.hw), row = row0 + n;  // the wave's, the lane's
    const int qrow = min(row, Lq - 1);
    const int lim = p.causal ? min(Lk - 1, qrow + off) : Lk - 1;       // last key the row sees
    const int lim_lo = p.causal ? min(Lk - 1, row0 + off) : Lk - 1;    // the wave's least,
    const int lim_hi = !mine || row0 >= Lq ? -1      // and most; none where the wave has no row
                       : p.causal          ? min(Lk - 1, min(row0 + 31, Lq - 1) + off)
                                           : Lk - 1;
    const int last = p.causal ? min(Lk - 1, min(tile0 + (1 << bm_shift), Lq) - 1 + off) : Lk - 1;
    const int tiles = last < 0 ? 0 : last / kKeys + 1;

    // ---- this lane's query row: dims 16 c + 8 h ..
    V8 qf[DP / 16];
    {
        const T *qp = static_cast<const T *>(p.q) + (long)(o.first + qrow) * p.q_ts + head * p.q_hs;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            u32x4_t x = {0, 0, 0, 0};
            if (16 * c + 8 * h < p.D) x = *reinterpret_cast<const u32x4_t *>(qp + 16 * c + 8 * h);
            qf[c] = __builtin_bit_cast(V8, x);
        }
    }
    // ---- staging: unit i of a tile is (key, unit) = ((tid + i NT) / UPR, % UPR)
    const int su = tid % UPR, sr = tid / UPR;        // NT is a multiple of UPR
    const bool in = su * 8 < p.D;               // past the head's dims: unit 0's, and zeros stored
    const T *kp = static_cast<const T *>(p.k) + (long)o.k_first * p.k_ts + kvh * p.k_hs + (in ? su * 8 : 0);
    const T *vp = static_cast<const T *>(p.v) + (long)o.k_first * p.v_ts + kvh * p.v_hs + (in ? su * 8 : 0);
    const T *kn = kp + sr * p.k_ts, *vn = vp + sr * p.v_ts;    // this thread's first row of the next tile
    u32x4_t kr[CH], vr[CH];
    auto load = [&](int tile) __attribute__((always_inline)) {
        if ((tile + 1) * kKeys <= Lk) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                kr[i] = *reinterpret_cast<const u32x4_t *>(kn + i * (NT / UPR) * p.k_ts);
                vr[i] = *reinterpret_cast<const u32x4_t *>(vn + i * (NT / UPR) * p.v_ts);
            }
            kn += kKeys * p.k_ts;
            vn += kKeys * p.v_ts;
        } else {                                       // past the end: the last key again
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const long key = min(tile * kKeys + sr + i * (NT / UPR), Lk - 1);
                kr[i] = *reinterpret_cast<const u32x4_t *>(kp + key * p.k_ts);
                vr[i] = *reinterpret_cast<const u32x4_t *>(vp + key * p.v_ts);
            }
        }
    };
    auto store = [&](int tile) __attribute__((always_inline)) {
        if (p.D < DP && !in)
#pragma unroll
            for (int i = 0; i < CH; ++i) kr[i] = vr[i] = u32x4_t{0, 0, 0, 0};
        unsigned char *ks = sm + (tile & 1) * 2 * TILE, *vs = ks + TILE;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int r = sr + i * (NT / UPR);
            *reinterpret_cast<u32x4_t *>(ks + r * ROWB + k_unit<ROWB>(r, su) * 16) = kr[i];
            *reinterpret_cast<u32x4_t *>(vs + r * ROWB + v_unit<ROWB>(r, su >> 1) * 32 + (su & 1) * 16) = vr[i];
        }
    };
    f32x16_t acc[DP / 32] = {};
    float m = -INFINITY, ref = 0.f, l = 0.f;
    constexpr float bias = AGAIN ? 0.f : E::kBias;   // in ref; AGAIN, where ref - bias may be rounded, beside it
    if (tiles) {
        load(0);
        store(0);
    }
    loads_done();
    // this lane's part of a transposed V read: key 4 h + i / 4, dims 16 g + 4 (i % 4) .. of 32
    const int vkey = 4 * h + ((lane & 15) >> 2), vg = lane >> 4 & 1, vb = (lane & 3) * 8;
    for (int tile = 0; tile < tiles; ++tile) {
        __syncthreads();
        load(tile + 1);                              // past the end: the last key's rows again
        const int k0 = tile * kKeys + kb;
        if (k0 <= lim_hi) {
            const unsigned char *ks = sm + (tile & 1) * 2 * TILE, *vs = ks + TILE;
            f32x16_t s[NB] = {};
            // operands are read two steps before the products that take them; the
            // barriers keep the compiler from moving the reads back to their use
            constexpr int NC = DP / 16;
            u32x4_t kf[3][NB];
            auto read_k = [&](int c) __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int r = kb + 32 * b + n;
                    kf[c % 3][b] = *reinterpret_cast<const u32x4_t *>(ks + r * ROWB + k_unit<ROWB>(r, 2 * c + h) * 16);
                }
            };
            read_k(0);
            read_k(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (c + 2 < NC) read_k(c + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int b = 0; b < NB; ++b) s[b] = E::mma(__builtin_bit_cast(V8, kf[c % 3][b]), qf[c], s[b]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // From here the wave goes before the SIMD's others: its vector work then runs
            // beside their score products and not after them (16384 tokens, 32 / 8 heads
            // of 128: 2265 -> 2192 us; the score products first: no gain).
            __builtin_amdgcn_s_setprio(1);
            if (k0 + 32 * NB - 1 > lim_lo) mask_tile(s, lim, k0, h);
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) t0 = fmaxf(t0, s[0][r]), t1 = fmaxf(t1, s[NB - 1][r]);
            raise_max<false>(halves_max(fmaxf(t0, t1)) * p.scale2, bias, m, ref, l, acc);
            if (AGAIN)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] = rounded_score(s[b][r], p.scale2) - ref + E::kBias;
            // The weights of 16 keys at a time (registers 8 f .. 8 f + 7 of a block);
            // between the products of one 16 go the exponentials and the V reads of
            // the next.  They are rounded to the inputs' type, relative to their size
            // and each by itself, as the output is once more: over many keys the errors
            // average out.  Their sum is of the unrounded ones, in fp32, a tile's by itself
            // first: many small weights beside a large one are not rounded away one by one.
            constexpr int NT2 = DP / 32, VB = NT2 < 4 ? NT2 : 4, PART = 8 / NT2;
            V8 pf[2 * NB];
            float lt = 0.f;
            auto weight = [&](int f, int e) __attribute__((always_inline)) {
                const float y = s[f >> 1][8 * (f & 1) + e];
                const float x = __builtin_amdgcn_exp2f(AGAIN ? y : fmaf(y, p.scale2, -ref));
                lt += x;
                pf[f][e] = E::from(x);
            };
            // V operands (f, t) in order, VB of them read ahead
            s16x4_t vf[2 * VB][2];
            auto read_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int r = kb + 16 * (i / NT2) + 8 * y + vkey, t = i % NT2;
                    auto *at = (__attribute__((address_space(3))) s16x4_t *)(vs + r * ROWB +
                                                                          v_unit<ROWB>(r, 2 * t + vg) * 32 + vb);
                    vf[i % (2 * VB)][y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
                }
            };
            auto v_of = [&](int i) __attribute__((always_inline)) {
                return __builtin_bit_cast(V8, __builtin_shufflevector(vf[i % (2 * VB)][0], vf[i % (2 * VB)][1], 0, 1, 2, 3,
                                                                      4, 5, 6, 7));
            };
            if constexpr (AGAIN) {
#pragma unroll
                for (int i = 0; i < 16 * NB; ++i) weight(i / 8, i % 8);
#pragma unroll
                for (int t = 0; t < NT2; ++t) {
                    V8 z[2 * NB];
                    uint32_t has = 0;
#pragma unroll
                    for (int f = 0; f < 2 * NB; ++f) {
                        read_v(f * NT2 + t);
                        z[f] = v_of(f * NT2 + t);
                        has |= has_marks<E>(z[f]);
                    }
                    if (__any((has & 0x80008000u) != 0)) {
                        f32x16_t marks = {};
#pragma unroll
                        for (int f = 0; f < 2 * NB; ++f)
                            marks = E::mma(take_marks<E>(z[f]), seen_keys<E>(f, lim - k0 - 4 * h), marks);
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[t][r] += from_marks(marks[r]);
                    }
#pragma unroll
                    for (int f = 0; f < 2 * NB; ++f) acc[t] = E::mma(z[f], pf[f], acc[t]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int i = 0; i < VB; ++i) read_v(i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 8; ++e) weight(0, e);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2 * NB * NT2; ++i) {
                    const int f = i / NT2, t = i % NT2;
                    if (i + VB < 2 * NB * NT2) read_v(i + VB);
                    __builtin_amdgcn_sched_barrier(0);
                    acc[t] = E::mma(v_of(i), pf[f], acc[t]);
                    if (f < 2 * NB - 1)
#pragma unroll
                        for (int e = 0; e < PART; ++e) weight(f + 1, t * PART + e);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            l += lt;
        }
        __builtin_amdgcn_s_setprio(0);
        if (tile + 1 < tiles) store(tile + 1);
    }
    l = halves_sum(l);
    // A weight of 0 times an infinity or a NaN is a NaN in the matrix product: an
    // output that is NaN may come from a key its row does not see.  Where a wave has
    // one, or a maximum past kFar, the workgroup goes through its keys once more, with
    // V's infinities and NaN taken out of the product and counted in one of their own
    // over the keys that each row sees.  16384 bf16 tokens, 32 / 8 heads of 128: 2.3 ms, with
    // one NaN among the values 5.0, with nothing but NaN 11.3 (4096 tokens: 0.15, 0.35,
    // 0.83); fp32, 4096 tokens: 0.74, 1.7, 2.6.
    int *flags = reinterpret_cast<int *>(sm + 4 * TILE);
    bool redo = false;
    if (!AGAIN) {
        redo = fabsf(m) > kFar && m != -INFINITY;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) redo |= acc[t][r] != acc[t][r];
        redo = __any(redo);
    }
    if (KS == 2) {
        // [row wave][acc registers, m, l][lane]
        constexpr int REGS = DP / 2 + 2;
        float *pair = reinterpret_cast<float *>(sm) + wr * REGS * 64 + lane;
        if (any_wave(flags, redo)) return kAgain;    // a barrier: the tiles are done with
        if (kb) {
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) pair[(16 * t + r) * 64] = acc[t][r];
            pair[(REGS - 2) * 64] = m;
            pair[(REGS - 1) * 64] = l;
        }
        __syncthreads();
        if (kb) return kDone;
        const float m1 = pair[(REGS - 2) * 64], mn = fmaxf(m, m1), rn = (mn == -INFINITY ? 0.f : mn) - bias;
        const float a0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - rn);
        const float a1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - bias - rn);
        ref = rn;
        m = mn;
        l = fmaf(a0, l, a1 * pair[(REGS - 1) * 64]);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][r] = fmaf(a0, acc[t][r], a1 * pair[(16 * t + r) * 64]);
    }
    if (row < Lq && !redo && mine) {
        const size_t at = (size_t)(o.first + row) * p.Hq + head;
        const bool none = lim < 0;                   // no key: 0; with keys l = 0 is no softmax, NaN
        const float inv = 1.f / l;
        T *op = static_cast<T *>(p.out) + at * p.D;
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int d = 32 * t + 8 * x + 4 * h;
                if (d < p.D) {
                    typedef decltype(E::from(0.f)) e4_t __attribute__((ext_vector_type(4)));
                    e4_t y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = E::from(none ? 0.f : acc[t][4 * x + e] * inv);
                    *reinterpret_cast<e4_t *>(op + d) = y;
                }
            }
        if (p.lse && h == 0) p.lse[at] = l == 0.f ? -INFINITY : (ref + (bias - E::kBias) + __builtin_amdgcn_logf(l)) * kLn2;
    }
    if (AGAIN || KS == 2 || !any_wave(flags, redo)) return kDone;
    return redo ? kAgain : kOthersAgain;
}

template <typename E, int DP, int KS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(DP > 128 ? 1 : DP > 64 ? 2 : 3))) void prompt_attn_kernel(
    PromptParams p, int slots) {
    const int left = prompt_block_attn<E, DP, KS, false>(p, slots, true);
    if (left != kDone) prompt_block_attn<E, DP, KS, true>(own_params(), slots, left == kAgain);
}

// fp32 on v_mfma_f32_32x32x16_bf16: every operand as three bf16 pieces whose sum it
// is (v1 = bf16(v), v2 = bf16(v - v1), v3 the rest; an fp32 value's 24 bits), the
// products of pieces i and j with i + j <= 4, six of nine; the others are below
// 2^-25 of the term.  The first pieces' products have accumulators of their own,
// the five smaller kinds others: no small product is added to a large sum before
// the end (head dims past 128 have registers for one set).  Six bf16 products take
// 3 / 8 of the time of v_mfma_f32_32x32x2 on the same operands: 2048 tokens of two
// sequences, 32 / 8 heads of 128, 328 -> 157 us.  K and V are split as they are
// staged, in [piece][key] planes: a tile's loads are issued a tile ahead, and its
// split goes between the products of the tile before (head dims past 128 have LDS for
// one buffer and split between barriers).  One wave per SIMD, for the registers of two
// sets of accumulators; with Q and the sets held in accumulation registers 147 us.
//
// AGAIN: as in prompt_block_attn, and with pieces that hold any value.
template <int DP, int BUFFERS, bool AGAIN>
__device__ __forceinline__ int prompt_block_f32(const PromptParams &p, int slots, bool mine) {
    constexpr int NW = 4, NT = 64 * NW, ROWB = 2 * DP, UPR = DP / 8, KEYS = 32, PLANE = KEYS * ROWB;
    constexpr int CH = KEYS * UPR / NT, NT2 = DP / 32, NC = DP / 16;
    constexpr int SETS = DP > 128 ? 1 : 2;           // of output accumulators
    extern __shared__ __align__(16) unsigned char sm[];   // [buffer][K pieces, V pieces][32 keys], flags
    const int tid = own_thread<AGAIN>(), lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int bm_shift = 5 + __builtin_ctz(NW) - p.hw;
    PromptBlock o;
    if (!prompt_block(p, slots, bm_shift, o)) return kDone;
    if (o.b < 0 || o.b >= p.B) {
        zero_rows<float>(p, o, bm_shift);
        return kDone;
    }
    const int head = o.head0 + (w & ((1 << p.hw) - 1)), kvh = o.head0 / (p.Hq / p.Hkv);
    const int Lq = o.len, Lk = o.Lk, off = Lk - Lq;
    const int tile0 = o.tile << bm_shift;
    const int row0 = tile0 + 32 * (w >> p.hw), row = row0 + n;
    const int qrow = min(row, Lq - 1);
    const int lim = p.causal ? min(Lk - 1, qrow + off) : Lk - 1;
    const int lim_lo = p.causal ? min(Lk - 1, row0 + off) : Lk - 1;
    const int lim_hi = !mine || row0 >= Lq ? -1
                       : p.causal          ? min(Lk - 1, min(row0 + 31, Lq - 1) + off)
                                           : Lk - 1;
    const int last = p.causal ? min(Lk - 1, min(tile0 + (1 << bm_shift), Lq) - 1 + off) : Lk - 1;
    const int tiles = last < 0 ? 0 : last / KEYS + 1;

    const float *qp = static_cast<const float *>(p.q) + (long)(o.first + qrow) * p.q_ts + head * p.q_hs;
    bf16x8_t qf[NC][3];                              // dims 16 c + 8 h ..
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float x[8] = {};
        if (16 * c + 8 * h < p.D) {
            const f32x4_t a = *reinterpret_cast<const f32x4_t *>(qp + 16 * c + 8 * h);
            const f32x4_t b = *reinterpret_cast<const f32x4_t *>(qp + 16 * c + 8 * h + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
        }
        if (AGAIN) split3_any(x, qf[c]);
        else split3_bf16(x, qf[c]);
    }
    const int su = tid % UPR, sr = tid / UPR;
    const bool in = su * 8 < p.D;
    const float *kp = static_cast<const float *>(p.k) + (long)o.k_first * p.k_ts + kvh * p.k_hs + (in ? su * 8 : 0);
    const float *vp = static_cast<const float *>(p.v) + (long)o.k_first * p.v_ts + kvh * p.v_hs + (in ? su * 8 : 0);
    f32x4_t kr[CH][2], vr[CH][2];
    auto load = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const long key = min(tile * KEYS + sr + i * (NT / UPR), Lk - 1);   // past the end: the last again
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                kr[i][y] = *reinterpret_cast<const f32x4_t *>(kp + key * p.k_ts + 4 * y);
                vr[i][y] = *reinterpret_cast<const f32x4_t *>(vp + key * p.v_ts + 4 * y);
            }
        }
    };
    // Part j of the loaded tile into its planes: unit j / 2 of K, or of V.
    auto store_part = [&](int tile, int j) __attribute__((always_inline)) {
        unsigned char *ks = sm + (BUFFERS == 2 ? tile & 1 : 0) * 6 * PLANE, *vs = ks + 3 * PLANE;
        const int i = j >> 1, r = sr + i * (NT / UPR);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p.D < DP && !in ? 0.f : (j & 1 ? vr : kr)[i][e / 4][e % 4];
        bf16x8_t y[3];
        if (AGAIN) split3_any(x, y);
        else split3_bf16(x, y);
#pragma unroll
        for (int z = 0; z < 3; ++z)
            if (j & 1)
                *reinterpret_cast<bf16x8_t *>(vs + z * PLANE + r * ROWB + v_unit<ROWB>(r, su >> 1) * 32 +
                                              (su & 1) * 16) = y[z];
            else
                *reinterpret_cast<bf16x8_t *>(ks + z * PLANE + r * ROWB + k_unit<ROWB>(r, su) * 16) = y[z];
    };
    auto store = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2 * CH; ++j) store_part(tile, j);
    };
    // c += the six products of a and b, the largest into c0
    auto mma6 = [&](const bf16x8_t (&a)[3], const bf16x8_t (&b)[3], f32x16_t &c0, f32x16_t &c1)
                    __attribute__((always_inline)) {
        c1 = Bf16::mma(a[0], b[2], c1);
        c1 = Bf16::mma(a[1], b[1], c1);
        c1 = Bf16::mma(a[2], b[0], c1);
        c1 = Bf16::mma(a[0], b[1], c1);
        c1 = Bf16::mma(a[1], b[0], c1);
        c0 = Bf16::mma(a[0], b[0], c0);
    };
    f32x16_t acc[SETS * NT2] = {};                   // [t]: first pieces; the other set: the smaller products
    float m = -INFINITY, ref = 0.f, l = 0.f;
    if (tiles) {
        load(0);
        store(0);
    }
    loads_done();
    if (BUFFERS == 2 && tiles) load(1);              // past the end: the last key's rows again
    const int vkey = 4 * h + ((lane & 15) >> 2), vg = lane >> 4 & 1, vb8 = (lane & 3) * 8;
    for (int tile = 0; tile < tiles; ++tile) {
        __syncthreads();
        if (BUFFERS == 1 && tile + 1 < tiles) load(tile + 1);
        const int k0 = tile * KEYS;
        // all waves split their parts; with a branch for those without rows 2048 tokens of
        // two sequences take 146 us instead of 135
        if (BUFFERS == 2 || k0 <= lim_hi) {
            const unsigned char *ks = sm + (BUFFERS == 2 ? tile & 1 : 0) * 6 * PLANE, *vs = ks + 3 * PLANE;
            f32x16_t s0 = {}, s1 = {};
            // Q stays in accumulation registers, which the products read as they are
            if (DP <= 128)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int x = 0; x < 3; ++x) asm volatile("" : "+a"(qf[c][x]));
            bf16x8_t kf[2][3];
            auto read_k = [&](int c) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < 3; ++x)
                    kf[c % 2][x] = *reinterpret_cast<const bf16x8_t *>(ks + x * PLANE + n * ROWB +
                                                                      k_unit<ROWB>(n, 2 * c + h) * 16);
            };
            read_k(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (c + 1 < NC) read_k(c + 1);
                __builtin_amdgcn_sched_barrier(0);
                mma6(kf[c % 2], qf[c], s0, s1);
                // the next tile's split goes between the products
                if (BUFFERS == 2)
#pragma unroll
                    for (int j = c * 2 * CH / NC; j < (c + 1) * 2 * CH / NC; ++j) store_part(tile + 1, j);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (BUFFERS == 2) load(tile + 2);
            s0 += s1;
            if (k0 + KEYS - 1 > lim_lo) {            // mask_tile, whose array of one costs a spill here
                int rel = lim - k0 - 4 * h;
                asm volatile("" : "+v"(rel));
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (key_of(r) > rel) s0[r] = -INFINITY;
            }
            float t = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) t = fmaxf(t, s0[r]);
            raise_max<(DP <= 128)>(halves_max(t) * p.scale2, 0.f, m, ref, l, acc);
            if (AGAIN)
#pragma unroll
                for (int r = 0; r < 16; ++r) s0[r] = rounded_score(s0[r], p.scale2) - ref;
            bf16x8_t pf[2][3];
            float lt = 0.f;                              // a tile's sum by itself, as in prompt_block_attn
            constexpr int PART = NT2 < 4 ? 8 / NT2 : 2;
            auto weights = [&](int f, int e0, int e1) __attribute__((always_inline)) {
#pragma unroll
                for (int e = e0; e < e1; ++e) {
                    const float x = __builtin_amdgcn_exp2f(AGAIN ? s0[8 * f + e] : fmaf(s0[8 * f + e], p.scale2, -ref));
                    lt += x;
                    const __bf16 h1 = (__bf16)x;
                    const float r1 = x - (float)h1;
                    const __bf16 h2 = (__bf16)r1;
                    pf[f][0][e] = h1;
                    pf[f][1][e] = h2;
                    pf[f][2][e] = (__bf16)(r1 - (float)h2);
                }
            };
            s16x4_t vf[2][3][2];
            auto read_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < 3; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int r = 16 * (i / NT2) + 8 * y + vkey, t2 = i % NT2;
                        auto *at = (__attribute__((address_space(3))) s16x4_t *)(
                            vs + x * PLANE + r * ROWB + v_unit<ROWB>(r, 2 * t2 + vg) * 32 + vb8);
                        vf[i % 2][x][y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
                    }
            };
            auto v_of = [&](int i, bf16x8_t (&z)[3]) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < 3; ++x)
                    z[x] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(vf[i % 2][x][0], vf[i % 2][x][1], 0, 1, 2,
                                                                               3, 4, 5, 6, 7));
            };
            if constexpr (AGAIN) {                   // infinities and NaN are in the third pieces alone
                weights(0, 0, 8);
                weights(1, 0, 8);
#pragma unroll
                for (int t2 = 0; t2 < NT2; ++t2) {
                    bf16x8_t z[2][3];
                    uint32_t has = 0;
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
                        read_v(f * NT2 + t2);
                        v_of(f * NT2 + t2, z[f]);
                        has |= has_marks<Bf16>(z[f][2]);
                    }
                    if (__any((has & 0x80008000u) != 0)) {
                        f32x16_t marks = {};
#pragma unroll
                        for (int f = 0; f < 2; ++f)
                            marks = Bf16::mma(take_marks<Bf16>(z[f][2]), seen_keys<Bf16>(f, lim - k0 - 4 * h), marks);
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[t2][r] += from_marks(marks[r]);
                    }
#pragma unroll
                    for (int f = 0; f < 2; ++f) mma6(z[f], pf[f], acc[t2], acc[(SETS - 1) * NT2 + t2]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                read_v(0);
                __builtin_amdgcn_sched_barrier(0);
                weights(0, 0, 8);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2 * NT2; ++i) {
                    if (i + 1 < 2 * NT2) read_v(i + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    bf16x8_t z[3];
                    v_of(i, z);
                    mma6(z, pf[i / NT2], acc[i % NT2], acc[(SETS - 1) * NT2 + i % NT2]);
                    if (i * PART < 8) weights(1, i * PART, i * PART + PART);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            l += lt;
        }
        if (BUFFERS == 1) {
            __syncthreads();
            if (tile + 1 < tiles) store(tile + 1);
        }
    }
    l = halves_sum(l);
    f32x16_t sum[NT2];
    bool redo = fabsf(m) > kFar && m != -INFINITY;   // as in prompt_block_attn
#pragma unroll
    for (int t = 0; t < NT2; ++t) {
        sum[t] = acc[t];
        if (SETS == 2) sum[t] += acc[(SETS - 1) * NT2 + t];
#pragma unroll
        for (int r = 0; r < 16; ++r) redo |= sum[t][r] != sum[t][r];
    }
    redo = !AGAIN && __any(redo);
    if (row < Lq && !redo && mine) {
        const size_t at = (size_t)(o.first + row) * p.Hq + head;
        float *op = static_cast<float *>(p.out) + at * p.D;
#pragma unroll
        for (int t = 0; t < NT2; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int d = 32 * t + 8 * x + 4 * h;
                if (d < p.D) {
                    f32x4_t y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = lim < 0 ? 0.f : sum[t][4 * x + e] / l;   // as in prompt_block_attn
                    *reinterpret_cast<f32x4_t *>(op + d) = y;
                }
            }
        if (p.lse && h == 0) p.lse[at] = l == 0.f ? -INFINITY : (ref + __builtin_amdgcn_logf(l)) * kLn2;
    }
    if (AGAIN || !any_wave(reinterpret_cast<int *>(sm + BUFFERS * 6 * PLANE), redo)) return kDone;
    return redo ? kAgain : kOthersAgain;
}

template <int DP, int BUFFERS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void prompt_attn_f32_kernel(PromptParams p,
                                                                                                        int slots) {
    const int left = prompt_block_f32<DP, BUFFERS, false>(p, slots, true);
    if (left != kDone) prompt_block_f32<DP, BUFFERS, true>(own_params(), slots, left == kAgain);
}

namespace {
// Workgroups of a call whose wr waves (of different rows) take 1 << hw heads.
long slots_of(const PromptParams &p, int wr, int hw) {
    return (long)(p.Nq >> (5 + __builtin_ctz((unsigned)wr) - hw)) + p.B + 2;
}
int heads_shift(const PromptParams &p, int wr) {
    const int share = __builtin_ctz((unsigned)(p.Hq / p.Hkv)), most = __builtin_ctz((unsigned)wr);
    return share < most ? share : most;
}
// Sets p.hw, the LDS limit of kernel `fn` and the launch's size, or returns an error.
int prepare(const void *fn, PromptParams &p, int wr, size_t lds, DynLds *granted, int *slots, unsigned *groups) {
    const int rc = ensure_dyn_lds(fn, lds, granted);
    if (rc) return rc;
    p.hw = heads_shift(p, wr);
    const long rows = slots_of(p, wr, p.hw), all = rows * (p.Hq >> p.hw);
    if (all > 0xffffffL) {                           // a grid has fewer than 2^32 threads
        set_error("prompt attention: %d tokens of %d sequences and %d heads need %ld workgroups (at most 2^24 - 1)",
                  p.Nq, p.B, p.Hq, all);
        return OJASX_ERR_INVALID;
    }
    *slots = (int)rows;
    *groups = (unsigned)all;
    return OJASX_OK;
}
template <typename E, int DP, int KS>
int launch16_split(PromptParams p, hipStream_t st) {
    static DynLds granted;
    const size_t lds = (size_t)4 * kKeys * 2 * DP + kFlags;
    int slots;
    unsigned groups;
    const int rc = prepare(reinterpret_cast<const void *>(&prompt_attn_kernel<E, DP, KS>), p, 4 / KS, lds, &granted,
                           &slots, &groups);
    if (rc) return rc;
    OJX_LAUNCH((prompt_attn_kernel<E, DP, KS>), dim3(groups), dim3(256), lds, st, p, slots);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}
template <typename E, int DP>
int launch16(const PromptParams &p, hipStream_t st) {
    const int hw = heads_shift(p, 4);
    if (slots_of(p, 4, hw) * (p.Hq >> hw) > split_below(DP)) return launch16_split<E, DP, 1>(p, st);
    return launch16_split<E, DP, 2>(p, st);
}
template <int DP, int BUFFERS>
int launch32(PromptParams p, hipStream_t st) {
    static DynLds granted;
    const size_t lds = (size_t)BUFFERS * 6 * 32 * 2 * DP + kFlags;
    int slots;
    unsigned groups;
    const int rc = prepare(reinterpret_cast<const void *>(&prompt_attn_f32_kernel<DP, BUFFERS>), p, 4, lds, &granted,
                           &slots, &groups);
    if (rc) return rc;
    OJX_LAUNCH((prompt_attn_f32_kernel<DP, BUFFERS>), dim3(groups), dim3(256), lds, st, p, slots);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API int ojasx_prompt_attention_device(const void *q, long q_token_stride, long q_head_stride,
                                            const void *k, long k_token_stride, long k_head_stride,
                                            const void *v, long v_token_stride, long v_head_stride,
                                            int dtype, int num_q_tokens, int num_kv_tokens, int num_heads,
                                            int num_kv_heads, int head_dim, const int *cu_seqlens_q,
                                            const int *cu_seqlens_kv, int num_sequences, int causal,
                                            float scale, int zero_rest, void *out, float *lse,
                                            void *stream) {
    using namespace ojx;
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    constexpr int most = 0x7fffffff - 1024;          // row numbers of tiles that end past them are ints
    if (num_q_tokens < 0 || num_kv_tokens < 0 || num_q_tokens > most || num_kv_tokens > most || num_heads <= 0 ||
        num_heads > 65535 || num_kv_heads <= 0 || num_heads % num_kv_heads || num_sequences <= 0 ||
        num_sequences > (1 << 24)) {
        set_error("prompt attention: %d query and %d key tokens of %d sequences, %d query and %d kv heads",
                  num_q_tokens, num_kv_tokens, num_sequences, num_heads, num_kv_heads);
        return OJASX_ERR_INVALID;
    }
    if (head_dim <= 0 || head_dim > 256 || head_dim % 8) {
        set_error("prompt attention: head_dim %d is no multiple of 8 up to 256", head_dim);
        return OJASX_ERR_INVALID;
    }
    if (!(scale > 0.f) || !(scale * kLog2e < INFINITY)) {
        set_error("prompt attention: scale must be positive and finite (times log2(e), in fp32)");
        return OJASX_ERR_INVALID;
    }
    if (num_q_tokens == 0) return OJASX_OK;
    if (!q || !out || !cu_seqlens_q || !cu_seqlens_kv || (num_kv_tokens && (!k || !v))) return OJASX_ERR_NULL;
    const size_t es = dtype == OJASX_DTYPE_F32 ? 4 : 2;
    if (!rows_of_16(q, q_token_stride, q_head_stride, es) || !rows_of_16(out, 0, 0, es) ||
        (num_kv_tokens && (!rows_of_16(k, k_token_stride, k_head_stride, es) ||
                           !rows_of_16(v, v_token_stride, v_head_stride, es)))) {
        set_error("prompt attention: rows are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    PromptParams p{};
    p.q = q, p.k = k, p.v = v;
    p.q_ts = q_token_stride, p.q_hs = q_head_stride;
    p.k_ts = k_token_stride, p.k_hs = k_head_stride;
    p.v_ts = v_token_stride, p.v_hs = v_head_stride;
    p.out = out, p.lse = lse, p.cu_q = cu_seqlens_q, p.cu_k = cu_seqlens_kv;
    p.B = num_sequences, p.Nq = num_q_tokens, p.Nk = num_kv_tokens;
    p.Hq = num_heads, p.Hkv = num_kv_heads, p.D = head_dim;
    p.causal = causal != 0, p.zero_rest = zero_rest != 0, p.scale2 = scale * kLog2e;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == OJASX_DTYPE_F32)
        return head_dim <= 64 ? launch32<64, 2>(p, st) : head_dim <= 128 ? launch32<128, 2>(p, st)
                                                                        : launch32<256, 1>(p, st);
    if (dtype == OJASX_DTYPE_BF16)
        return head_dim <= 64    ? launch16<Bf16, 64>(p, st)
               : head_dim <= 128 ? launch16<Bf16, 128>(p, st)
                                 : launch16<Bf16, 256>(p, st);
    return head_dim <= 64    ? launch16<F16, 64>(p, st)
           : head_dim <= 128 ? launch16<F16, 128>(p, st)
                             : launch16<F16, 256>(p, st);
}

}  // extern "C"
