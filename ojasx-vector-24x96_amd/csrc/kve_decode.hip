// kve_decode.hip -- attention of one query token per sequence over the evicting KV cache
// (layout: kve.h), with the softmax's weights added to each token's count.
//
//   s_t = (q . k_t) scale,   p_t = exp(s_t - max s) / sum,   out = sum_t p_t v_t,
//   weight_t += the sum of p_t over the query heads of the kv head.
//
// Matrix products without a shuffle.  A workgroup takes the query heads of a kv head as the 16
// columns of v_mfma_f32_16x16x32 (bf16, fp16) or 16x16x4 (fp32): the scores are K Q^T, the
// output is V^T P^T, and both products give a lane the column (query head) lane % 16, so maxima,
// sums and rescaling stay in the lane.  The order of the terms within a product is free as long
// as both operands agree: row i of the score product's half u is token 8 (i / 4) + 4 u + i % 4
// of a tile of 32, and so a lane of quarter c = lane / 16 ends with the scores of tokens 8 c ..
// 8 c + 7, exactly the eight weights that the value product wants from it as its operand (fp32:
// row i is token i, and the four scores of a lane are its operands of four products).  The other
// operand, V^T, needs eight tokens of one dimension in a lane: a lane loads eight rows of eight
// dimensions, whole rows by sixteen lanes, and turns the 8 x 8 values in registers with byte
// permutations.  K, V and P never pass through LDS.
//
// Work: the tiles of all sequences are cut into chunks of equal size, as many as the card takes
// workgroups, whatever the lengths are; a workgroup's four waves take turns at the tiles of
// its chunk, join in LDS and leave (out, max, sums) to kve_join_kernel, which also turns the
// scores kept by the first kernel (fp32) into weights, once the sums over whole sequences are
// known.  Writes among the reads cost far more than their bytes: the scores, 3 % of what the
// kernel reads with four query heads of a kv head, took 27 us of 175 when each tile's were written
// at once, and 20 now that a chunk's are kept in LDS and written when it is done.  A workgroup with
// a whole sequence finishes output and weights itself.
//
// Bound by reading the pages.  Measured, bf16, 32 / 8 heads of 128: 64 sequences of 192000 tokens in
// all, 167 us (4.8 TB/s; without counting 146, 5.4) and join 17; one of 131072, 103 to 114 and 13; fp32, one of
// 2048: 10 and 6.5, both a launch and the chain of its loads.
//
// Scores, maxima, sums, counted weights and outputs are fp32.  For the value product of bf16 and fp16 a
// weight is the sum of two numbers of the type, and each tile's values are multiplied by both: to 2^-14 of
// it in bf16, 2^-20 in fp16 (there times 2^15, so that the smallest keep their share, those below 2^-20 to
// 2^-40 of the largest).  Both are above 0 where the weight is (fp16: from 2^-38 on): a value of infinity
// meets no 0 that the split has made.  One number each would be off by 2^-8 and 2^-11, as much as the
// output's own rounding.  The second product cost nothing that shows: the matrix units are busy in 4 % of the
// cycles instead of 3.
#include <cfloat>
#include <cmath>

#include "kve.h"

namespace ojx {

namespace {
constexpr int kNT = 256;
constexpr int kNW = kNT / 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMostGroup = 128;          // query heads of a kv head
constexpr int kLeastTiles = 4;           // tiles of a chunk, one for each wave
// Chunks that the tiles are cut into: four times what the card takes at once, so that the last ones end
// together; fewer where a kv head has many query heads, whose maxima and sums every item of the second
// kernel reads of all chunks.  64 sequences of 192000 bf16 tokens, 32 / 8 heads of 128, us with 512, 768,
// 1024 and 1536: 195, 186, 187, 181; one of 131072: 125, 129, 127, 131; 256 of 500: 130, 130, 130, 142;
// eight of 6000 with 32 / 8 heads of 256: 114, 119, 112, 130.  Four of 20000 with 40 / 1 heads, without the
// second rule: 56, 66, 85, 97.
constexpr int kMostChunks = 1024, kFewestChunks = 256, kChunkHeads = 8192;
// Scores of a chunk in LDS, so that as many workgroups of a CU find room as its registers take: two, and four
// of D = 64.
constexpr int kScoreFloats = 12288, kScoreFloats64 = 7168;

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u2_t __attribute__((ext_vector_type(2)));

// What a workgroup has: chunk j of k of sequence b, heads block hb of kv head h, and its tokens [t0, t1)
// of n held ones.  b < 0: nothing.  Chunks are numbered by sequence, then by place; the groups (kv head,
// heads block) of a chunk are neighbours.
struct KveItem {
    int b, h, hb, j, k, n, t0, t1;
    long first;                 // number of the item of chunk 0 of this group; the next is `groups` on
};

struct KveDecodeParams {
    KveView c;
    const void *q;              // [B][Hq][D]
    void *out;
    const int *held;
    float *part_o;              // [item][Rb][D]
    float *part_ml;             // [item][Rb][2]: max, sum
    KveItem *items;      // what the first kernel's workgroups had, for the second's
    float *scores;              // [B][Hkv][tiles][R][tokens of a tile] times log2(e), or null: no weights
    int Hq, R, HB, Rb;          // query heads, of a kv head, blocks of those, heads of a block
    int most, stride;           // bound on a sequence's tokens; the same in whole tiles
    int chunks, target;         // chunks that launch and partial results have room for; that the tiles are cut into
    int lds_scores;             // floats of scores in LDS
    float scale;                // scale factor x log2(e)
};

// Sum of v over the workgroup, in order of the threads' numbers; sh: kNW + 1 ints.
__device__ __forceinline__ int block_sum(int v, int *sh) {
    v = wave_scan_i(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < kNW; ++i) s += sh[i];
    return s;
}

// The workgroup's item.  The tiles of all sequences are cut into chunks of one size, whatever the lengths are.
template <int TT>
__device__ __forceinline__ KveItem kve_item(const KveDecodeParams &p, int *sh) {
    const int groups = p.c.Hkv * p.HB, B = p.c.B, tid = threadIdx.x;
    const long ci = blockIdx.x / groups;
    const int grp = blockIdx.x % groups;
    auto tiles = [&](int b) { return (min(max(p.held[b], 0), p.most) + TT - 1) / TT; };
    // tiles of a chunk; the sum of tiles stays within an int (the host's check)
    int mine = 0;
    for (int b = tid; b < B; b += kNT) mine += tiles(b);
    const long total = block_sum(mine, sh);
    const long size = max((long)kLeastTiles, (total * groups + p.target - 1) / p.target);
    long before = 0;
    KveItem it{-1, 0, 0, 0, 0, 0, 0, 0, 0};
    for (int b0 = 0; b0 < B; b0 += kNT) {
        const int b = b0 + tid, nt = b < B ? tiles(b) : 0;
        const int k = b < B ? max(1, (int)((nt + size - 1) / size)) : 0;     // no tokens: a chunk of none
        int incl = wave_scan_i(k);                                           // over the workgroup
        __syncthreads();
        if ((tid & 63) == 63) sh[tid >> 6] = incl;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int i = 0; i < kNW; ++i) {
            if (i < tid >> 6) incl += sh[i];
            all += sh[i];
        }
        const long j = ci - before - (incl - k);
        if (j >= 0 && j < k) {                    // one thread at most
            sh[kNW + 0] = b;
            sh[kNW + 1] = (int)j;
            sh[kNW + 2] = k;
        }
        if (ci >= before && ci < before + all) {  // the same for all threads
            __syncthreads();
            it.b = sh[kNW], it.j = sh[kNW + 1], it.k = sh[kNW + 2];
            break;
        }
        before += all;
    }
    // lengths that another stream changes meanwhile may ask for more chunks than there is room for
    it.k = min((long)it.k, p.chunks - (ci - it.j));
    if (it.b < 0 || it.j >= it.k) {
        it.b = -1;
        return it;
    }
    it.h = grp / p.HB, it.hb = grp % p.HB;
    it.first = (long)blockIdx.x - (long)it.j * groups;
    it.n = min(max(p.held[it.b], 0), p.most);
    const long nt = (it.n + TT - 1) / TT;
    it.t0 = (int)(nt * it.j / it.k) * TT;
    it.t1 = min(it.n, (int)(nt * (it.j + 1) / it.k) * TT);
    return it;
}
constexpr int kItemInts = kNW + 3;

__device__ __forceinline__ float swap32(float v, bool max_) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float x = __uint_as_float(a[0]), y = __uint_as_float(a[1]);
    return max_ ? fmaxf(x, y) : x + y;
}
__device__ __forceinline__ float swap16(float v, bool max_) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float x = __uint_as_float(a[0]), y = __uint_as_float(a[1]);
    return max_ ? fmaxf(x, y) : x + y;
}
// Over the four lanes of one column.
__device__ __forceinline__ float column_max(float v) { return swap16(swap32(v, true), true); }
__device__ __forceinline__ float column_sum(float v) { return swap16(swap32(v, false), false); }

// What the value product's weights are multiplied by.
template <typename T>
__device__ __forceinline__ constexpr float weight_scale() {
    return __is_same(T, __half) ? 32768.f : 1.f;
}

template <typename T>
struct Half;
template <>
struct Half<__hip_bfloat16> {
    typedef b8_t V8;
    static __device__ __forceinline__ f4_t mma(V8 a, V8 b, f4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // hi: 2^-8 below the weight and cut off, so that lo is at least 2^-8 of it
    static __device__ __forceinline__ void split(const float (&p)[8], V8 &hi, V8 &lo) {
        u4_t h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned a = __float_as_uint(p[2 * i] * (1.f - 0x1p-8f)), b = __float_as_uint(p[2 * i + 1] * (1.f - 0x1p-8f));
            h[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            lo[2 * i] = (__bf16)(p[2 * i] - __uint_as_float(a & 0xffff0000u));
            lo[2 * i + 1] = (__bf16)(p[2 * i + 1] - __uint_as_float(b & 0xffff0000u));
        }
        hi = __builtin_bit_cast(V8, h);
    }
};
template <>
struct Half<__half> {
    typedef h8_t V8;
    static __device__ __forceinline__ f4_t mma(V8 a, V8 b, f4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    // hi: 2^-10 below the weight and cut off, so that lo is at least 2^-10 of it; half of one whose 2^-10 is
    // next to the smallest number
    static __device__ __forceinline__ void split(const float (&p)[8], V8 &hi, V8 &lo) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = p[2 * i] * weight_scale<__half>(), b = p[2 * i + 1] * weight_scale<__half>();
            const auto h = __builtin_amdgcn_cvt_pkrtz(a * (a < 0x1p-13f ? 0.5f : 1.f - 0x1p-10f),
                                                      b * (b < 0x1p-13f ? 0.5f : 1.f - 0x1p-10f));
            hi[2 * i] = (_Float16)h[0], hi[2 * i + 1] = (_Float16)h[1];
            lo[2 * i] = (_Float16)(a - (float)hi[2 * i]);
            lo[2 * i + 1] = (_Float16)(b - (float)hi[2 * i + 1]);
        }
    }
};

// One tile of TT tokens of a page (or of two pages) in registers.
template <typename T, int D>
struct Tile {                                   // bf16, fp16: 32 tokens
    static constexpr int TT = 32, E = 8;        // tokens of a tile, and of a lane's scores
    static constexpr int NK = D / 32, DL = D / 16 < 8 ? D / 16 : 8, NV = D / 16 / DL;
    typedef typename Half<T>::V8 V8;
    V8 k[2][NK];
    unsigned v[E][NV][DL / 2];
    // a lane's token within the tile whose row of K it loads for half u
    static __device__ __forceinline__ int key(int i, int u) { return (i >> 2) * 8 + u * 4 + (i & 3); }
    static __device__ __forceinline__ int key_block(int i) { return i >> 3; }       // of 16 slots
    static __device__ __forceinline__ int value_block(int c) { return c >> 1; }
    __device__ __forceinline__ void load_k(const T *rows, int i, int c) {           // row of slot 0 of key_block
#pragma unroll
        for (int j = 0; j < NK; ++j)              // in the order of the products
#pragma unroll
            for (int u = 0; u < 2; ++u)
                k[u][j] = *reinterpret_cast<const V8 *>(rows + (key(i, u) & 15) * D + j * 32 + c * 8);
    }
    __device__ __forceinline__ void load_v(const T *rows, int i, int c) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const T *src = rows + ((c & 1) * 8 + e) * D + n * 128 + i * DL;
                if constexpr (DL == 8) {
                    const u4_t x = *reinterpret_cast<const u4_t *>(src);
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[e][n][w] = x[w];
                } else {
                    const u2_t x = *reinterpret_cast<const u2_t *>(src);
                    v[e][n][0] = x[0], v[e][n][1] = x[1];
                }
            }
    }
    __device__ __forceinline__ void clear_value(int e) {
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int w = 0; w < DL / 2; ++w) v[e][n][w] = 0;
    }
    // scores of the lane's tokens with 16 columns of queries
    __device__ __forceinline__ void scores(const V8 (&q)[NK], float (&s)[E]) const {
        f4_t a[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) a[u] = Half<T>::mma(k[u][j], q[j], a[u]);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = a[0][r], s[4 + r] = a[1][r];
    }
    // eight tokens of one dimension: dimension d of the lane's in half n
    __device__ __forceinline__ V8 column(int n, int d) const {
        u4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = __builtin_amdgcn_perm(v[2 * i + 1][n][d / 2], v[2 * i][n][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(V8, x);
    }
    // o += V^T P^T, two columns at a time, so that no product waits for the one before
    template <int NT>
    __device__ __forceinline__ void values(const float (&p)[NT][E], f4_t (&o)[NT][D / 16]) const {
        V8 hi[NT], lo[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) Half<T>::split(p[t], hi[t], lo[t]);
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int d = 0; d < DL; d += 2) {
                const V8 a = column(n, d), b = column(n, d + 1);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    f4_t &x = o[t][n * DL + d], &y = o[t][n * DL + d + 1];
                    x = Half<T>::mma(a, hi[t], x);
                    y = Half<T>::mma(b, hi[t], y);
                    x = Half<T>::mma(a, lo[t], x);
                    y = Half<T>::mma(b, lo[t], y);
                }
            }
    }
    static __device__ __forceinline__ void load_q(const T *q, int c, V8 (&f)[NK]) {
#pragma unroll
        for (int j = 0; j < NK; ++j) f[j] = *reinterpret_cast<const V8 *>(q + j * 32 + c * 8);
    }
    // Row 4 c + r of the value product's block a is dimension dim(a / DL, c, r) + a % DL.
    static __device__ __forceinline__ int dim(int n, int c, int r) { return n * 128 + (c * 4 + r) * DL; }
};

template <int D>
struct Tile<float, D> {                         // 16 tokens
    static constexpr int TT = 16, E = 4, NK = D / 16, NV = D / 64, DL = 4;
    typedef f4_t V8;
    f4_t k[NK], v[E][NV];
    static __device__ __forceinline__ int key_block(int) { return 0; }
    static __device__ __forceinline__ int value_block(int) { return 0; }
    __device__ __forceinline__ void load_k(const float *rows, int i, int c) {
#pragma unroll
        for (int j = 0; j < NK; ++j) k[j] = *reinterpret_cast<const f4_t *>(rows + i * D + j * 16 + c * 4);
    }
    __device__ __forceinline__ void load_v(const float *rows, int i, int c) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int n = 0; n < NV; ++n)
                v[e][n] = *reinterpret_cast<const f4_t *>(rows + (c * 4 + e) * D + n * 64 + i * 4);
    }
    __device__ __forceinline__ void clear_value(int e) {
#pragma unroll
        for (int n = 0; n < NV; ++n) v[e][n] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void scores(const V8 (&q)[NK], float (&s)[E]) const {
        // two sums at once: a product of this shape waits long for the one before
        f4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int m = 0; m < 4; m += 2) {
                a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][m], q[j][m], a, 0, 0, 0);
                b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j][m + 1], q[j][m + 1], b, 0, 0, 0);
            }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = a[r] + b[r];
    }
    template <int NT>
    __device__ __forceinline__ void values(const float (&p)[NT][E], f4_t (&o)[NT][D / 16]) const {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        o[t][n * 4 + m] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(v[e][n][m], p[t][e], o[t][n * 4 + m], 0, 0, 0);
    }
    static __device__ __forceinline__ void load_q(const float *q, int c, V8 (&f)[NK]) {
#pragma unroll
        for (int j = 0; j < NK; ++j) f[j] = *reinterpret_cast<const f4_t *>(q + j * 16 + c * 4);
    }
    static __device__ __forceinline__ int dim(int n, int c, int r) { return n * 64 + (c * 4 + r) * 4; }
};

// Adds to the weights of the item's tokens [t0, t1) of their kv head: the sum over its query heads of 2^(score -
// most(head)) inv(head).  scores: tiles [R][TT] from token 0 on.  A thread has kTokens tokens under way at a
// time: each needs its block table entry before its weight.
template <int TT, typename S, typename M, typename I>
__device__ __forceinline__ void add_weights(const KveDecodeParams &p, const KveItem &it, int t0, int t1, S scores, M most,
                                            I inv) {
    constexpr int kTokens = 4;
    const long hrow = (long)it.h << p.c.pshift;
    for (int first = t0 + (int)threadIdx.x; first < t1; first += kTokens * kNT) {
        long row[kTokens];
        float weight[kTokens], sum[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int t = first + i * kNT;
            row[i] = kve_row(p.c, it.b, min(t, t1 - 1));
            if (t >= t1) row[i] = -1;
            sum[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i) weight[i] = row[i] < 0 ? 0.f : p.c.w[row[i] + hrow];
#pragma unroll 4
        for (int r = 0; r < p.R; ++r) {
            float s[kTokens];
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                const int t = min(first + i * kNT, t1 - 1);
                s[i] = scores[(long)(t / TT) * (p.R * TT) + r * TT + t % TT];
            }
            const float m = most(r), f = inv(r);
#pragma unroll
            for (int i = 0; i < kTokens; ++i) sum[i] += exp2f(s[i] - m) * f;
        }
#pragma unroll
        for (int i = 0; i < kTokens; ++i)
            if (row[i] >= 0) p.c.w[row[i] + hrow] = weight[i] + sum[i];
    }
}
}  // namespace

// NT: blocks of 16 query heads that share a pass over the chunk.
template <typename T, int D, int NT>
__global__ __launch_bounds__(kNT) void kve_decode_kernel(KveDecodeParams p) {
#pragma clang fp contract(off)                   // s - m with both rounded alike: 0 for the largest score
    typedef Tile<T, D> Tl;
    constexpr int TT = Tl::TT, E = Tl::E, NA = D / 16;
    __shared__ int ish[kItemInts];
    __shared__ float ml[kNW][NT * 16][2];
    __shared__ float buf[kNW / 2][NT * NA * 4][64];
    extern __shared__ float lds_scores[];
    const KveItem it = kve_item<TT>(p, ish);
    // a whole sequence is done here, unless its weights take other workgroups' heads too
    const bool alone = it.k == 1 && (!p.scores || p.HB == 1);
    if (threadIdx.x == 0) {
        KveItem left = it;
        if (alone) left.b = -1;
        p.items[blockIdx.x] = left;
    }
    if (it.b < 0) return;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, c = lane >> 4;
    const int head0 = it.hb * p.Rb, heads = min(p.Rb, p.R - head0);     // of the kv head
    typename Tl::V8 q[NT][Tl::NK] = {};
#pragma unroll
    for (int t = 0; t < NT; ++t)
        if (t * 16 + i < heads)
            Tl::load_q(static_cast<const T *>(p.q) + ((size_t)it.b * p.Hq + it.h * p.R + head0 + t * 16 + i) * D, c, q[t]);
    f4_t o[NT][NA];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        m[t] = -INFINITY, l[t] = 0.f;
#pragma unroll
        for (int a = 0; a < NA; ++a) o[t][a] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    // Keys are loaded a tile ahead, into the registers of those that the scores are done with, values
    // as soon as their product is.  Loads come back in order, so the block table entries that the next
    // ones' addresses need are asked for before them, two tiles ahead: behind them, they would be there
    // only when all that was asked for before is (4.6 TB/s, where the pages can be read at 6).  For the
    // same reason no load of the loop hangs on a condition, under which the compiler would not know how
    // many to wait for: past its last tile a wave loads that one again, from the cache.
    const int *bt = p.c.bt + (long)it.b * p.c.max_pages;
    const int pmask = (1 << p.c.pshift) - 1, kb = Tl::key_block(i) * 16, vb = Tl::value_block(c) * 16;
    auto entry = [&](int t) { return bt[min(t >> p.c.pshift, p.c.max_pages - 1)]; };
    auto mapped = [&](int page) { return page >= 0 && page < p.c.num_pages; };
    auto row = [&](int page, int t) {
        return ((((long)(mapped(page) ? page : 0) * p.c.Hkv) + it.h) << p.c.pshift) + (t & pmask);
    };
    Tl tl;
    auto load_k = [&](int page, int t) {
        tl.load_k(reinterpret_cast<const T *>(p.c.k) + row(page, t + kb) * D, i, c);
    };
    auto load_v = [&](int page, int t) {
        tl.load_v(reinterpret_cast<const T *>(p.c.v) + row(page, t + vb) * D, i, c);
    };
    // A tile's scores, [R][tokens]: in LDS, as far as they find room, until the chunk is done.
    float *scores = p.scores + ((long)it.b * p.c.Hkv + it.h) * p.R * p.stride;
    auto store = [&](float *tile, const float (&raw)[NT][E]) {
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            if (b * 16 + i >= heads) continue;
            float *to = tile + (head0 + b * 16 + i) * TT + c * E;
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<f4_t *>(to + e) = f4_t{raw[b][e], raw[b][e + 1], raw[b][e + 2], raw[b][e + 3]};
        }
    };
    constexpr int kStep = kNW * TT;
    int t = it.t0 + wv * TT;
    int vp = 0, kp1 = 0, vp1 = 0;                 // of the tile's values, and of the next one's keys and values
    if (t < it.t1) {                              // and the loop with it, which no other way leads into
        const int kp = entry(t + kb);
        vp = entry(t + vb);
        const int next = t + kStep < it.t1 ? t + kStep : t;
        kp1 = entry(next + kb), vp1 = entry(next + vb);
        load_k(kp, t);
        __builtin_amdgcn_sched_barrier(0);        // in this order, as in the loop
        load_v(vp, t);
        do {
            const int next = t + kStep < it.t1 ? t + kStep : t, next2 = next + kStep < it.t1 ? next + kStep : next;
            const int kp2 = entry(next2 + kb), vp2 = entry(next2 + vb);
            __builtin_amdgcn_sched_barrier(0);        // no later
            const bool vin = mapped(vp);
            const int left = it.n - t - c * E;        // tokens from the lane's first one on
            const bool whole = __all(vin && left >= E);
            float w[NT][E];
#pragma unroll
            for (int b = 0; b < NT; ++b) tl.scores(q[b], w[b]);
            load_k(kp1, next);
            float raw[NT][E];
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                float (&s)[E] = w[b], most = -FLT_MAX;   // not -inf: some token is there, if all score that
#pragma unroll
                for (int e = 0; e < E; ++e) raw[b][e] = s[e] *= p.scale;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < E; ++e) most = fmaxf(most, s[e]);
                } else {
                    if (!vin || left <= 0) most = -INFINITY;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (!vin || e >= left) s[e] = -INFINITY;
                        most = fmaxf(most, s[e]);
                    }
                }
                if (__any(most > m[b])) {
                    most = fmaxf(m[b], column_max(most));
                    const float f = most == -INFINITY ? 1.f : exp2f(m[b] - most);
                    m[b] = most;
                    l[b] *= f;
#pragma unroll
                    for (int a = 0; a < NA; ++a) o[b][a] *= f;
                }
                const float base = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s[e] = __builtin_amdgcn_exp2f(s[e] - base);
                    l[b] += s[e];
                }
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!vin || e >= left) tl.clear_value(e);
            }
            tl.template values<NT>(w, o);
            load_v(vp1, next);
            if (p.scores) {
                const long tile = (long)(t - it.t0) * p.R;
                if (tile + p.R * TT <= p.lds_scores) store(lds_scores + tile, raw);
                else store(scores + (long)t * p.R, raw);
            }
            vp = vp1, kp1 = kp2, vp1 = vp2;
            t += kStep;
        } while (t < it.t1);
    }
    // the four waves' (max, sums, out) joined: 2 into 0 and 3 into 1, then 1 into 0
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        l[b] = column_sum(l[b]);
        if (c == 0) ml[wv][b * 16 + i][0] = m[b], ml[wv][b * 16 + i][1] = l[b];
    }
    __syncthreads();
    const int here = p.lds_scores / (p.R * TT) * TT;       // tokens whose scores are in LDS
    if (!alone) {
        const int n = min((it.t1 - it.t0 + TT - 1) / TT * TT, here) * p.R;
        float *to = scores + (long)it.t0 * p.R;
        for (int x = threadIdx.x * 4; x < n; x += kNT * 4)
            *reinterpret_cast<f4_t *>(to + x) = *reinterpret_cast<const f4_t *>(lds_scores + x);
    }
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        float most = ml[0][b * 16 + i][0];
#pragma unroll
        for (int x = 1; x < kNW; ++x) most = fmaxf(most, ml[x][b * 16 + i][0]);
        const float f = m[b] == -INFINITY ? 0.f : exp2f(m[b] - most);
        l[b] = 0.f;
#pragma unroll
        for (int x = 0; x < kNW; ++x) {
            const float mx = ml[x][b * 16 + i][0], g = mx == -INFINITY ? 0.f : exp2f(mx - most);
            l[b] += ml[x][b * 16 + i][1] * g;
        }
        if (f != 1.f) {                           // a wave without tokens has sums of 0, and no infinity to turn into NaN
#pragma unroll
            for (int a = 0; a < NA; ++a) o[b][a] *= f;
        }
        m[b] = most;
    }
    auto give = [&](float (*to)[64]) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[(b * NA + a) * 4 + r][lane] = o[b][a][r];
    };
    auto take = [&](float (*of)[64]) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[b][a][r] += of[(b * NA + a) * 4 + r][lane];
    };
    if (wv >= 2) give(buf[wv - 2]);
    __syncthreads();
    if (wv < 2) take(buf[wv]);
    __syncthreads();
    if (wv == 1) give(buf[0]);
    __syncthreads();
    if (wv == 0) {
        take(buf[0]);
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const int head = b * 16 + i;
            if (head >= heads) continue;
            if (alone) {
                // no tokens: 0; tokens that all score -inf: 0 / 0
                T *to = static_cast<T *>(p.out) + ((size_t)it.b * p.Hq + it.h * p.R + head0 + head) * D;
                const float sum = l[b] * weight_scale<T>();
#pragma unroll
                for (int n = 0; n < NA / Tl::DL; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int d = 0; d < Tl::DL; ++d)
                            store_act(to, Tl::dim(n, c, r) + d, m[b] == -INFINITY ? 0.f : o[b][n * Tl::DL + d][r] / sum);
                if (c == 0) ml[0][head][0] = m[b], ml[0][head][1] = 1.f / l[b];
            } else {
                const long at = (long)blockIdx.x * p.Rb + head;
                float *to = p.part_o + at * D;
#pragma unroll
                for (int n = 0; n < NA / Tl::DL; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int d = 0; d < Tl::DL; ++d) to[Tl::dim(n, c, r) + d] = o[b][n * Tl::DL + d][r];
                if (c == 0) *reinterpret_cast<float2 *>(p.part_ml + at * 2) = make_float2(m[b], l[b]);
            }
        }
    }
    if (!alone || !p.scores) return;
    __syncthreads();
    add_weights<TT>(p, it, 0, min(it.n, here), lds_scores, [&](int r) { return ml[0][r][0]; }, [&](int r) { return ml[0][r][1]; });
    add_weights<TT>(p, it, here, it.n, scores, [&](int r) { return ml[0][r][0]; }, [&](int r) { return ml[0][r][1]; });
}

// The chunks of a sequence joined, and its weights: workgroup = item of the first kernel.  Its share
// of the output is every k-th part of the group's, summed over all chunks; its share of the weights
// the tokens of its own chunk, over all query heads of the kv head (the first heads block's item does
// it).
template <typename T, int D, int TT>
__global__ __launch_bounds__(kNT) void kve_join_kernel(KveDecodeParams p) {
    __shared__ float most[kMostGroup], inv[kMostGroup], total[kMostGroup];
    const KveItem it = p.items[blockIdx.x];
    if (it.b < 0) return;
    const int tid = threadIdx.x, groups = p.c.Hkv * p.HB;
    const bool counts = p.scores && it.hb == 0;
    // maxima and sums of the heads that this item needs: its own block's, or all of the kv head; `each`
    // lanes for a head, as many heads at once as the workgroup has
    const int h0 = counts ? 0 : it.hb * p.Rb, h1 = counts ? p.R : min(p.R, h0 + p.Rb);
    int each = 64;
    while (each > 4 && each * (h1 - h0) > kNT) each /= 2;
    for (int r0 = h0; r0 < h1; r0 += kNT / each) {
        const int r = min(r0 + tid / each, h1 - 1), sub = tid % each;
        const float *of = p.part_ml + ((it.first + r / p.Rb - it.hb) * p.Rb + r % p.Rb) * 2;
        const long step = (long)groups * p.Rb * 2;
        float m = -INFINITY, l = 0.f;
#pragma unroll 4
        for (int j = sub; j < it.k; j += each) {
            const float2 x = *reinterpret_cast<const float2 *>(of + j * step);
            const float to = fmaxf(m, x.x), f = m == -INFINITY ? 0.f : exp2f(m - to), g = x.x == -INFINITY ? 0.f : exp2f(x.x - to);
            l = l * f + x.y * g;
            m = to;
        }
        for (int o = 1; o < each; o *= 2) {
            const float xm = __shfl_xor(m, o), xl = __shfl_xor(l, o);
            const float to = fmaxf(m, xm), f = m == -INFINITY ? 0.f : exp2f(m - to), g = xm == -INFINITY ? 0.f : exp2f(xm - to);
            l = l * f + xl * g;
            m = to;
        }
        if (sub == 0) most[r] = m, inv[r] = 1.f / l, total[r] = l * weight_scale<T>();
    }
    __syncthreads();
    // outputs: units of four values, each summed by `lanes` lanes
    const int heads = min(p.Rb, p.R - it.hb * p.Rb), units = heads * (D / 4);
    int lanes = 1;
    while (lanes < 64 && lanes < it.k) lanes *= 2;
    const int u0 = (int)((long)units * it.j / it.k), u1 = (int)((long)units * (it.j + 1) / it.k);
    const int sub = tid % lanes;
    for (int u = u0; u < u1; u += kNT / lanes) {           // whole waves stay in it: the sum below is theirs
        const int mine = u + tid / lanes, at = min(mine, u1 - 1), head = at / (D / 4), r = it.hb * p.Rb + head;
        const float m = most[r];
        f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int j = sub; j < it.k; j += lanes) {
            const long of = (it.first + (long)j * groups) * p.Rb + head;
            const float mj = p.part_ml[of * 2];
            const f4_t x = *reinterpret_cast<const f4_t *>(p.part_o + of * D + at % (D / 4) * 4);
            const float f = exp2f(mj - m);
            // a chunk without tokens has zeros, which no infinity or NaN may meet
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += mj == -INFINITY ? 0.f : x[e] * f;
        }
        for (int o = 1; o < lanes; o *= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], o);
        if (sub == 0 && mine < u1) {
            // no tokens: 0; tokens that all score -inf: 0 / 0
            T *to = static_cast<T *>(p.out) + ((size_t)it.b * p.Hq + it.h * p.R + r) * D + at % (D / 4) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) store_act(to, e, m == -INFINITY ? 0.f : sum[e] / total[r]);
        }
    }
    if (!counts) return;
    const float *scores = p.scores + ((long)it.b * p.c.Hkv + it.h) * p.R * p.stride;
    add_weights<TT>(p, it, it.t0, it.t1, scores, [&](int r) { return most[r]; }, [&](int r) { return inv[r]; });
}

namespace {
struct KvePlan {
    int R, NT, HB, Rb, TT, most, stride, target, lds_scores;
    long chunks, items, o_bytes, ml_bytes, item_bytes, s_bytes;
    long bytes() const { return o_bytes + ml_bytes + item_bytes + s_bytes; }
};
int kve_plan(const OjasxKVECache *c, const KveView &v, int num_q_heads, int max_held, int count, KvePlan *p) {
    if (num_q_heads <= 0 || num_q_heads % v.Hkv || max_held < 0) {
        set_error("KV decode: %d query heads for %d kv heads, max_held %d", num_q_heads, v.Hkv, max_held);
        return OJASX_ERR_INVALID;
    }
    p->R = num_q_heads / v.Hkv;
    if (p->R > kMostGroup) {
        set_error("KV decode: %d query heads of a kv head (at most %d)", p->R, kMostGroup);
        return OJASX_ERR_INVALID;
    }
    p->TT = v.dtype == OJASX_DTYPE_F32 ? 16 : 32;
    p->NT = p->R > 16 && !(v.dtype == OJASX_DTYPE_F32 && v.D == 256) ? 2 : 1;   // two would spill there
    p->HB = (p->R + p->NT * 16 - 1) / (p->NT * 16);
    p->Rb = (p->R + p->HB - 1) / p->HB;
    p->most = max_held && max_held < v.cap ? max_held : v.cap;
    const long groups = (long)v.Hkv * p->HB, tiles = ((long)p->most + p->TT - 1) / p->TT;
    p->stride = (int)(tiles * p->TT);
    // the chunks of a kv head: of size tiles * groups / target (all sequences' tiles), one more for each
    // sequence, and none smaller than kLeastTiles
    const int target = kChunkHeads / p->R;
    p->target = target > kMostChunks ? kMostChunks : target < kFewestChunks ? kFewestChunks : target;
    const long a = p->target / groups + v.B, b = v.B * ((tiles + kLeastTiles - 1) / kLeastTiles);
    p->chunks = a < b ? a : b;
    p->items = p->chunks * groups;
    if (p->items > 0xffffff || tiles * v.B > 0x7fffffffL) {
        set_error("KV decode: %d sequences of up to %d tokens with %d kv heads are more than a launch takes", v.B,
                  p->most, v.Hkv);
        return OJASX_ERR_INVALID;
    }
    p->o_bytes = p->items * p->Rb * v.D * 4;
    p->ml_bytes = (p->items * p->Rb * 8 + 15) / 16 * 16;     // what follows is 16-byte aligned
    p->item_bytes = p->items * (long)sizeof(KveItem);
    p->s_bytes = count ? (long)v.B * num_q_heads * p->stride * 4 : 0;
    const long all = (long)p->R * p->stride, room = v.D == 64 && p->NT == 1 ? kScoreFloats64 : kScoreFloats;
    p->lds_scores = count && p->HB == 1 ? (int)(all < room ? all : room) : 0;
    return OJASX_OK;
}

template <typename T, int D, int NT>
int decode(const KvePlan &pl, hipStream_t st, const KveDecodeParams &p) {
    const dim3 grid((unsigned)pl.items), block(kNT);
    const size_t lds = (size_t)pl.lds_scores * 4;
    static DynLds granted;
    if (lds) OJX_HIP(raise_dyn_lds(reinterpret_cast<const void *>(&kve_decode_kernel<T, D, NT>), lds, &granted));
    OJX_LAUNCH((kve_decode_kernel<T, D, NT>), grid, block, lds, st, p);
    OJX_LAUNCH((kve_join_kernel<T, D, Tile<T, D>::TT>), grid, block, 0, st, p);
    return OJASX_OK;
}
template <typename T, int D>
int decode(const KvePlan &pl, hipStream_t st, const KveDecodeParams &p) {
    constexpr int kNT2 = sizeof(T) == 4 && D == 256 ? 1 : 2;
    return pl.NT == 1 ? decode<T, D, 1>(pl, st, p) : decode<T, D, kNT2>(pl, st, p);
}
template <typename T>
int decode(int D, const KvePlan &pl, hipStream_t st, const KveDecodeParams &p) {
    return D == 64 ? decode<T, 64>(pl, st, p) : D == 128 ? decode<T, 128>(pl, st, p) : decode<T, 256>(pl, st, p);
}
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API long ojasx_kve_decode_workspace(const OjasxKVECache *cache, int num_q_heads, int max_held, int count) {
    using namespace ojx;
    KveView v{};
    KvePlan pl{};
    int rc = kve_view(cache, &v);
    if (!rc) rc = kve_plan(cache, v, num_q_heads, max_held, count, &pl);
    return rc ? rc : pl.bytes();
}

OJASX_API int ojasx_kve_decode_device(const OjasxKVECache *cache, const void *q, int num_q_heads, const int *held,
                                      int max_held, float scale_factor, int count, void *out, void *workspace,
                                      long workspace_bytes, void *stream) {
    using namespace ojx;
    KveDecodeParams p{};
    KvePlan pl{};
    int rc = kve_view(cache, &p.c);
    if (!rc) rc = kve_plan(cache, p.c, num_q_heads, max_held, count, &pl);
    if (rc) return rc;
    if (!q || !held || !out) return OJASX_ERR_NULL;
    p.scale = (scale_factor > 0.f || scale_factor != scale_factor ? scale_factor : 1.f / sqrtf((float)p.c.D)) * kLog2e;
    if (!(p.scale > 0.f) || p.scale > FLT_MAX) {
        set_error("KV decode: scale factor %g times log2(e) is not finite", (double)scale_factor);
        return OJASX_ERR_INVALID;
    }
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) {
        set_error("KV decode: queries and outputs are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < pl.bytes()) {
        set_error("KV decode: the workspace has to be 16-byte aligned and of %ld bytes, got %ld",
                  pl.bytes(), workspace_bytes);
        return OJASX_ERR_INVALID;
    }
    char *ws = static_cast<char *>(workspace);
    p.part_o = reinterpret_cast<float *>(ws);
    p.part_ml = reinterpret_cast<float *>(ws + pl.o_bytes);
    p.scores = count ? reinterpret_cast<float *>(ws + pl.o_bytes + pl.ml_bytes) : nullptr;
    p.items = reinterpret_cast<KveItem *>(ws + pl.o_bytes + pl.ml_bytes + pl.s_bytes);
    p.q = q, p.out = out, p.held = held;
    p.Hq = num_q_heads, p.R = pl.R, p.HB = pl.HB, p.Rb = pl.Rb, p.most = pl.most, p.stride = pl.stride,
    p.chunks = (int)pl.chunks, p.target = pl.target, p.lds_scores = pl.lds_scores;
    hipStream_t st = static_cast<hipStream_t>(stream);
    rc = p.c.dtype == OJASX_DTYPE_F32 ? decode<float>(p.c.D, pl, st, p)
         : p.c.dtype == OJASX_DTYPE_BF16 ? decode<__hip_bfloat16>(p.c.D, pl, st, p) : decode<__half>(p.c.D, pl, st, p);
    if (rc) return rc;
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

}  // extern "C"
