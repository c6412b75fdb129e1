// kv4_decode.hip -- attention of one query token per sequence over the 4-bit
// paged KV cache (format: kv4.h), on v_mfma_f32_16x16x32_f16 over the codes.
//
// With e = c - 8, K_d = lo_g + s_g c_d = mid_g + s_g e_d, mid = lo + 8 s, and V_d
// likewise (g the group of dimension d),
//   <q, K> = sum_g s_g <q_g, e_g> + mid_g sum(q_g),
//   out_d  = sum_t (p_t s_tg) e_td + sum_t p_t mid_tg  (over sum_t p_t),
// so the matrix operands are the integers -8 .. 7, exact in fp16, and the steps
// stay outside in fp32.  (With the codes 0 .. 15 themselves the two terms are
// each as large as lo, about two standard deviations of V, and their sum, an
// average over many tokens, much smaller: what fp32 rounds off them would show.)
// A column of the products is a (query head j,
// group g) pair: column j G + g of the score product holds q_j with every
// group but g zeroed, so one accumulator gives all groups' partial sums, each
// lane applies the steps of its own group only, and a sum over the G
// neighbouring lanes completes the score.  The weights p_t s_tg of that column
// are the B operand of the value product, whose rows are all the dimensions;
// the rows of the column's own group are kept.  16 / G query heads of a kv head
// share a workgroup's pass over the cache.
//
// Tokens go in tiles of 64 = 4 blocks of 16 slots.  Row rho of the score
// product's A operand in step i is slot 4 i + rho % 4 of block rho / 4, so a
// lane of quarter h = lane / 16 ends with the scores of all 16 slots of block
// h (result row 4 h + r) -- exactly the 8 + 8 tokens that the value product's
// operand layout asks of that quarter: the weights go from one product into
// the other within the lane, with no exchange.
//
// Queries: a head's values times a power of two that takes its largest to
// [2^14, 2^15) are fp16 as they are for bf16 and fp16 (what falls below fp16's
// normal range is below 2^-28 of the largest), and two fp16 pieces for fp32.
// Weights: times a power of two that takes the largest step of the tile to
// 2^15 or less, so that they fill fp16's range; one fp16 piece (2^-12) for bf16
// outputs, a second one for what it leaves for fp16 and fp32 outputs.  Scores,
// maxima, sums and outputs are fp32.
//
// The pass is split over the slots (gridDim.x); kv4_merge_kernel joins the
// splits' (out, max, sum).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv4.h"

namespace ojx {

namespace {
constexpr int kNT = 256;
constexpr int kNW = kNT / 64;
constexpr float kLog2e = 1.44269504088896340736f;

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u4_t __attribute__((ext_vector_type(4)));

struct Kv4DecodeParams {
    Kv4View c;
    const void *q;
    void *out;
    float *part_o, *part_ml;    // [B][Hq][splits][D], [B][Hq][splits][2]
    const int *seen;
    int Hq, R, splits;
    float scale;                // scale factor x log2(e)
};

// Slots of a sequence: used block-table entries and the tokens in entry e.
struct Kv4Extent {
    int entries, last, tail;    // entry `last` holds `tail` tokens, the others are full
};
__device__ __forceinline__ Kv4Extent kv4_extent(const Kv4View &c, int seen) {
    Kv4Extent x{0, 0, 0};
    if (seen <= 0) return x;
    const int P = 1 << c.pshift, opened = ((seen - 1) >> c.pshift) + 1;
    x.entries = min(opened, c.max_pages);
    x.last = kv4_entry(c, opened - 1);
    x.tail = (seen - 1) % P + 1;
    return x;
}

__device__ __forceinline__ h2_t as_h2(uint32_t u) { return __builtin_bit_cast(h2_t, u); }
// c - 8 of the two codes that a mask with 0x000f000f (0x00f000f0) leaves, as
// fp16: 0x6400 | c is 1024 + c, 0x6400 | 16 c is 1024 + 16 c.
__device__ __forceinline__ h2_t codes_low(uint32_t w) {
    const uint32_t u = (w & 0x000f000fu) | 0x64006400u;
    return as_h2(u) - h2_t{(_Float16)1032.f, (_Float16)1032.f};
}
__device__ __forceinline__ h2_t codes_high(uint32_t w) {
    const uint32_t u = (w & 0x00f000f0u) | 0x64006400u;
    return as_h2(u) * h2_t{(_Float16)0.0625f, (_Float16)0.0625f} -
           h2_t{(_Float16)72.f, (_Float16)72.f};
}
__device__ __forceinline__ float mid(h2_t st) { return fmaf(8.f, (float)st[0], (float)st[1]); }
__device__ __forceinline__ h8_t join(h2_t a, h2_t b, h2_t c, h2_t d) {
    return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Sum over the G neighbouring lanes of a column group (G = 1, 2, 4, 8).
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    if (G > 1) v += __int_as_float(dpp_i<0xB1>(__float_as_int(v)));
    if (G > 2) v += __int_as_float(dpp_i<0x4E>(__float_as_int(v)));
    if (G > 4) v += __int_as_float(dpp_i<0x141>(__float_as_int(v)));
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    if (G > 1) v = fmaxf(v, __int_as_float(dpp_i<0xB1>(__float_as_int(v))));
    if (G > 2) v = fmaxf(v, __int_as_float(dpp_i<0x4E>(__float_as_int(v))));
    if (G > 4) v = fmaxf(v, __int_as_float(dpp_i<0x141>(__float_as_int(v))));
    return v;
}
// Over the four quarters of the wave (lanes of one column).
__device__ __forceinline__ float quarters_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarters_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// 2^e that takes |v| > 0 to [2^14, 2^15); 1 for 0, infinities and NaN.
__device__ __forceinline__ float to_range(float v) {
    const int e = (int)((__float_as_uint(v) >> 23) & 0xff);
    // 2^(14 - (e - 127)), held to normal numbers
    return e == 0 || e == 255 ? (e == 0 && v != 0.f ? 0x1p126f : 1.f)
                              : __uint_as_float((uint32_t)min(max(268 - e, 1), 254) << 23);
}

template <int NW>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[NW]) {
    if (NW == 2) {
        const uint2 a = *reinterpret_cast<const uint2 *>(p);
        w[0] = a.x, w[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) {
            const u4_t a = reinterpret_cast<const u4_t *>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = a[e];
        }
    }
}
}  // namespace

template <typename T, int D, int GS>
__global__ __launch_bounds__(kNT) void kv4_decode_kernel(Kv4DecodeParams p) {
    constexpr int G = D / GS, HS = 16 / G, NJ = D / 32;
    constexpr int QP = sizeof(T) == 4 ? 2 : 1;                      // fp16 pieces of a query value
    constexpr int WP = std::is_same<T, __hip_bfloat16>::value ? 1 : 2;   // and of a weight
    __shared__ float so[kNW][HS][D];
    __shared__ float sm[kNW][HS][2];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int n = lane & 15, h = lane >> 4, j = n / G, g = n % G;
    const int b = blockIdx.z, slices = (p.R + HS - 1) / HS;
    const int kvh = blockIdx.y / slices, j0 = blockIdx.y % slices * HS;
    const int nj = min(HS, p.R - j0), head0 = kvh * p.R + j0;
    const Kv4Extent ext = kv4_extent(p.c, p.seen[b]);
    const int bps = p.c.pshift - 4;                                  // log2 of blocks per page
    const int blocks = ext.entries << bps, tiles = (blocks + 3) >> 2;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int t0 = blockIdx.x * per, t1 = min(tiles, t0 + per);
    if (t0 >= t1 && blockIdx.x > 0) return;                          // the merge knows the same

    // ---- the column's query: its group's dimensions, as fp16 pieces
    h8_t qf[QP][NJ];
    float qsum = 0.f, kq;
    {
        float x[NJ][8], mx = 0.f;
        const T *qr = static_cast<const T *>(p.q) + ((size_t)b * p.Hq + head0 + min(j, nj - 1)) * D;
#pragma unroll
        for (int jj = 0; jj < NJ; ++jj) {
            const bool mine = jj * 32 / GS == g && j < nj;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[jj][e] = mine ? load_act(qr, 32 * jj + 8 * h + e) : 0.f;
                mx = fmaxf(mx, fabsf(x[jj][e]));
            }
        }
        const float f = to_range(quarters_max(group_max<G>(mx)));
#pragma unroll
        for (int jj = 0; jj < NJ; ++jj)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = x[jj][e] * f;
                qsum += v;
                const _Float16 a = (_Float16)v;
                qf[0][jj][e] = a;
                if (QP > 1) qf[QP - 1][jj][e] = (_Float16)(v - (float)a);
            }
        qsum = quarters_sum(qsum);
        kq = p.scale / f;
    }

    f4_t acc[NJ][2];
#pragma unroll
    for (int i = 0; i < NJ; ++i) acc[i][0] = acc[i][1] = f4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, z = 0.f, f = 1.f;
    const int *bt = p.c.bt + (size_t)b * p.c.max_pages;
    for (int tile = t0 + w; tile < t1; tile += kNW) {
        // the block of this lane's K rows (n / 4 of the tile) and of its
        // weights (h): index in the pool, and the tokens it holds
        long kblk, vblk;
        int held;
        {
            auto at = [&](int x, int *tokens) __attribute__((always_inline)) {
                const int blk = 4 * tile + x, e = blk >> bps, o = blk & ((1 << bps) - 1);
                const int page = e < ext.entries ? bt[e] : -1;
                const bool ok = page >= 0 && page < p.c.num_pages;
                const int in_page = e == ext.last ? ext.tail : 1 << p.c.pshift;
                if (tokens) *tokens = ok ? min(max(in_page - 16 * o, 0), 16) : 0;
                return ((((long)(ok ? page : 0)) * p.c.Hkv + kvh) << bps) + o;
            };
            kblk = at(n >> 2, nullptr);
            vblk = at(h, &held);
        }
        uint32_t kw[4][NJ], vw[NJ][4];
        u4_t ksr[4], vsr[4];
        const uint8_t *kp = p.c.kc + kblk * (D * 8) + (n & 3) * (D / 2) + h * NJ * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<NJ>(kp + 4 * i * (D / 2), kw[i]);
        const u4_t *ksp = reinterpret_cast<const u4_t *>(p.c.ks + (vblk * G + g) * 16);
        const u4_t *vsp = reinterpret_cast<const u4_t *>(p.c.vs + (vblk * G + g) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) ksr[i] = ksp[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) vsr[i] = vsp[i];
        const uint8_t *vp = p.c.vc + vblk * (D * 8) + n * 16;
#pragma unroll
        for (int i = 0; i < NJ; ++i) load_words<4>(vp + i * 256, vw[i]);
        const bool whole = __all(held == 16);
        if (!whole) {           // what a slot without a token holds reaches nothing
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (4 * i + r >= held) ksr[i][r] = 0, vsr[i][r] = 0;
        }
        // ---- scores of the 16 tokens of block h, for this lane's column
        float sc[4][4], tmax = -INFINITY;
        h2_t smax = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int jj = 0; jj < NJ; ++jj) {
                const uint32_t v = kw[i][jj];
                const h8_t kf = join(codes_low(v), codes_high(v), codes_low(v >> 8), codes_high(v >> 8));
                if (QP > 1) a = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[QP - 1][jj], a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[0][jj], a, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const h2_t st = as_h2(ksr[i][r]);
                float v = group_sum<G>(fmaf(mid(st), qsum, (float)st[0] * a[r]));
                if (!whole && 4 * i + r >= held) v = -INFINITY;
                sc[i][r] = v;
                tmax = fmaxf(tmax, v);
                smax = __builtin_elementwise_max(smax, as_h2(vsr[i][r]));
            }
        }
        // ---- running maximum and the weights' power of two
        const float mn = fmaxf(m, quarters_max(tmax)), ref = mn == -INFINITY ? 0.f : mn;
        const float fn = fminf(to_range(quarters_max((float)smax[0])), 0x1p100f);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - ref) * kq);
        m = mn;
        const float fa = alpha * (fn / f);
        if (WP == 1 && !__all(fa == 1.f)) {
#pragma unroll
            for (int i = 0; i < NJ; ++i) acc[i][0] *= fa, acc[i][1] *= fa;
        }
        l *= alpha;
        z *= alpha;
        // where the outputs have fp16's or fp32's bits a tile's products get an
        // accumulator of their own, added to the sum so far in one rounding per
        // value (512 fp32 tokens per wave: 3.3e-7 off the exact sum, 4.3e-7 when
        // the matrix instructions add to the running sum themselves)
        f4_t part[WP == 1 ? 1 : NJ][2];
        if (WP > 1) {
#pragma unroll
            for (int i = 0; i < NJ; ++i) part[i][0] = part[i][1] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
        f = fn;
        // ---- weights and the value product
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            h8_t wf[WP];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float wv[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 2 * u + y;
                    const h2_t st = as_h2(vsr[i][r]);
                    const float pv = __builtin_amdgcn_exp2f((sc[i][r] - ref) * kq);
                    l += pv;
                    z = fmaf(pv, mid(st), z);
                    wv[r] = pv * ((float)st[0] * f);
                    // rounded to fp32 here: the pieces below are of one value (the
                    // compiler rounds the product to fp16 at once for one of them)
                    if (WP > 1) asm volatile("" : "+v"(wv[r]));
                }
                // token order of a mask with 0x000f000f: 0, 2, then 1, 3
                constexpr int order[4] = {0, 2, 1, 3};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const _Float16 a = (_Float16)wv[order[e]];
                    wf[0][4 * y + e] = a;
                    if (WP > 1) wf[WP - 1][4 * y + e] = (_Float16)(wv[order[e]] - (float)a);
                }
            }
#pragma unroll
            for (int i = 0; i < NJ; ++i) {
                const uint32_t a = vw[i][2 * u], c = vw[i][2 * u + 1];
                const h8_t ev = join(codes_low(a), codes_low(a >> 8), codes_low(c), codes_low(c >> 8));
                const h8_t od = join(codes_high(a), codes_high(a >> 8), codes_high(c), codes_high(c >> 8));
                f4_t *to = WP == 1 ? acc[i] : part[WP == 1 ? 0 : i];
#pragma unroll
                for (int x = WP - 1; x >= 0; --x) {
                    to[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ev, wf[x], to[0], 0, 0, 0);
                    to[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(od, wf[x], to[1], 0, 0, 0);
                }
            }
        }
        if (WP > 1) {
#pragma unroll
            for (int i = 0; i < NJ; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][e][r] = fmaf(acc[i][e][r], fa, part[WP == 1 ? 0 : i][e][r]);
        }
    }
    l = quarters_sum(l);
    z = quarters_sum(z);
    m *= kq;                                   // in log2 units, the same for a head's groups

    // ---- the waves' passes joined
    if (j < nj) {
        const float inv = 1.f / f;
#pragma unroll
        for (int i = 0; i < NJ; ++i)
            if (i * 32 / GS == g)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        so[w][j][32 * i + 2 * (4 * h + r) + e] = fmaf(acc[i][e][r], inv, z);
        if (g == 0 && h == 0) sm[w][j][0] = m, sm[w][j][1] = l;
    }
    __syncthreads();
    for (int x = tid; x < nj * D; x += kNT) {
        const int jj = x / D, d = x % D;
        float mm = -INFINITY;
#pragma unroll
        for (int k = 0; k < kNW; ++k) mm = fmaxf(mm, sm[k][jj][0]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        float o = 0.f, ll = 0.f;
#pragma unroll
        for (int k = 0; k < kNW; ++k) {
            const float a = __builtin_amdgcn_exp2f(sm[k][jj][0] - ref);
            o = fmaf(a, so[k][jj][d], o);
            ll = fmaf(a, sm[k][jj][1], ll);
        }
        const size_t row = (size_t)b * p.Hq + head0 + jj;
        if (p.splits == 1) {
            store_act(static_cast<T *>(p.out), row * D + d, ll == 0.f ? 0.f : o / ll);
        } else {
            p.part_o[(row * p.splits + blockIdx.x) * D + d] = o;
            if (d == 0) {
                float *ml = p.part_ml + (row * p.splits + blockIdx.x) * 2;
                ml[0] = mm;
                ml[1] = ll;
            }
        }
    }
}

// One workgroup per (query head, sequence): the splits that took tokens.
template <typename T>
__global__ __launch_bounds__(kNT) void kv4_merge_kernel(Kv4DecodeParams p, int D) {
    const int head = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
    const Kv4Extent ext = kv4_extent(p.c, p.seen[b]);
    const int tiles = ((ext.entries << (p.c.pshift - 4)) + 3) >> 2;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int used = per ? (tiles + per - 1) / per : 0;
    const size_t row = (size_t)b * p.Hq + head;
    const float *ml = p.part_ml + row * p.splits * 2, *po = p.part_o + row * p.splits * D;
    float mm = -INFINITY;
    for (int s = 0; s < used; ++s) mm = fmaxf(mm, ml[2 * s]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    if (d >= D) return;
    float o = 0.f, l = 0.f;
    for (int s = 0; s < used; ++s) {
        const float a = __builtin_amdgcn_exp2f(ml[2 * s] - ref);
        o = fmaf(a, po[(size_t)s * D + d], o);
        l = fmaf(a, ml[2 * s + 1], l);
    }
    store_act(static_cast<T *>(p.out), row * D + d, l == 0.f ? 0.f : o / l);
}

namespace {
int decode_heads_per_slice(int D, int GS) { return 16 / (D / GS); }

// Splits of the slots of a sequence: about four workgroups per CU over the
// whole call, each at least four tiles (one per wave) long.
int decode_splits(const OjasxKV4Cache *c, int Hq, int max_seen) {
    const int HS = decode_heads_per_slice(c->head_dim, c->group_size);
    const int R = Hq / c->num_kv_heads;
    const long groups = (long)c->num_sequences * c->num_kv_heads * ((R + HS - 1) / HS);
    const long slots = max_seen > 0 ? std::min((long)max_seen, (long)c->max_pages * c->page_size)
                                    : (long)c->max_pages * c->page_size;
    const long tiles = (slots + 63) / 64;
    long s = (1024 + groups - 1) / groups;
    if (s > (tiles + kNW - 1) / kNW) s = (tiles + kNW - 1) / kNW;
    return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

int decode_check(const OjasxKV4Cache *c, int Hq) {
    if (Hq <= 0 || Hq > 65535 || Hq % c->num_kv_heads || c->num_sequences > 65535) {
        set_error("4-bit KV decode: %d query heads for %d kv heads, %d sequences (at most 65535)", Hq,
                  c->num_kv_heads, c->num_sequences);
        return OJASX_ERR_INVALID;
    }
    return OJASX_OK;
}

template <typename T>
int launch_decode(const Kv4DecodeParams &p, int D, int GS, hipStream_t st) {
    const int HS = decode_heads_per_slice(D, GS);
    const dim3 grid(p.splits, p.c.Hkv * ((p.R + HS - 1) / HS), p.c.B);
    if (D == 64 && GS == 32) OJX_LAUNCH((kv4_decode_kernel<T, 64, 32>), grid, dim3(kNT), 0, st, p);
    else if (D == 64) OJX_LAUNCH((kv4_decode_kernel<T, 64, 64>), grid, dim3(kNT), 0, st, p);
    else if (D == 128 && GS == 32) OJX_LAUNCH((kv4_decode_kernel<T, 128, 32>), grid, dim3(kNT), 0, st, p);
    else if (D == 128 && GS == 64) OJX_LAUNCH((kv4_decode_kernel<T, 128, 64>), grid, dim3(kNT), 0, st, p);
    else if (D == 128) OJX_LAUNCH((kv4_decode_kernel<T, 128, 128>), grid, dim3(kNT), 0, st, p);
    else if (GS == 32) OJX_LAUNCH((kv4_decode_kernel<T, 256, 32>), grid, dim3(kNT), 0, st, p);
    else if (GS == 64) OJX_LAUNCH((kv4_decode_kernel<T, 256, 64>), grid, dim3(kNT), 0, st, p);
    else OJX_LAUNCH((kv4_decode_kernel<T, 256, 128>), grid, dim3(kNT), 0, st, p);
    if (p.splits > 1)
        OJX_LAUNCH(kv4_merge_kernel<T>, dim3(p.Hq, p.c.B), dim3(kNT), 0, st, p, D);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API long ojasx_kv4_decode_workspace(const OjasxKV4Cache *cache, int num_q_heads, int max_seen) {
    using namespace ojx;
    Kv4View v;
    int rc = kv4_view(cache, &v);
    if (!rc) rc = decode_check(cache, num_q_heads);
    if (rc) return rc;
    const long s = decode_splits(cache, num_q_heads, max_seen);
    return s == 1 ? 0 : s * cache->num_sequences * num_q_heads * (cache->head_dim + 2) * (long)sizeof(float);
}

OJASX_API int ojasx_kv4_decode_device(const OjasxKV4Cache *cache, const void *q, int num_q_heads, int dtype,
                                      const int *seen, int max_seen, float scale_factor, void *out,
                                      void *workspace, long workspace_bytes, void *stream) {
    using namespace ojx;
    Kv4DecodeParams p{};
    int rc = kv4_view(cache, &p.c);
    if (!rc) rc = decode_check(cache, num_q_heads);
    if (rc) return rc;
    if (!q || !seen || !out) return OJASX_ERR_NULL;
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    const int D = cache->head_dim;
    p.splits = decode_splits(cache, num_q_heads, max_seen);
    const size_t rows = (size_t)cache->num_sequences * num_q_heads;
    if (p.splits > 1) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
            workspace_bytes < (long)(rows * p.splits * (D + 2) * sizeof(float))) {
            set_error("4-bit KV decode: workspace of %ld bytes at %p (ojasx_kv4_decode_workspace; 16-byte "
                      "aligned)", workspace_bytes, workspace);
            return OJASX_ERR_INVALID;
        }
        p.part_o = static_cast<float *>(workspace);
        p.part_ml = p.part_o + rows * p.splits * D;
    }
    p.q = q, p.out = out, p.seen = seen, p.Hq = num_q_heads, p.R = num_q_heads / cache->num_kv_heads;
    p.scale = (scale_factor > 0.f ? scale_factor : 1.0f / sqrtf((float)D)) * kLog2e;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == OJASX_DTYPE_F32    ? launch_decode<float>(p, D, cache->group_size, st)
           : dtype == OJASX_DTYPE_BF16 ? launch_decode<__hip_bfloat16>(p, D, cache->group_size, st)
                                       : launch_decode<__half>(p, D, cache->group_size, st);
}

}  // extern "C"
