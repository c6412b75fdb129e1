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
// average over many tokens, much smaller: what fp32 rounds off them would show.
// Keys for bf16 outputs keep 0 .. 15 and lo: the scores are exact enough.)
//
// A column of the products is a (query head j, group g) pair: column j G + g of
// the score product holds q_j with every group but g zeroed, so one accumulator
// gives all groups' partial sums, each lane applies the steps of its own group
// only, and a sum over the G neighbouring lanes completes the score.  The weights
// p_t s_tg of that column are the B operand of the value product, whose rows are
// all the dimensions; the rows of the column's own group are kept.  16 / G query
// heads of a kv head share a workgroup's pass over the cache.  Where a kv head has
// no more than a quarter of them, its columns come C = 4 times, and copy c has the
// weights of slots 4 c .. 4 c + 3 of each block, the others' being 0: a quarter of
// the exponentials and steps for every lane.  The copies are joined as the waves
// are, each with its own maximum and sum.
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
// Work: the tiles of all sequences in one row, cut into equal runs, one for each
// of the W workgroups of a (kv head, slice of its query heads), whatever the
// sequences' lengths.  A workgroup goes through the sequences of its run; a
// sequence that lies in one run is written whole, of the others each run leaves
// (out, max, sum) in slot run + sequence, and kv4_merge_kernel joins them.
//
// Bound by the reading of the pages (a copy runs at 4.9 TB/s here): 131072 bf16 tokens,
// 32 / 8 heads of 128, groups of 64, 39 us for 151 MB, 3.8 TB/s (32 where the last-level
// cache holds them all); 64 sequences of 192000 tokens in all, groups of 32, 58 us for 247
// MB, 4.2 TB/s, and 100 us with 64 / 8 heads, which take two passes over the cache; with
// narrow heads by a wave's way through its tiles: 16 sequences of 32000 held fp16
// tokens, 16 heads of 64, 15 to 16.5 us for 35 MB.  The merge is a second launch, 4 to 5 us.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "kv4.h"

namespace ojx {

namespace {
constexpr int kNT = 256;
constexpr int kNW = kNT / 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMostRange = 0x1p40f;              // takes the smallest fp16 step to 2^16

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

struct Kv4DecodeParams {
    Kv4View c;
    const void *q;
    void *out;
    float *part_o, *part_ml;    // [W + B][Hq][D], [W + B][Hq][2]
    const int *seen;
    int Hq, R, W;
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
__device__ __forceinline__ int kv4_tiles(const Kv4View &c, int seen) {
    const Kv4Extent x = kv4_extent(c, seen);
    return ((x.entries << (c.pshift - 4)) + 3) >> 2;
}
// Sum over the lanes before and with this one.
__device__ __forceinline__ int wave_scan(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// Run i of a row of T tiles in W runs: q + 1 tiles each for the first T % W, then q.
struct Runs {
    int W, q, r;
    __device__ __forceinline__ Runs(int T, int most) : W(min(most, T)), q(0), r(0) {
        if (W) q = T / W, r = T - q * W;
    }
    __device__ __forceinline__ int start(int i) const { return i * q + min(i, r); }
    __device__ __forceinline__ int of(int tile) const {
        const int big = (q + 1) * r;
        return tile < big ? tile / (q + 1) : r + (tile - big) / q;
    }
};

// A row's output of its weighted sum o, the weights' sum l and the largest score m.
__device__ __forceinline__ float kv4_out(float o, float l, float m) {
    return m == -INFINITY ? 0.f : o / l;         // l = 0: only scores of -inf, no softmax, NaN
}

// The tiles of all sequences, those before sequence b and its own, from one look at
// each length.  Whole waves call it.
__device__ __forceinline__ int kv4_all_tiles(const Kv4View &c, const int *seen, int b, int *before, int *own) {
    const int lane = threadIdx.x & 63;
    int all = 0, bef = 0, mine = 0;
    for (int i = lane; i < c.B; i += 64) {
        const int n = kv4_tiles(c, seen[i]);
        all += n;
        if (i < b) bef += n;
        if (i == b) mine = n;
    }
    *own = __builtin_amdgcn_readlane(mine, b & 63);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o), bef += __shfl_xor(bef, o);
    *before = bef;
    return all;
}

// The two codes that a mask with 0x000f000f (0x00f000f0) leaves, as fp16, less 8
// with MID: 0x6400 | c is 1024 + c, 0x6400 | 16 c is 1024 + 16 c.  `magic` is
// 0x64006400 in a register, where the mask and the or are one instruction.
template <bool MID>
__device__ __forceinline__ h2_t codes_low(uint32_t w, uint32_t magic) {
    constexpr _Float16 k = (_Float16)(MID ? 1032.f : 1024.f);
    return as_h2((w & 0x000f000fu) | magic) - h2_t{k, k};
}
template <bool MID>
__device__ __forceinline__ h2_t codes_high(uint32_t w, uint32_t magic) {
    constexpr _Float16 k = (_Float16)(MID ? 72.f : 64.f);
    return as_h2((w & 0x00f000f0u) | magic) * h2_t{(_Float16)0.0625f, (_Float16)0.0625f} - h2_t{k, k};
}
// lo, or the value of code 8.
template <bool MID>
__device__ __forceinline__ float base(h2_t st) {
    return MID ? fmaf(8.f, (float)st[0], (float)st[1]) : (float)st[1];
}
__device__ __forceinline__ h8_t join(h2_t a, h2_t b, h2_t c, h2_t d) {
    return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Sum over the G neighbouring lanes of a column group (G = 1, 2, 4, 8).
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {   // folds into the instruction that uses it
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    if (G > 1) v += dpp_f<0xB1>(v);
    if (G > 2) v += dpp_f<0x4E>(v);
    if (G > 4) v += dpp_f<0x141>(v);
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    if (G > 1) v = fmaxf(v, dpp_f<0xB1>(v));
    if (G > 2) v = fmaxf(v, dpp_f<0x4E>(v));
    if (G > 4) v = fmaxf(v, dpp_f<0x141>(v));
    return v;
}
// Over the four quarters of the wave (lanes of one column): v_permlane16_swap of a
// register with itself leaves row 2 i and row 2 i + 1 of each pair side by side,
// v_permlane32_swap the halves.
__device__ __forceinline__ float quarters_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 2^e that takes |v| > 0 to [2^14, 2^15), held to normal numbers; 2^126 for 0, 1
// for infinities and NaN.
__device__ __forceinline__ float to_range(float v) {
    const int e = (int)((__float_as_uint(v) >> 23) & 0xff);
    return e == 255 ? 1.f : __uint_as_float((uint32_t)min(max(268 - e, 1), 253) << 23);
}

// A wave-uniform read of what no kernel of this file writes: a scalar load.
__device__ __forceinline__ int uniform_int(const int *p) {
    typedef __attribute__((address_space(4))) const int const_t;
    return *reinterpret_cast<const_t *>(reinterpret_cast<uintptr_t>(p));
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

template <typename T_, int D, int GS, int C>
__global__ __launch_bounds__(kNT) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2, 8))) void kv4_decode_kernel(
    Kv4DecodeParams p) {
    constexpr int G = D / GS, HS = 16 / G, NJ = D / 32;
    constexpr int HE = HS / C, NI = 4 / C;                           // heads of a slice, slot groups of a copy
    constexpr int QP = sizeof(T_) == 4 ? 2 : 1;                     // fp16 pieces of a query value
    constexpr int WP = std::is_same<T_, __hip_bfloat16>::value ? 1 : 2;   // and of a weight
    constexpr bool KMID = WP > 1;             // keys: codes 0 .. 15 do for bf16 outputs
    __shared__ float so[kNW][HS][D];                                 // the waves' outputs
    __shared__ float sm[kNW][HS][2];                                 // and (max, sum)
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, h = lane >> 4, j = n / G, g = n % G;
    const int slices = (p.R + HE - 1) / HE;
    const int kvh = blockIdx.y / slices, j0 = blockIdx.y % slices * HE;
    const int jh = j % HE, cp = j / HE;
    const int nj = min(HE, p.R - j0), head0 = kvh * p.R + j0;
    const int bps = p.c.pshift - 4;                                  // log2 of blocks per page
    // ---- this workgroup's run of tiles, and the sequence that it begins in
    int pos, end, b, first;                                          // first: number of b's first tile
    if (p.c.B <= 64) {
        const int own = lane < p.c.B ? kv4_tiles(p.c, p.seen[lane]) : 0;
        const int up = p.c.B == 1 ? __builtin_amdgcn_readfirstlane(own) : wave_scan(own);
        const Runs runs(__builtin_amdgcn_readlane(up, 63), p.W);
        if ((int)blockIdx.x >= runs.W) return;
        pos = runs.start(blockIdx.x);
        end = runs.start(blockIdx.x + 1);
        b = p.c.B == 1 ? 0 : __builtin_ctzll(__ballot(up > pos));
        first = __builtin_amdgcn_readlane(up - own, b);
    } else {
        int none, own0;
        const Runs runs(kv4_all_tiles(p.c, p.seen, 0, &none, &own0), p.W);
        if ((int)blockIdx.x >= runs.W) return;
        pos = runs.start(blockIdx.x);
        end = runs.start(blockIdx.x + 1);
        first = 0;
        b = p.c.B;
        for (int i0 = 0; i0 < p.c.B; i0 += 64) {
            const int i = i0 + lane, own = i < p.c.B ? kv4_tiles(p.c, p.seen[i]) : 0, up = wave_scan(own);
            const unsigned long long over = __ballot(first + up > pos);
            if (over) {
                const int at = __builtin_ctzll(over);
                first += __shfl(up - own, at);
                b = i0 + at;
                break;
            }
            first += __shfl(up, 63);
        }
    }
    pos = __builtin_amdgcn_readfirstlane(pos);
    end = __builtin_amdgcn_readfirstlane(end);
    b = __builtin_amdgcn_readfirstlane(b);
    first = __builtin_amdgcn_readfirstlane(first);
    uint32_t magic = 0x64006400u;
    asm volatile("" : "+v"(magic));
    for (; pos < end && b < p.c.B; ++b) {      // whatever the lengths are by now
    const Kv4Extent ext = kv4_extent(p.c, uniform_int(p.seen + b));
    const int tiles = ((ext.entries << bps) + 3) >> 2;
    if (tiles == 0) continue;
    const int t0 = pos - first, t1 = min(tiles, end - first);
    const bool whole_sequence = t0 == 0 && t1 == tiles;
    pos = first + t1;
    first += tiles;

    // ---- the column's query: its group's dimensions, as fp16 pieces
    h8_t qf[QP][NJ];
    float qsum = 0.f, kq;
    {
        float x[NJ][8], mx = 0.f;
        const T_ *qr = static_cast<const T_ *>(p.q) + ((size_t)b * p.Hq + head0 + min(jh, nj - 1)) * D;
#pragma unroll
        for (int jj = 0; jj < NJ; ++jj) load8(qr + 32 * jj + 8 * h, x[jj]);
#pragma unroll
        for (int jj = 0; jj < NJ; ++jj) {
            const bool mine = jj * 32 / GS == g && jh < nj;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!mine) x[jj][e] = 0.f;
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
        kq = fmaxf(p.scale / f, 0x1p-126f);    // a query of zeros: never 0, which times a hidden score is NaN
    }

    f4_t acc[NJ][2];
#pragma unroll
    for (int i = 0; i < NJ; ++i) acc[i][0] = acc[i][1] = f4_t{0.f, 0.f, 0.f, 0.f};
    // m: an integer no less than the largest score (log2), so that rescaling is
    // exact; f: the weights' power of two, which only falls
    float m = -INFINITY, l = 0.f, z = 0.f, f = kMostRange;
    bool far = false;            // of any column of the wave
    const int *bt = p.c.bt + (size_t)b * p.c.max_pages;
    int page[4], blk[4], held[4];
    auto read_pages = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < 4; ++x) page[x] = uniform_int(bt + min((4 * tile + x) >> bps, ext.entries - 1));
    };
    // The tile's four blocks in the pool and the tokens they hold.
    auto locate = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int i = 4 * tile + x, e = i >> bps, o = i & ((1 << bps) - 1);
            const bool ok = e < ext.entries && page[x] >= 0 && page[x] < p.c.num_pages;
            held[x] = ok ? min(max((e == ext.last ? ext.tail : 1 << p.c.pshift) - 16 * o, 0), 16) : 0;
            blk[x] = (((ok ? page[x] : 0) * p.c.Hkv + kvh) << bps) + o;
        }
    };
    auto pick = [&](const int (&v)[4], int x) __attribute__((always_inline)) {
        return x == 0 ? v[0] : x == 1 ? v[1] : x == 2 ? v[2] : v[3];
    };
    // K rows (of block n / 4) and steps (of block h) of the tile that locate() found.
    uint32_t kw[4][NJ];
    u4_t ksr[NI];
    auto load_k = [&]() __attribute__((always_inline)) {
        const uint8_t *kp = p.c.kc + (long)pick(blk, n >> 2) * (D * 8) + (n & 3) * (D / 2) + h * NJ * 4;
        const u4_t *ksp = reinterpret_cast<const u4_t *>(p.c.ks) + ((long)pick(blk, h) * G + g) * 4 + cp * NI;
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<NJ>(kp + 4 * i * (D / 2), kw[i]);
#pragma unroll
        for (int i = 0; i < NI; ++i) ksr[i] = ksp[i];
    };
    // A tile's V is loaded while its scores are computed, the next tile's K while
    // the weights are: both in flight without registers of their own.
    if (t0 + w < t1) {
        read_pages(t0 + w);
        locate(t0 + w);
        load_k();
        read_pages(t0 + w + kNW);
    }
    for (int tile = t0 + w; tile < t1; tile += kNW) {
        uint32_t vw[NJ][4];
        u4_t vsr[NI];
        const long vblk = pick(blk, h);
        const u4_t *vsp = reinterpret_cast<const u4_t *>(p.c.vs) + (vblk * G + g) * 4 + cp * NI;
        const uint8_t *vp = p.c.vc + vblk * (D * 8) + n * 16;
#pragma unroll
        for (int i = 0; i < NI; ++i) vsr[i] = vsp[i];
#pragma unroll
        for (int i = 0; i < NJ; ++i) load_words<4>(vp + i * 256, vw[i]);
        const int held_all = held[0] + held[1] + held[2] + held[3];
        const bool whole = held_all == 64;
        const int mine = pick(held, h) - 4 * NI * cp;     // of this copy's slots
        if (!whole) {           // what a slot without a token holds reaches nothing
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (4 * i + r >= mine) ksr[i][r] = 0, vsr[i][r] = 0;
        }
        // ---- scores of the copy's tokens of block h, for this lane's column
        float sc[NI][4], tmax = -INFINITY;
        h2_t smax = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int jj = 0; jj < NJ; ++jj) {
                const uint32_t v = kw[i][jj];
                const h8_t kf = join(codes_low<KMID>(v, magic), codes_high<KMID>(v, magic),
                                     codes_low<KMID>(v >> 8, magic), codes_high<KMID>(v >> 8, magic));
                if (QP > 1) a = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[QP - 1][jj], a, 0, 0, 0);
                a = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[0][jj], a, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[i % NI][r] = i < NI || i / NI == cp ? a[r] : sc[i % NI][r];
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const h2_t st = as_h2(ksr[i][r]);
                float v = group_sum<G>(fmaf(base<KMID>(st), qsum, (float)st[0] * sc[i][r]));
                if (!whole && 4 * i + r >= mine) v = -INFINITY;
                sc[i][r] = v;
                tmax = fmaxf(tmax, v);
                smax = __builtin_elementwise_max(smax, as_h2(vsr[i][r]));
            }
        }
        if (tile + kNW < t1) {
            locate(tile + kNW);
            load_k();
            read_pages(tile + 2 * kNW);
        }
        // ---- running maximum and the weights' power of two.  With a token held the
        // maximum is finite, also where all scores are -inf: a sum of 0 then tells
        // such a row, which is NaN, from one without tokens, which is 0.
        const bool any = held_all > 0;
        const float mn = fmaxf(fmaxf(m, any ? -FLT_MAX : -INFINITY), ceilf(quarters_max(tmax) * kq));
        const float fn = fminf(f, to_range(quarters_max((float)smax[0])));
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - ref);
        const float fa = alpha * (fn / f);
        m = mn;
        f = fn;
        // bf16 outputs: the weights' factor 2^k goes into the exponent, and l and z
        // carry it as the products do; the others multiply the steps, exactly
        const float e = WP == 1 ? (float)((int)(__float_as_uint(f) >> 23) - 127) : 0.f;
        float kw = kq, shift = e - ref;
        if (!__all(fa == 1.f)) {
            far = __any(fabsf(ref) > 0x1p20f);
            if (WP == 1)
#pragma unroll
                for (int i = 0; i < NJ; ++i) acc[i][0] *= fa, acc[i][1] *= fa;
            l *= WP == 1 ? fa : alpha;
            z *= WP == 1 ? fa : alpha;
        }
        // A weight is exp2(score kq - ref), the product not rounded.  From 2^24 on the
        // maximum is rounded by more than 1, and a weight could pass its type's range
        // (or all of them be 0): there the product is rounded as the maximum was.
        if (far) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = sc[i][r] * kq;
                    asm volatile("" : "+v"(x));
                    sc[i][r] = x - ref;
                }
            kw = 1.f;
            shift = e;
        }
        // where the outputs have fp16's or fp32's bits a tile's products get an
        // accumulator of their own, added to the sum so far in one rounding per
        // value (512 fp32 tokens per wave: 3.3e-7 off the exact sum, 4.3e-7 when
        // the matrix instructions add to the running sum themselves)
        f4_t part[WP == 1 ? 1 : NJ][2];
        if (WP > 1) {
#pragma unroll
            for (int i = 0; i < NJ; ++i) part[i][0] = part[i][1] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
        // ---- weights and the value product
        h4_t wt[WP][NI];
        auto weigh = [&](int i) __attribute__((always_inline)) {
            float wv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const h2_t st = as_h2(vsr[i][r]);
                const float pv = __builtin_amdgcn_exp2f(fmaf(sc[i][r], kw, shift));
                l += pv;
                z = fmaf(pv, base<true>(st), z);
                wv[r] = pv * (WP == 1 ? (float)st[0] : (float)st[0] * f);
                // rounded to fp32 here: the pieces below are of one value (the
                // compiler rounds the product to fp16 at once for one of them)
                if (WP > 1) asm volatile("" : "+v"(wv[r]));
            }
            // token order of a mask with 0x000f000f: 0, 2, then 1, 3
            constexpr int order[4] = {0, 2, 1, 3};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const _Float16 a = (_Float16)wv[order[e]];
                wt[0][i][e] = a;
                if (WP > 1) wt[WP - 1][i][e] = (_Float16)(wv[order[e]] - (float)a);
            }
        };
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            h8_t wf[WP];
#pragma unroll
            for (int y = 0; y < 2; ++y)
                if (2 * u + y < NI) weigh(2 * u + y);
#pragma unroll
            for (int x = 0; x < WP; ++x) {
                const int i = 2 * u;                 // slots of other copies: no weight
                const u32x2_t none = {0, 0};
                const u32x2_t a = __builtin_bit_cast(u32x2_t, wt[x][i % NI]);
                const u32x2_t c = __builtin_bit_cast(u32x2_t, wt[x][(i + 1) % NI]);
                const u32x2_t ma = C == 1 || i / NI == cp ? a : none, mc = C == 1 || (i + 1) / NI == cp ? c : none;
                wf[x] = __builtin_bit_cast(h8_t, u4_t{ma[0], ma[1], mc[0], mc[1]});
            }
#pragma unroll
            for (int i = 0; i < NJ; ++i) {
                const uint32_t a = vw[i][2 * u], c = vw[i][2 * u + 1];
                const h8_t ev = join(codes_low<true>(a, magic), codes_low<true>(a >> 8, magic),
                                     codes_low<true>(c, magic), codes_low<true>(c >> 8, magic));
                const h8_t od = join(codes_high<true>(a, magic), codes_high<true>(a >> 8, magic),
                                     codes_high<true>(c, magic), codes_high<true>(c >> 8, magic));
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

    // ---- the waves' passes joined
    if (jh < nj) {
        const float inv = 1.f / f;
#pragma unroll
        for (int i = 0; i < NJ; ++i)
            if (i * 32 / GS == g)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        so[w][j][32 * i + 2 * (4 * h + r) + e] =
                            WP == 1 ? (acc[i][e][r] + z) * inv : fmaf(acc[i][e][r], inv, z);
        if (g == 0 && h == 0) sm[w][j][0] = m, sm[w][j][1] = WP == 1 ? l * inv : l;
    }
    __syncthreads();
    for (int x = tid; x < nj * D; x += kNT) {
        const int jj = x / D, d = x % D;
        float mm = -INFINITY;
#pragma unroll
        for (int k = 0; k < kNW * C; ++k) mm = fmaxf(mm, sm[k / C][k % C * HE + jj][0]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        float o = 0.f, ll = 0.f;
#pragma unroll
        for (int k = 0; k < kNW * C; ++k) {
            const int col = k % C * HE + jj;
            const float a = __builtin_amdgcn_exp2f(sm[k / C][col][0] - ref);
            o = fmaf(a, so[k / C][col][d], o);
            ll = fmaf(a, sm[k / C][col][1], ll);
        }
        if (whole_sequence) {
            store_act(static_cast<T_ *>(p.out), ((size_t)b * p.Hq + head0 + jj) * D + d, kv4_out(o, ll, mm));
        } else {
            const size_t row = (size_t)(blockIdx.x + b) * p.Hq + head0 + jj;
            p.part_o[row * D + d] = o;
            if (d == 0) {
                p.part_ml[2 * row] = mm;
                p.part_ml[2 * row + 1] = ll;
            }
        }
    }
    __syncthreads();                           // so and sm are free for the next sequence
    }
}

// One workgroup per (query head, sequence).  A sequence cut by runs: thread
// (four dims, group of slots) adds every SG-th slot's output times its weight,
// kPre of them loaded before the weights are known.
template <typename T, int D>
__global__ __launch_bounds__(kNT) void kv4_merge_kernel(Kv4DecodeParams p) {
    constexpr int DQ = D / 4, SG = kNT / DQ, kPre = 4;
    __shared__ float ws[kNT], wm[kNW], wl[kNW];
    __shared__ float4 os[SG][DQ];
    const int head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int d = tid % DQ, sg = tid / DQ;
    int first, tiles;
    const Runs runs(kv4_all_tiles(p.c, p.seen, b, &first, &tiles), p.W);
    T *out = static_cast<T *>(p.out) + ((size_t)b * p.Hq + head) * D;
    if (tiles == 0) {
        if (tid < DQ)
#pragma unroll
            for (int e = 0; e < 4; ++e) store_act(out, 4 * d + e, 0.f);
        return;
    }
    const int i0 = runs.of(first), used = runs.of(first + tiles - 1) - i0 + 1;
    if (used == 1) return;                               // written whole
    const size_t row0 = (size_t)(i0 + b) * p.Hq + head;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + row0;
    const float4 *po = reinterpret_cast<const float4 *>(p.part_o) + row0 * DQ + d;
    const size_t step = (size_t)p.Hq * DQ;
    float4 pre[kPre];
#pragma unroll
    for (int u = 0; u < kPre; ++u) pre[u] = po[step * min(sg + u * SG, used - 1)];
    float m = -INFINITY;
    for (int s = tid; s < used; s += kNT) m = fmaxf(m, ml[(size_t)s * p.Hq].x);
    m = wave_max_f(m);
    if ((tid & 63) == 0) wm[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kNW; ++k) m = fmaxf(m, wm[k]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, const float4 &x) __attribute__((always_inline)) {
        o.x = fmaf(w, x.x, o.x), o.y = fmaf(w, x.y, o.y), o.z = fmaf(w, x.z, o.z), o.w = fmaf(w, x.w, o.w);
    };
    for (int s0 = 0; s0 < used; s0 += kNT) {             // kNT slots' weights at a time
        const int s = s0 + tid, n = min(kNT, used - s0);
        float w = 0.f;
        if (s < used) {
            const float2 x = ml[(size_t)s * p.Hq];
            w = __builtin_amdgcn_exp2f(x.x - ref);
            l = fmaf(w, x.y, l);
        }
        __syncthreads();
        ws[tid] = w;
        __syncthreads();
        int k = sg;
        if (s0 == 0) {
#pragma unroll
            for (int u = 0; u < kPre; ++u)
                if (sg + u * SG < n) add(ws[sg + u * SG], pre[u]);
            k += kPre * SG;
        }
        for (; k < n; k += kPre * SG) {
            float4 x[kPre];
#pragma unroll
            for (int u = 0; u < kPre; ++u) x[u] = po[step * min(s0 + k + u * SG, used - 1)];
#pragma unroll
            for (int u = 0; u < kPre; ++u)
                if (k + u * SG < n) add(ws[k + u * SG], x[u]);
        }
    }
    l = wave_sum_f(l);
    if ((tid & 63) == 0) wl[tid >> 6] = l;
    os[sg][d] = o;
    __syncthreads();
    if (tid >= D) return;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < kNW; ++k) l += wl[k];
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < SG; ++k) v += reinterpret_cast<const float *>(os[k])[tid];
    store_act(out, tid, kv4_out(v, l, m));
}

namespace {
// Copies of the columns, kernel us with one and with four: 64 sequences of 3000 bf16
// tokens, 16 / 16 heads of 64 (G = 1) 68.6, 52.7; 32 / 8 of 64 (G = 1) 35.5, 28.5; 16 /
// 8 of 128 (G = 2) 45.1, 40.5; one sequence of 500 5.5 to 7.1 either way.  With more
// heads than a quarter of the columns four copies would pass over the cache twice.
int decode_copies(int R, int D, int GS) { return 4 * R <= 16 / (D / GS) ? 4 : 1; }
int decode_heads_per_slice(int R, int D, int GS) { return 16 / (D / GS) / decode_copies(R, D, GS); }

// Runs W: two workgroups per CU over the whole call, no more than there can be tiles.
// A call of 64 sequences of 192000 bf16 tokens in all, 32 / 8 heads of 128, with one,
// two, three and four: 77, 65, 71 and 73 us; 131072 of one sequence 42, 38, 42, 44.
int decode_runs(const OjasxKV4Cache *c, int Hq, int max_seen) {
    const int R = Hq / c->num_kv_heads, HS = decode_heads_per_slice(R, c->head_dim, c->group_size);
    const long groups = (long)c->num_kv_heads * ((R + HS - 1) / HS);
    const long cap = (long)c->max_pages * c->page_size;
    const long slots = max_seen > 0 ? std::min((long)max_seen, cap) : cap;
    const long tiles = (slots + 63) / 64 * c->num_sequences;
    return (int)std::max(1L, std::min((512 + groups - 1) / groups, tiles));
}

int decode_check(const OjasxKV4Cache *c, int Hq) {
    const long tiles = ((long)c->max_pages * c->page_size + 63) / 64 * c->num_sequences;
    if (Hq <= 0 || Hq > 65535 || Hq % c->num_kv_heads || c->num_sequences > 65535 || tiles > 0x3fffffffL) {
        set_error("4-bit KV decode: %d query heads for %d kv heads, %d sequences (at most 65535) of up to %d pages "
                  "(2^36 tokens in all)", Hq, c->num_kv_heads, c->num_sequences, c->max_pages);
        return OJASX_ERR_INVALID;
    }
    return OJASX_OK;
}

template <typename T>
int launch_decode(const Kv4DecodeParams &p, int D, int GS, hipStream_t st) {
    const int HS = decode_heads_per_slice(p.R, D, GS);
    const dim3 grid(p.W, p.c.Hkv * ((p.R + HS - 1) / HS));
    const bool copies = decode_copies(p.R, D, GS) > 1;
#define OJX_KV4_DECODE(D_, GS_)                                                                            \
    if (D == D_ && GS == GS_) {                                                                            \
        if constexpr (D_ / GS_ <= 4)                                                                       \
            if (copies) OJX_LAUNCH((kv4_decode_kernel<T, D_, GS_, 4>), grid, dim3(kNT), 0, st, p);         \
        if (!copies) OJX_LAUNCH((kv4_decode_kernel<T, D_, GS_, 1>), grid, dim3(kNT), 0, st, p);            \
    }
    OJX_KV4_DECODE(64, 32)
    OJX_KV4_DECODE(64, 64)
    OJX_KV4_DECODE(128, 32)
    OJX_KV4_DECODE(128, 64)
    OJX_KV4_DECODE(128, 128)
    OJX_KV4_DECODE(256, 32)
    OJX_KV4_DECODE(256, 64)
    OJX_KV4_DECODE(256, 128)
#undef OJX_KV4_DECODE
    const dim3 rows(p.Hq, p.c.B);
    if (D == 64) OJX_LAUNCH((kv4_merge_kernel<T, 64>), rows, dim3(kNT), 0, st, p);
    else if (D == 128) OJX_LAUNCH((kv4_merge_kernel<T, 128>), rows, dim3(kNT), 0, st, p);
    else OJX_LAUNCH((kv4_merge_kernel<T, 256>), rows, dim3(kNT), 0, st, p);
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
    return ((long)decode_runs(cache, num_q_heads, max_seen) + cache->num_sequences) * num_q_heads *
           (cache->head_dim + 2) * (long)sizeof(float);
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
    if (reinterpret_cast<uintptr_t>(q) & 15) {
        set_error("4-bit KV decode: q is 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    const int D = cache->head_dim;
    p.scale = (scale_factor > 0.f ? scale_factor : 1.0f / sqrtf((float)D)) * kLog2e;
    if (std::isnan(scale_factor) || !std::isfinite(p.scale)) {
        set_error("4-bit KV decode: scale_factor %g is not finite (times log2(e), in fp32)", (double)scale_factor);
        return OJASX_ERR_INVALID;
    }
    p.W = decode_runs(cache, num_q_heads, max_seen);
    const size_t rows = ((size_t)p.W + cache->num_sequences) * num_q_heads;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < (long)(rows * (D + 2) * sizeof(float))) {
        set_error("4-bit KV decode: workspace of %ld bytes at %p (ojasx_kv4_decode_workspace; 16-byte aligned)",
                  workspace_bytes, workspace);
        return OJASX_ERR_INVALID;
    }
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = p.part_o + rows * D;
    p.q = q, p.out = out, p.seen = seen, p.Hq = num_q_heads, p.R = num_q_heads / cache->num_kv_heads;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == OJASX_DTYPE_F32    ? launch_decode<float>(p, D, cache->group_size, st)
           : dtype == OJASX_DTYPE_BF16 ? launch_decode<__hip_bfloat16>(p, D, cache->group_size, st)
                                       : launch_decode<__half>(p, D, cache->group_size, st);
}

}  // extern "C"
