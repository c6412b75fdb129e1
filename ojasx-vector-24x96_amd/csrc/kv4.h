// kv4.h -- the 4-bit paged KV cache's format, shared by its write side
// (kv4_append.hip) and its attention (kv4_decode.hip).
//
// Of a token's K or V row of one kv head (D values, fp32), each group of GS
// consecutive dimensions is held as lo = fp16(min), s = fp16(fp32((max - lo) /
// 15)), at least 0, and codes c_d = clamp(round_half_even((x_d - lo) / s), 0,
// 15), for the values lo + s c_d.  s = 0 holds codes 0.  lo and s saturate at
// +-65504; a group with an infinity or a NaN holds s = lo = NaN.
//
// A block is 16 slots of a page; block b of a page and kv head holds
//   K codes  [16 slots][D / 2 bytes]: a row is 4-byte words, word h (D / 32) +
//            j the 8 dimensions 32 j + 8 h .. + 7: the code of dimension 2 i
//            of them in bits 4 i, of 2 i + 1 in bits 16 + 4 i (the pairs that a
//            mask with 0x000f000f leaves are neighbours);
//   V codes  [D / 2 pairs][16 slots], byte = dimension 2 i in the low four
//            bits, 2 i + 1 in the high ones;
//   steps    [D / GS][16 slots] fp16 pairs (s, lo), K and V alike;
// blocks in the order [page][kv head][block of the page].
//
// Position t of a sequence lies in its page j = t / P; the first `sink` pages
// stay, the others take turns: entry e = j < sink ? j : sink + (j - sink) mod
// (max_pages - sink) of the sequence's row of the block table.
#pragma once

#include "common.h"

namespace ojx {

struct Kv4View {
    uint8_t *kc, *vc;
    __half2 *ks, *vs;
    const int *bt;              // [B][max_pages]
    const double *turns;        // [rot / 2] or null
    int B, max_pages, sink, pshift, num_pages;   // page = 1 << pshift slots
    int Hkv, rot, interleaved;
};

int kv4_view(const OjasxKV4Cache *c, Kv4View *v);   // 0 or an error code

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u4_t __attribute__((ext_vector_type(4)));

// Eight consecutive values as fp32 (16-byte aligned).
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const f4_t a = *reinterpret_cast<const f4_t *>(p), b = *reinterpret_cast<const f4_t *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
__device__ __forceinline__ void load8(const __hip_bfloat16 *p, float (&x)[8]) {
    const u4_t a = *reinterpret_cast<const u4_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(a[i] << 16);
        x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 a = *reinterpret_cast<const h8 *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
}

__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<f4_t *>(p) = f4_t{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f4_t *>(p + 4) = f4_t{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(__hip_bfloat16 *p, const float (&x)[8]) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    b8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (__bf16)x[i];
    *reinterpret_cast<b8 *>(p) = a;
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    h8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];
    *reinterpret_cast<h8 *>(p) = a;
}

// The angles of position pos, as the factors of a lane's dimensions d0 .. d0 + 7: x_e <-
// x_e co[e] + (the value it turns with) sn[e].  turns: frequencies / (2 pi) of the `half` =
// rotary_dim / 2 pairs.  Whole waves call it, each with `half` entries of LDS of its own.
__device__ __forceinline__ void token_angles(const double *turns, int half, bool interleaved, int pos, int d0,
                                             double2 *cs, double (&co)[8], double (&sn)[8]) {
    for (int i = threadIdx.x & 63; i < half; i += 64) {
        const double f = turns[i], t = (double)pos * f;
        const double frac = (t - rint(t)) + fma((double)pos, f, -t);
        double s, c;
        sincospi(2.0 * frac, &s, &c);
        cs[i] = make_double2(c, s);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool rotates = d0 < 2 * half, low = d0 < half;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = interleaved ? (d0 + e) / 2 : low ? d0 + e : d0 - half + e;
        const double2 a = rotates ? cs[i] : make_double2(1.0, 0.0);
        co[e] = a.x;
        sn[e] = (interleaved ? e % 2 == 0 : low) ? -a.y : a.y;
    }
}

// Entry of the block table that holds page j of a sequence.
__device__ __forceinline__ int kv4_entry(const Kv4View &c, int j) {
    return j < c.sink ? j : c.sink + (j - c.sink) % (c.max_pages - c.sink);
}

// First page after the sink ones that a sequence of `seen` tokens still holds.
__device__ __forceinline__ int kv4_first_page(const Kv4View &c, int seen) {
    const int opened = (int)(((long)seen + (1 << c.pshift) - 1) >> c.pshift);
    return opened - (c.max_pages - c.sink);
}

// The block that position t of sequence b lies in, in whole-pool block order,
// or -1: a position before the first, of a page that a sequence of `seen`
// tokens no longer holds, or of a page the block table does not map.
__device__ __forceinline__ long kv4_block(const Kv4View &c, int b, int t, int seen, int h) {
    if (t < 0) return -1;
    const int j = t >> c.pshift;
    if (j >= c.sink && j < kv4_first_page(c, seen)) return -1;
    const int page = c.bt[(long)b * c.max_pages + kv4_entry(c, j)];
    if (page < 0 || page >= c.num_pages) return -1;
    return ((((long)page * c.Hkv + h) << c.pshift) + (t & ((1 << c.pshift) - 1))) >> 4;
}

// Where row n of a packed batch lies: its sequence b (-1: of none), the token's
// position and the tokens of the sequence after the batch.  Sequence b owns rows
// cu[b] .. cu[b + 1] - 1 at positions start[b] ..; without cu row n is sequence
// n's one token.  Whole waves call it with one n.
struct Kv4Row {
    int b, pos, seen;
};
__device__ __forceinline__ Kv4Row kv4_row(const int *cu, const int *start, int B, int n) {
    if (!cu) {
        const int s = start[n];
        return {n, s, s + 1};
    }
    const int lane = threadIdx.x & 63;
    if (B < 64) {                // both lists in one load each, the entries by lane
        const int c = cu[min(lane, B)], s = start[min(lane, B - 1)];
        const int b = __popcll(__ballot(lane <= B && c <= n)) - 1;
        if (b < 0 || b >= B) return {-1, 0, 0};
        const int first = __builtin_amdgcn_readlane(c, b), s0 = __builtin_amdgcn_readlane(s, b);
        return {b, s0 + (n - first), s0 + (__builtin_amdgcn_readlane(c, b + 1) - first)};
    }
    int count = 0;
    for (int i0 = 0; i0 <= B; i0 += 64) {
        const int i = i0 + lane;
        count += __popcll(__ballot(i <= B && cu[min(i, B)] <= n));
    }
    const int b = count - 1;
    if (b < 0 || b >= B) return {-1, 0, 0};
    const int first = cu[b], s0 = start[b];
    return {b, s0 + (n - first), s0 + (cu[b + 1] - first)};
}

}  // namespace ojx
