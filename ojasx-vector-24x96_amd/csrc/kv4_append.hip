// kv4_append.hip -- the write side of the 4-bit paged KV cache (format: kv4.h):
// rotation of queries and keys by their positions, encoding of keys and values
// into the pages, and reading tokens back.
//
// Rotation: dimensions (i, i + rot / 2), or (2 i, 2 i + 1) interleaved, turn by
// the angle pos inv_freq[i].  The angle is held in turns, pos (inv_freq / 2 pi),
// as an fp64 product and its rounding error, so that taking the whole turns
// away leaves 2^-53 of the frequency's own rounding at any position (fp32
// angles are off by 0.004 at position 65536).  (x, y) -> (x c - y s, y c + x s)
// runs in fp64 with one rounding to fp32: the codes then follow from the
// format's definition, and do not depend on how a product was rounded.
//
// Bound by memory and, for 16-bit rows, about as much by vector instructions (they
// issue in half of the cycles; the rotation is fp64).  8192 tokens, 32 / 8 heads of
// 128, queries rotated along: bf16 45 to 49 us for 178 MB, 3.8 TB/s, fp32 88 us for
// 346 MB, 3.9 TB/s (a copy runs at 4.9 here).  One token: 4 us, a launch and three
// loads that wait for each other.  Reading the 8192 tokens back as bf16: 15 us for
// 44 MB (a lane loads its values' codes byte by byte).
#include "kv4.h"

namespace ojx {

namespace {
constexpr int kNT = 256;

struct Kv4AppendParams {
    Kv4View c;
    const void *q, *k, *v;
    long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;    // token and head strides, elements
    void *q_out, *k_out;                        // contiguous [n][heads][D]
    const int *start, *cu;
    int n, Hq, parts;
};

// Minimum, maximum and sum over the LANES (4, 8 or 16) lanes of a group.
template <int LANES>
__device__ __forceinline__ void group_stats(float &mn, float &mx, float &sum) {
#define OJX_GROUP_STEP(CTRL)                                          \
    mn = fminf(mn, __int_as_float(dpp_i<CTRL>(__float_as_int(mn)))); \
    mx = fmaxf(mx, __int_as_float(dpp_i<CTRL>(__float_as_int(mx)))); \
    sum += __int_as_float(dpp_i<CTRL>(__float_as_int(sum)));
    OJX_GROUP_STEP(0xB1)
    OJX_GROUP_STEP(0x4E)
    if (LANES > 4) { OJX_GROUP_STEP(0x141) }
    if (LANES > 8) { OJX_GROUP_STEP(0x140) }
#undef OJX_GROUP_STEP
}

// fp16 of a float, rounded to nearest even.  The value passes through a
// register the compiler cannot see behind: it would round the fp64 expression
// it came from to fp16 at once, where the format rounds to fp32 first.
__device__ __forceinline__ _Float16 to_half(float f) {
    asm volatile("" : "+v"(f));
    return (_Float16)f;
}

// fp32 of x / 15: the product with the double nearest 1 / 15, corrected by its
// remainder, is the quotient to a double's last place (a full fp64 division
// takes three times the instructions).
__device__ __forceinline__ float div15(double x) {
    constexpr double r = 1.0 / 15.0;
    const double q = x * r;
    return (float)fma(fma(-15.0, q, x), r, q);
}

// Encodes a lane's eight dimensions of a K (V) row into block `blk`, slot t.
// unit: which eight of the row's D / 8.
template <int D, int GS>
__device__ __forceinline__ void encode_unit(const float (&x)[8], bool value, int unit, long blk, int t,
                                            uint8_t *codes, __half2 *steps) {
    float mn = x[0], mx = x[0], poison = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        poison = fmaf(x[i], 0.f, poison);       // NaN from an infinity or a NaN, else 0
    }
    group_stats<GS / 8>(mn, mx, poison);
    const _Float16 lo = to_half(fminf(fmaxf(mn, -65504.f), 65504.f) + poison);
    const float step = div15((double)mx - (double)(float)lo);
    // lo may have been rounded above max: no step below 0
    const _Float16 s = to_half(fminf(fmaxf(step, 0.f), 65504.f) + poison);
    const float lo32 = (float)lo, s32 = (float)s, inv = s32 > 0.f ? 1.0f / s32 : 0.f;
    // An fp32 quotient is off by less than 2^-18: only beside a half can it round
    // another way than the exact one, whose remainder decides there.
    float near[8];
    bool beside = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = (x[i] - lo32) * inv;
        near[i] = rintf(f);
        beside |= fabsf(f - near[i]) > 0.4999f;
    }
    if (beside && s32 > 0.f) {
        const double half = 0.5 * (double)s32;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double e = fma(-(double)near[i], (double)s32, (double)x[i] - (double)lo32);
            const bool odd = fabsf(near[i]) < 16.f && ((int)near[i] & 1) != 0;
            if (e > half || (e == half && odd)) near[i] += 1.f;
            else if (e < -half || (e == -half && odd)) near[i] -= 1.f;
        }
    }
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) code[i] = (uint32_t)fminf(fmaxf(near[i], 0.f), 15.f);   // NaN: 0
    if (blk < 0) return;
    if (!value) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= code[2 * i] << (4 * i) | code[2 * i + 1] << (16 + 4 * i);
        const int word = (unit & 3) * (D / 32) + (unit >> 2);
        reinterpret_cast<uint32_t *>(codes + blk * (D * 8) + t * (D / 2))[word] = w;
    } else {
        uint8_t *dst = codes + blk * (D * 8) + unit * 64 + t;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[16 * i] = (uint8_t)(code[2 * i] | code[2 * i + 1] << 4);
    }
    if (unit % (GS / 8) == 0) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        reinterpret_cast<h2 *>(steps)[(blk * (D / GS) + unit / (GS / 8)) * 16 + t] = h2{s, lo};
    }
}
}  // namespace

// Waves: wave i of the launch takes token i / parts and every parts-th 64 units of
// eight dimensions of its query, key and value rows.  It computes the token's
// angles itself (a lane per pair), so waves need no barrier.  64 units are whole
// rows: a lane's dimensions are the same in all of them, and its eight angles stay
// in registers (read from LDS for every unit they cost more than the rest).
// kAtOnce units' loads are in flight together.
constexpr int kAtOnce = 3;

template <typename T, int D, int GS>
__global__ __launch_bounds__(kNT) void kv4_append_kernel(Kv4AppendParams p) {
    __shared__ double2 angles[kNT / 64][D / 2];  // cos and sin of the token's angles
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int UPR = D / 8, RPW = 64 / UPR;   // units of eight per row, rows per 64 units
    const int wave = blockIdx.x * (kNT / 64) + w, n = wave / p.parts, part = wave - n * p.parts;
    if (n >= p.n) return;
    const int Hkv = p.c.Hkv, rows = p.Hq + 2 * Hkv, step = p.parts * RPW;
    const int half = p.c.rot >> 1, d0 = lane % UPR * 8, unit = lane % UPR;
    const bool turns = d0 < p.c.rot, low = d0 < half;
    const int other = !turns || p.c.interleaved ? 0 : low ? half : -half;   // where the values lie they turn with
    const Kv4Row r = kv4_row(p.cu, p.start, p.c.B, n);
    // the token's block of kv head 0; head h's is h pages of blocks further
    const long blk0 = r.b < 0 ? -1 : kv4_block(p.c, r.b, r.pos, r.seen, 0);
    double2 *cs = angles[w];
    double co[8], sn[8];                         // x_e <- x_e co + (its other) sn
    token_angles(p.c.turns, half, p.c.interleaved, r.pos, d0, cs, co, sn);
    for (int row0 = part * RPW + lane / UPR; row0 - lane / UPR < rows; row0 += kAtOnce * step) {
        float x[kAtOnce][8], y[kAtOnce][8];
        // past the last row: row 0's values, not used
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = row0 + i * step < rows ? row0 + i * step : 0;
            const bool isq = row < p.Hq, isv = row >= p.Hq + Hkv;
            const T *src = d0 + (isq ? static_cast<const T *>(p.q) + n * p.q_ts + row * p.q_hs
                                 : isv ? static_cast<const T *>(p.v) + n * p.v_ts + (row - p.Hq - Hkv) * p.v_hs
                                       : static_cast<const T *>(p.k) + n * p.k_ts + (row - p.Hq) * p.k_hs);
            load8(src, x[i]);
            load8(src + other, y[i]);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = row0 + i * step;
            if (row >= rows) continue;
            const bool isq = row < p.Hq, isv = row >= p.Hq + Hkv;
            const int head = isq ? row : isv ? row - p.Hq - Hkv : row - p.Hq;
            T *out = isq ? static_cast<T *>(p.q_out) : isv ? nullptr : static_cast<T *>(p.k_out);
            if (out) out += ((size_t)n * (isq ? p.Hq : Hkv) + head) * D + d0;
            if (r.b < 0) {                           // a row of no sequence
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
                if (out) store8(out, x[i]);
                continue;
            }
            if (turns && !isv) {
                if (p.c.interleaved)
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] = x[i][e ^ 1];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = (float)fma((double)x[i][e], co[e], (double)y[i][e] * sn[e]);
            }
            if (out) store8(out, x[i]);
            if (!isq) {
                const long blk = blk0 < 0 ? -1 : blk0 + ((long)head << (p.c.pshift - 4));
                encode_unit<D, GS>(x[i], isv, unit, blk, r.pos & 15, isv ? p.c.vc : p.c.kc, isv ? p.c.vs : p.c.ks);
            }
        }
    }
}

struct Kv4ReadParams {
    Kv4View c;
    const int *start, *cu, *seen;
    void *k_out, *v_out;        // contiguous [n][Hkv][D]
    int n, parts;
};

// The appended tokens' values: waves as in kv4_append_kernel.
template <typename T, int D, int GS>
__global__ __launch_bounds__(kNT) void kv4_read_kernel(Kv4ReadParams p) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int UPR = D / 8;
    const int wave = blockIdx.x * (kNT / 64) + w, n = wave / p.parts, part = wave - n * p.parts;
    if (n >= p.n) return;
    Kv4Row r = kv4_row(p.cu, p.start, p.c.B, n);
    if (p.seen && r.b >= 0) r.seen = p.seen[r.b];
    const int Hkv = p.c.Hkv, units = 2 * Hkv * UPR, t = r.pos & 15;
    // the token's block of kv head 0; head h's is h pages of blocks further
    const long blk0 = r.b < 0 || r.pos >= r.seen ? -1 : kv4_block(p.c, r.b, r.pos, r.seen, 0);
    for (int u = part * 64 + lane; u < units; u += p.parts * 64) {
        const int row = u / UPR, unit = u % UPR;
        const bool isv = row >= Hkv;
        const int head = isv ? row - Hkv : row;
        const long blk = blk0 + ((long)head << (p.c.pshift - 4));
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (blk0 >= 0) {
            const __half2 st = (isv ? p.c.vs : p.c.ks)[(blk * (D / GS) + unit / (GS / 8)) * 16 + t];
            const float s = __low2float(st), lo = __high2float(st);
            if (!isv) {
                const int word = (unit & 3) * (D / 32) + (unit >> 2);
                const uint32_t c =
                    reinterpret_cast<const uint32_t *>(p.c.kc + blk * (D * 8) + t * (D / 2))[word];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = fmaf(s, (float)(c >> (4 * i) & 15u), lo);
                    x[2 * i + 1] = fmaf(s, (float)(c >> (16 + 4 * i) & 15u), lo);
                }
            } else {
                const uint8_t *src = p.c.vc + blk * (D * 8) + unit * 64 + t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t c = src[16 * i];
                    x[2 * i] = fmaf(s, (float)(c & 15u), lo);
                    x[2 * i + 1] = fmaf(s, (float)(c >> 4), lo);
                }
            }
        }
        store8(static_cast<T *>(isv ? p.v_out : p.k_out) + ((size_t)n * Hkv + head) * D + unit * 8, x);
    }
}

int kv4_view(const OjasxKV4Cache *c, Kv4View *v) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_steps || !c->v_steps || !c->block_table) {
        set_error("4-bit KV cache: a NULL buffer");
        return OJASX_ERR_NULL;
    }
    const int D = c->head_dim, GS = c->group_size;
    if ((D != 64 && D != 128 && D != 256) || (GS != 32 && GS != 64 && GS != 128) || GS > D) {
        set_error("4-bit KV cache: head_dim %d, group_size %d (64, 128 or 256; 32, 64 or 128 and at most "
                  "head_dim)", D, GS);
        return OJASX_ERR_INVALID;
    }
    const int P = c->page_size;
    if (P < 16 || P > 32768 || (P & (P - 1))) {
        set_error("4-bit KV cache: page_size %d is no power of two from 16 to 32768", P);
        return OJASX_ERR_INVALID;
    }
    if (c->num_sequences <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535 || c->num_pages <= 0 ||
        c->sink_pages < 0 || c->max_pages <= c->sink_pages) {
        set_error("4-bit KV cache: %d sequences, %d kv heads, %d pages, %d of a sequence with %d sink pages",
                  c->num_sequences, c->num_kv_heads, c->num_pages, c->max_pages, c->sink_pages);
        return OJASX_ERR_INVALID;
    }
    if ((long)c->num_pages * c->num_kv_heads * (P / 16) > 0x7fffffffL) {
        set_error("4-bit KV cache: %d pages of %d slots for %d heads are more than 2^31 blocks of 16", c->num_pages,
                  P, c->num_kv_heads);
        return OJASX_ERR_INVALID;
    }
    if (c->rotary_dim < 0 || c->rotary_dim > D || c->rotary_dim % 16 || (c->rotary_dim && !c->turns)) {
        set_error("4-bit KV cache: rotary_dim %d (a multiple of 16 up to %d, with turns)", c->rotary_dim, D);
        return OJASX_ERR_INVALID;
    }
    if ((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes) |
         reinterpret_cast<uintptr_t>(c->k_steps) | reinterpret_cast<uintptr_t>(c->v_steps)) & 15) {
        set_error("4-bit KV cache: codes and steps are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    v->kc = c->k_codes;
    v->vc = c->v_codes;
    v->ks = static_cast<__half2 *>(c->k_steps);
    v->vs = static_cast<__half2 *>(c->v_steps);
    v->bt = c->block_table;
    v->turns = c->turns;
    v->B = c->num_sequences;
    v->max_pages = c->max_pages;
    v->sink = c->sink_pages;
    v->pshift = __builtin_ctz((unsigned)P);
    v->num_pages = c->num_pages;
    v->Hkv = c->num_kv_heads;
    v->rot = c->rotary_dim;
    v->interleaved = c->interleaved != 0;
    return OJASX_OK;
}

namespace {
// Waves per token: one for each 64 units while the launch is small, one in all when
// that makes 4096 waves (16 a CU): more of them compute the same angles again.
// Append, bf16, 32 / 8 heads of 128, us with one wave a token, by this rule, and
// with a wave for each 64 units: 64 tokens 11.8, 5.5, 5.7; 2048 tokens 18.7, 17.4,
// 29.8; 8192 tokens 44.6, 44.6, 97.6.
int wave_parts(int n, long units) {
    const long most = (units + 63) / 64, want = 4096 / n;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}
// Tokens of a launch: a grid has fewer than 2^32 threads.
constexpr int kMostTokens = 1 << 25;
unsigned wave_groups(int n, int parts) { return (unsigned)(((long)n * parts + kNT / 64 - 1) / (kNT / 64)); }

// The (element type, head_dim, group_size) instances of a kernel.
#define OJX_KV4_DISPATCH(KERNEL, T, D, GS, ...)                                               \
    do {                                                                                      \
        if (D == 64 && GS == 32) OJX_LAUNCH((KERNEL<T, 64, 32>), __VA_ARGS__);                \
        else if (D == 64) OJX_LAUNCH((KERNEL<T, 64, 64>), __VA_ARGS__);                       \
        else if (D == 128 && GS == 32) OJX_LAUNCH((KERNEL<T, 128, 32>), __VA_ARGS__);         \
        else if (D == 128 && GS == 64) OJX_LAUNCH((KERNEL<T, 128, 64>), __VA_ARGS__);         \
        else if (D == 128) OJX_LAUNCH((KERNEL<T, 128, 128>), __VA_ARGS__);                    \
        else if (GS == 32) OJX_LAUNCH((KERNEL<T, 256, 32>), __VA_ARGS__);                     \
        else if (GS == 64) OJX_LAUNCH((KERNEL<T, 256, 64>), __VA_ARGS__);                     \
        else OJX_LAUNCH((KERNEL<T, 256, 128>), __VA_ARGS__);                                  \
    } while (0)

#define OJX_KV4_DISPATCH_T(KERNEL, dtype, D, GS, ...)                                         \
    do {                                                                                      \
        if (dtype == OJASX_DTYPE_F32) OJX_KV4_DISPATCH(KERNEL, float, D, GS, __VA_ARGS__);    \
        else if (dtype == OJASX_DTYPE_BF16)                                                   \
            OJX_KV4_DISPATCH(KERNEL, __hip_bfloat16, D, GS, __VA_ARGS__);                     \
        else OJX_KV4_DISPATCH(KERNEL, __half, D, GS, __VA_ARGS__);                            \
    } while (0)
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API int ojasx_kv4_append_device(const OjasxKV4Cache *cache, const void *q, long q_token_stride,
                                      long q_head_stride, int num_q_heads, void *q_out, const void *k,
                                      long k_token_stride, long k_head_stride, void *k_out, const void *v,
                                      long v_token_stride, long v_head_stride, int num_tokens, int dtype,
                                      const int *start, const int *cu_seqlens, void *stream) {
    using namespace ojx;
    Kv4AppendParams p{};
    int rc = kv4_view(cache, &p.c);
    if (rc) return rc;
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    if (num_tokens < 0 || num_tokens > kMostTokens || num_q_heads < 0 || num_q_heads > 65535 ||
        (!cu_seqlens && num_tokens != cache->num_sequences)) {
        set_error("4-bit KV append: %d tokens (at most 2^25), %d query heads (without cu_seqlens one token for "
                  "each of the %d sequences)", num_tokens, num_q_heads, cache->num_sequences);
        return OJASX_ERR_INVALID;
    }
    if (num_tokens == 0) return OJASX_OK;
    if (!k || !v || !start || (num_q_heads && (!q || !q_out))) return OJASX_ERR_NULL;
    const size_t es = dtype == OJASX_DTYPE_F32 ? 4 : 2;
    if (!rows_of_16(k, k_token_stride, k_head_stride, es) || !rows_of_16(v, v_token_stride, v_head_stride, es) ||
        (num_q_heads && (!rows_of_16(q, q_token_stride, q_head_stride, es) || !rows_of_16(q_out, 0, 0, es))) ||
        (k_out && !rows_of_16(k_out, 0, 0, es))) {
        set_error("4-bit KV append: rows are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    p.q = q, p.k = k, p.v = v;
    p.q_ts = q_token_stride, p.q_hs = q_head_stride;
    p.k_ts = k_token_stride, p.k_hs = k_head_stride;
    p.v_ts = v_token_stride, p.v_hs = v_head_stride;
    p.q_out = q_out, p.k_out = k_out;
    p.start = start, p.cu = cu_seqlens;
    p.n = num_tokens, p.Hq = num_q_heads;
    const int D = cache->head_dim, GS = cache->group_size;
    const long units = ((long)num_q_heads + 2L * cache->num_kv_heads) * (D / 8);
    p.parts = wave_parts(num_tokens, units);
    const dim3 grid(wave_groups(num_tokens, p.parts));
    hipStream_t st = static_cast<hipStream_t>(stream);
    OJX_KV4_DISPATCH_T(kv4_append_kernel, dtype, D, GS, grid, dim3(kNT), 0, st, p);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

OJASX_API int ojasx_kv4_read_device(const OjasxKV4Cache *cache, const int *start, const int *cu_seqlens,
                                    const int *seen, int num_tokens, void *k_out, void *v_out, int dtype, void *stream) {
    using namespace ojx;
    Kv4ReadParams p{};
    int rc = kv4_view(cache, &p.c);
    if (rc) return rc;
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    if (num_tokens < 0 || num_tokens > kMostTokens || (!cu_seqlens && num_tokens != cache->num_sequences)) {
        set_error("4-bit KV read: %d tokens (at most 2^25; without cu_seqlens one for each of the %d sequences)", num_tokens,
                  cache->num_sequences);
        return OJASX_ERR_INVALID;
    }
    if (num_tokens == 0) return OJASX_OK;
    if (!start || !k_out || !v_out) return OJASX_ERR_NULL;
    if (!rows_of_16(k_out, 0, 0, 4) || !rows_of_16(v_out, 0, 0, 4)) {
        set_error("4-bit KV read: outputs are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    p.start = start, p.cu = cu_seqlens, p.seen = seen, p.k_out = k_out, p.v_out = v_out, p.n = num_tokens;
    const int D = cache->head_dim, GS = cache->group_size;
    p.parts = wave_parts(num_tokens, 2L * cache->num_kv_heads * (D / 8));
    const dim3 grid(wave_groups(num_tokens, p.parts));
    hipStream_t st = static_cast<hipStream_t>(stream);
    OJX_KV4_DISPATCH_T(kv4_read_kernel, dtype, D, GS, grid, dim3(kNT), 0, st, p);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

}  // extern "C"
