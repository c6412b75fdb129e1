// kve_append.hip -- the write side of the evicting KV cache (layout: kve.h): queries and keys
// rotated by their positions, keys and values into their slots, with weights and positions.
//
// The rotation is that of the 4-bit cache (kv4_append.hip): angles in fp64 turns, products in
// fp64, one rounding to fp32 and one to the element type.  What does not rotate is copied bit
// for bit.
//
// Bound by the copy of the rows: 8192 bf16 tokens with 32 / 8 heads of 128 take 42 us, 4.8 TB/s of
// rows in and out; a token each of 64 sequences takes 4.8 us, a launch and the chain of table entry,
// angles and rows.  Loading a token's first rows before its place and angles are known leaves room
// for fewer waves (53 us).
#include "kve.h"

namespace ojx {

namespace {
constexpr int kNT = 256;
constexpr int kAtOnce = 3;      // units' loads of a lane in flight together

struct KveAppendParams {
    KveView c;
    const void *q, *k, *v;
    long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;    // token and head strides, elements
    void *q_out;                                // contiguous [n][heads][D]
    const float *weight;                        // [n][Hkv] or null
    const int *start, *position, *cu;
    int n, Hq, parts;
};

// Eight values as they lie in memory.
template <typename T>
struct Raw8 {
    u4_t a[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) a[i] = reinterpret_cast<const u4_t *>(p)[i];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) reinterpret_cast<u4_t *>(p)[i] = a[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (unsigned i = 0; i < sizeof(T) / 2; ++i) a[i] = u4_t{0, 0, 0, 0};
    }
};
}  // namespace

// Wave i of the launch takes token i / parts and every parts-th 64 units of eight dimensions of
// its query, key and value rows; a lane's dimensions are the same in all of them, so its angles
// stay in registers.
template <typename T, int D>
__global__ __launch_bounds__(kNT) void kve_append_kernel(KveAppendParams p) {
    __shared__ double2 angles[kNT / 64][D / 2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int UPR = D / 8, RPW = 64 / UPR;   // units of eight per row, rows per 64 units
    const int wave = blockIdx.x * (kNT / 64) + w, n = wave / p.parts, part = wave - n * p.parts;
    if (n >= p.n) return;
    const int Hkv = p.c.Hkv, rows = p.Hq + 2 * Hkv, step = p.parts * RPW;
    const int half = p.c.rot >> 1, d0 = lane % UPR * 8;
    const bool turns = d0 < p.c.rot, low = d0 < half;
    const int other = !turns || p.c.interleaved ? 0 : low ? half : -half;   // where the values lie they turn with
    const Kv4Row r = kv4_row(p.cu, p.start, p.c.B, n);
    const int slot = r.pos;                      // kv4_row counts from start: the slot here
    const int pos = r.b < 0 ? 0 : (int)((unsigned)p.position[r.b] + (unsigned)slot - (unsigned)p.start[r.b]);
    // the pool row of kv head 0
    const long at = r.b < 0 || slot < 0 || slot >= p.c.cap ? -1 : kve_row(p.c, r.b, slot);
    double co[8], sn[8];
    token_angles(p.c.turns, half, p.c.interleaved, pos, d0, angles[w], co, sn);
    for (int row0 = part * RPW + lane / UPR; row0 - lane / UPR < rows; row0 += kAtOnce * step) {
        Raw8<T> x[kAtOnce], y[kAtOnce];
        // past the last row: row 0's values, not used
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = row0 + i * step < rows ? row0 + i * step : 0;
            const bool isq = row < p.Hq, isv = row >= p.Hq + Hkv;
            const T *src = d0 + (isq ? static_cast<const T *>(p.q) + n * p.q_ts + row * p.q_hs
                                 : isv ? static_cast<const T *>(p.v) + n * p.v_ts + (row - p.Hq - Hkv) * p.v_hs
                                       : static_cast<const T *>(p.k) + n * p.k_ts + (row - p.Hq) * p.k_hs);
            x[i].load(src);
            y[i].load(src + other);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int row = row0 + i * step;
            if (row >= rows) continue;
            const bool isq = row < p.Hq, isv = row >= p.Hq + Hkv;
            const int head = isq ? row : isv ? row - p.Hq - Hkv : row - p.Hq;
            if (r.b < 0) {                           // a row of no sequence
                x[i].clear();
                if (isq) x[i].store(static_cast<T *>(p.q_out) + ((size_t)n * p.Hq + head) * D + d0);
                continue;
            }
            const long to = at + ((long)head << p.c.pshift);
            T *out = isq ? static_cast<T *>(p.q_out) + ((size_t)n * p.Hq + head) * D + d0
                         : reinterpret_cast<T *>(isv ? p.c.v : p.c.k) + to * D + d0;
            if (!isq && at < 0) continue;
            if (turns && !isv) {
                float a[8], b[8];
                load8(reinterpret_cast<const T *>(x[i].a), a);
                load8(reinterpret_cast<const T *>(y[i].a), b);
                if (p.c.interleaved)
#pragma unroll
                    for (int e = 0; e < 8; ++e) b[e] = a[e ^ 1];
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = (float)fma((double)a[e], co[e], (double)b[e] * sn[e]);
                store8(out, z);
            } else {
                x[i].store(out);
            }
            if (isv && d0 == 0) {
                p.c.w[to] = p.weight ? p.weight[(size_t)n * Hkv + head] : 0.f;
                p.c.pos[to] = pos;
            }
        }
    }
}

int kve_view(const OjasxKVECache *c, KveView *v) {
    if (!c || !c->keys || !c->values || !c->weights || !c->positions || !c->block_table) {
        set_error("evicting KV cache: a NULL buffer");
        return OJASX_ERR_NULL;
    }
    const int D = c->head_dim, P = c->page_size;
    if (D != 64 && D != 128 && D != 256) {
        set_error("evicting KV cache: head_dim %d (64, 128 or 256)", D);
        return OJASX_ERR_INVALID;
    }
    if (c->dtype != OJASX_DTYPE_F32 && c->dtype != OJASX_DTYPE_BF16 && c->dtype != OJASX_DTYPE_F16) {
        set_error("evicting KV cache: unsupported dtype %d", c->dtype);
        return OJASX_ERR_INVALID;
    }
    if (P < 16 || P > 32768 || (P & (P - 1))) {
        set_error("evicting KV cache: page_size %d is no power of two from 16 to 32768", P);
        return OJASX_ERR_INVALID;
    }
    if (c->num_sequences <= 0 || c->num_kv_heads <= 0 || c->num_kv_heads > 65535 || c->num_pages <= 0 ||
        c->max_pages <= 0) {
        set_error("evicting KV cache: %d sequences, %d kv heads, %d pages, %d of a sequence", c->num_sequences,
                  c->num_kv_heads, c->num_pages, c->max_pages);
        return OJASX_ERR_INVALID;
    }
    // room for the steps of a loop past a sequence's end
    if ((long)c->max_pages * P > 0x7ff00000L) {
        set_error("evicting KV cache: %d pages of %d slots of a sequence are more than 2^31 - 2^20 slots", c->max_pages, P);
        return OJASX_ERR_INVALID;
    }
    if (c->rotary_dim < 0 || c->rotary_dim > D || c->rotary_dim % 16 || (c->rotary_dim && !c->turns)) {
        set_error("evicting KV cache: rotary_dim %d (a multiple of 16 up to %d, with turns)", c->rotary_dim, D);
        return OJASX_ERR_INVALID;
    }
    if ((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) & 15) {
        set_error("evicting KV cache: keys and values are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    v->k = static_cast<char *>(c->keys);
    v->v = static_cast<char *>(c->values);
    v->w = c->weights;
    v->pos = c->positions;
    v->bt = c->block_table;
    v->turns = c->turns;
    v->B = c->num_sequences;
    v->max_pages = c->max_pages;
    v->pshift = __builtin_ctz((unsigned)P);
    v->num_pages = c->num_pages;
    v->Hkv = c->num_kv_heads;
    v->D = D;
    v->dtype = c->dtype;
    v->rot = c->rotary_dim;
    v->interleaved = c->interleaved != 0;
    v->cap = c->max_pages * P;
    return OJASX_OK;
}

namespace {
// Waves per token: one for each 64 units while the launch is small, one in all when that makes
// 4096 waves (16 a CU): more of them compute the same angles again (the 4-bit cache's rule).
int wave_parts(int n, long units) {
    const long most = (units + 63) / 64, want = 4096 / n;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}
constexpr int kMostTokens = 1 << 25;            // a grid has fewer than 2^32 threads

template <typename T>
void append(int D, dim3 grid, hipStream_t st, const KveAppendParams &p) {
    if (D == 64) OJX_LAUNCH((kve_append_kernel<T, 64>), grid, dim3(kNT), 0, st, p);
    else if (D == 128) OJX_LAUNCH((kve_append_kernel<T, 128>), grid, dim3(kNT), 0, st, p);
    else OJX_LAUNCH((kve_append_kernel<T, 256>), grid, dim3(kNT), 0, st, p);
}
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API int ojasx_kve_append_device(const OjasxKVECache *cache, const void *q, long q_token_stride,
                                      long q_head_stride, int num_q_heads, void *q_out, const void *k,
                                      long k_token_stride, long k_head_stride, const void *v,
                                      long v_token_stride, long v_head_stride, const float *weight,
                                      int num_tokens, const int *start, const int *position,
                                      const int *cu_seqlens, void *stream) {
    using namespace ojx;
    KveAppendParams p{};
    int rc = kve_view(cache, &p.c);
    if (rc) return rc;
    if (num_tokens < 0 || num_tokens > kMostTokens || num_q_heads < 0 || num_q_heads > 65535 ||
        (!cu_seqlens && num_tokens != cache->num_sequences)) {
        set_error("KV append: %d tokens (at most 2^25), %d query heads (without cu_seqlens one token for each of "
                  "the %d sequences)", num_tokens, num_q_heads, cache->num_sequences);
        return OJASX_ERR_INVALID;
    }
    if (num_tokens == 0) return OJASX_OK;
    if (!k || !v || !start || (num_q_heads && (!q || !q_out))) return OJASX_ERR_NULL;
    const size_t es = p.c.dtype == OJASX_DTYPE_F32 ? 4 : 2;
    if (!rows_of_16(k, k_token_stride, k_head_stride, es) || !rows_of_16(v, v_token_stride, v_head_stride, es) ||
        (num_q_heads && (!rows_of_16(q, q_token_stride, q_head_stride, es) || !rows_of_16(q_out, 0, 0, es)))) {
        set_error("KV append: rows are 16-byte aligned");
        return OJASX_ERR_INVALID;
    }
    p.q = q, p.k = k, p.v = v;
    p.q_ts = q_token_stride, p.q_hs = q_head_stride;
    p.k_ts = k_token_stride, p.k_hs = k_head_stride;
    p.v_ts = v_token_stride, p.v_hs = v_head_stride;
    p.q_out = q_out, p.weight = weight;
    p.start = start, p.position = position ? position : start, p.cu = cu_seqlens;
    p.n = num_tokens, p.Hq = num_q_heads;
    const int D = p.c.D;
    p.parts = wave_parts(num_tokens, ((long)num_q_heads + 2L * p.c.Hkv) * (D / 8));
    const dim3 grid((unsigned)(((long)num_tokens * p.parts + kNT / 64 - 1) / (kNT / 64)));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (p.c.dtype == OJASX_DTYPE_F32) append<float>(D, grid, st, p);
    else if (p.c.dtype == OJASX_DTYPE_BF16) append<__hip_bfloat16>(D, grid, st, p);
    else append<__half>(D, grid, st, p);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

}  // extern "C"
