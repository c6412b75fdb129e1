// kve_evict.hip -- eviction from the evicting KV cache (layout: kve.h) by the weight that its
// tokens got.
//
// Of each sequence and kv head that holds more than `budget` tokens, `budget` stay: those at
// positions below `sink`, those of the `recent` newest positions, and of the others the ones of
// largest weight, ties to the lowest slot.  A kept token from behind the budget takes the place of
// a dropped one before it, the i-th of them the i-th place: no row is both read and written, so
// all moves run at once, and no more rows move than have to.
//
// A token's rank is 32 bits that order like its weight: all ones where it is protected, 1 for a
// NaN, 0 where no page is mapped.  A workgroup finds the rank of the last kept token byte by byte
// from counts in LDS, then numbers the places and the tokens for them with wave ballots.
#include <climits>

#include "kve.h"

namespace ojx {

namespace {
constexpr int kNT = 1024;
constexpr int kNW = kNT / 64;
constexpr int kCopies = 16;              // counters of a digit, so that equal digits of a wave's lanes collide less
constexpr int kRanksInLds = 32768;       // tokens whose ranks are kept (128 KB); of more they are formed again
constexpr int kMoveInPlace = 256;        // moves that the selecting workgroup does itself
constexpr int kMoveNT = 256;
constexpr size_t kSelectLds = 256 * kCopies * 4 + 2048;   // static LDS of the selecting kernel, rounded up

struct KveEvictParams {
    KveView c;
    const int *held;
    int *moves;                 // [B][Hkv][2][most_moves]: places, tokens for them
    int *counts;                // [B][Hkv]
    int budget, sink, recent, most, most_moves, in_lds;
};

__device__ __forceinline__ int block_sum(int v, int *sh) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < kNW; ++i) s += sh[i];
    return s;
}
__device__ __forceinline__ int block_max(int v, int *sh) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = max(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = sh[0];
#pragma unroll
    for (int i = 1; i < kNW; ++i) s = max(s, sh[i]);
    return s;
}

// Rows `of` of a kv head to rows `to`: 16-byte unit u of the keys' and the values' row together.
template <int UNITS>
__device__ __forceinline__ void move_unit(const KveView &c, long to, long of, int u) {
    char *base = u < UNITS ? c.k : c.v;
    const int at = (u & (UNITS - 1)) * 16;
    *reinterpret_cast<u4_t *>(base + to * (UNITS * 16) + at) = *reinterpret_cast<const u4_t *>(base + of * (UNITS * 16) + at);
}
// Moves first, first + step, ... of the n of a (sequence, kv head), by the calling threads.
template <int UNITS>
__device__ __forceinline__ void move_rows(const KveEvictParams &p, int b, int h, const int *to, const int *of, int n, int thread,
                                          int threads) {
    const long hrow = (long)h << p.c.pshift;
    for (long i = thread; i < (long)n * (2 * UNITS); i += threads) {
        const int m = (int)(i / (2 * UNITS)), u = (int)(i % (2 * UNITS));
        const long d = kve_row(p.c, b, to[m]), s = kve_row(p.c, b, of[m]);
        if (d < 0 || s < 0) continue;
        move_unit<UNITS>(p.c, d + hrow, s + hrow, u);
        if (u == 0) p.c.w[d + hrow] = p.c.w[s + hrow];
        if (u == 1) p.c.pos[d + hrow] = p.c.pos[s + hrow];
    }
}
}  // namespace

// Workgroup (kv head, sequence).  UNITS: 16-byte units of a row; MOVES: it moves the rows too.
template <int UNITS, bool MOVES>
__global__ __launch_bounds__(kNT) void kve_select_kernel(KveEvictParams p) {
    extern __shared__ uint32_t ranks[];
    __shared__ int counts[256 * kCopies], total[256], sh[kNW], picked[2];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = min(max(p.held[b], 0), p.most);
    int *number = p.counts + (long)b * p.c.Hkv + h;
    if (n <= p.budget) {
        if (tid == 0) *number = 0;
        return;
    }
    const long hrow = (long)h << p.c.pshift;
    int newest = INT_MIN;
    for (int t = tid; t < n; t += kNT) {
        const long row = kve_row(p.c, b, t);
        if (row >= 0) newest = max(newest, p.c.pos[row + hrow]);
    }
    newest = block_max(newest, sh);
    auto form = [&](int t) -> uint32_t {
        const long row = kve_row(p.c, b, t);
        if (row < 0) return 0;
        const int pos = p.c.pos[row + hrow];
        const float w = p.c.w[row + hrow] + 0.f;           // -0: 0
        if (pos < p.sink || (long)pos > (long)newest - p.recent) return 0xffffffffu;
        if (w != w) return 1;
        const uint32_t u = __float_as_uint(w);
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    if (p.in_lds)
        for (int t = tid; t < n; t += kNT) ranks[t] = form(t);
    auto rank = [&](int t) { return p.in_lds ? ranks[t] : form(t); };
    // the rank of the budget-th largest: `above` are larger
    uint32_t last = 0;
    int above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256 * kCopies; i += kNT) counts[i] = 0;
        __syncthreads();
        for (int t = tid; t < n; t += kNT) {
            const uint32_t r = rank(t);
            if (shift == 24 || (r ^ last) >> (shift + 8) == 0) atomicAdd(&counts[(r >> shift & 255) * kCopies + lane % kCopies], 1);
        }
        __syncthreads();
        if (tid < 256) {
            int s = 0;
            for (int i = 0; i < kCopies; ++i) s += counts[tid * kCopies + i];
            total[tid] = s;
        }
        __syncthreads();
        if (wv == 0) {                           // four digits a lane, the largest first
            int mine[4], s = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) s += mine[i] = total[255 - (lane * 4 + i)];
            int before = s;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(before, o);
                if (lane >= o) before += x;
            }
            before += above - s;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < p.budget && before + mine[i] >= p.budget) picked[0] = 255 - (lane * 4 + i), picked[1] = before;
                before += mine[i];
            }
        }
        __syncthreads();
        last |= (uint32_t)picked[0] << shift;
        above = picked[1];
    }
    const int ties = p.budget - above;           // tokens of rank `last` that stay, the lowest slots
    // wave w has slots [w * span, (w + 1) * span)
    const int span = ((n + kNW - 1) / kNW + 63) & ~63, s0 = min(n, wv * span), s1 = min(n, s0 + span);
    auto before_waves = [&](int v) {             // sum of v (one value a wave) over the waves before
        __syncthreads();
        if (lane == 0) sh[wv] = v;
        __syncthreads();
        int s = 0;
        for (int i = 0; i < wv; ++i) s += sh[i];
        return s;
    };
    int mine = 0;
    for (int t = s0 + lane; t - lane < s1; t += 64) mine += __popcll(__ballot(t < s1 && rank(min(t, n - 1)) == last));
    const int tie0 = before_waves(mine);
    const unsigned long below = (1ul << lane) - 1;
    auto kept = [&](int t, int &tie) {           // of the wave's 64 slots from t - lane on; tie: ties before them
        const uint32_t r = rank(min(t, n - 1));
        const unsigned long same = __ballot(t < s1 && r == last);
        const bool keep = r > last || (r == last && tie + __popcll(same & below) < ties);
        tie += __popcll(same);
        return keep;
    };
    int tie = tie0, places = 0, tokens = 0;
    for (int t = s0 + lane; t - lane < s1; t += 64) {
        const bool keep = kept(t, tie);
        places += __popcll(__ballot(t < s1 && t < p.budget && !keep));
        tokens += __popcll(__ballot(t < s1 && t >= p.budget && keep));
    }
    int place = before_waves(places), token = before_waves(tokens);
    const int n_moves = block_sum(lane == 0 ? tokens : 0, sh);
    int *to = p.moves + ((long)b * p.c.Hkv + h) * 2 * p.most_moves, *of = to + p.most_moves;
    tie = tie0;
    for (int t = s0 + lane; t - lane < s1; t += 64) {
        const bool keep = kept(t, tie);
        const unsigned long a = __ballot(t < s1 && t < p.budget && !keep), c = __ballot(t < s1 && t >= p.budget && keep);
        if (a >> lane & 1) to[min(place + (int)__popcll(a & below), p.most_moves - 1)] = t;
        if (c >> lane & 1) of[min(token + (int)__popcll(c & below), p.most_moves - 1)] = t;
        place += __popcll(a);
        token += __popcll(c);
    }
    if (tid == 0) *number = n_moves;
    if (MOVES) {
        __syncthreads();
        move_rows<UNITS>(p, b, h, to, of, min(n_moves, p.most_moves), tid, kNT);
    }
}

// The moves of the selecting launch: workgroup (part, kv head, sequence).
template <int UNITS>
__global__ __launch_bounds__(kMoveNT) void kve_move_kernel(KveEvictParams p) {
    const int h = blockIdx.y, b = blockIdx.z;
    const long at = (long)b * p.c.Hkv + h;
    const int *to = p.moves + at * 2 * p.most_moves;
    move_rows<UNITS>(p, b, h, to, to + p.most_moves, min(p.counts[at], p.most_moves), blockIdx.x * kMoveNT + threadIdx.x,
                     gridDim.x * kMoveNT);
}

namespace {
struct KveEvictPlan {
    int most, most_moves;
    long bytes;
};
int evict_plan(const KveView &v, int budget, int sink, int recent, int max_held, KveEvictPlan *p) {
    if (budget <= 0 || sink < 0 || recent < 0 || (long)sink + recent > budget || max_held < 0) {
        set_error("KV eviction: budget %d for %d sink and %d recent tokens, max_held %d", budget, sink, recent, max_held);
        return OJASX_ERR_INVALID;
    }
    if (v.B > 65535) {
        set_error("KV eviction: %d sequences (at most 65535)", v.B);
        return OJASX_ERR_INVALID;
    }
    p->most = max_held && max_held < v.cap ? max_held : v.cap;
    const int over = p->most - budget;
    p->most_moves = over <= 0 ? 0 : over < budget ? over : budget;
    p->bytes = p->most_moves ? ((long)v.B * v.Hkv * (2L * p->most_moves + 1) * 4 + 15) / 16 * 16 : 0;
    return OJASX_OK;
}

template <int UNITS>
int evict(const KveEvictParams &p, hipStream_t st) {
    const dim3 grid(p.c.Hkv, p.c.B);
    const size_t lds = p.in_lds ? round_up((size_t)p.most * 4, 16) : 0;
    const bool wide = lds + kSelectLds > 65536;
    if (p.most_moves <= kMoveInPlace) {
        static DynLds granted;
        if (wide) OJX_HIP(raise_dyn_lds(reinterpret_cast<const void *>(&kve_select_kernel<UNITS, true>), lds, &granted));
        OJX_LAUNCH((kve_select_kernel<UNITS, true>), grid, dim3(kNT), lds, st, p);
        return OJASX_OK;
    }
    static DynLds granted;
    if (wide) OJX_HIP(raise_dyn_lds(reinterpret_cast<const void *>(&kve_select_kernel<UNITS, false>), lds, &granted));
    OJX_LAUNCH((kve_select_kernel<UNITS, false>), grid, dim3(kNT), lds, st, p);
    // parts of a (sequence, kv head): 8 moves or more each, no more than four times what fills the card
    const long pairs = (long)p.c.B * p.c.Hkv, wanted = (p.most_moves + 7) / 8, fill = (4096 + pairs - 1) / pairs;
    OJX_LAUNCH((kve_move_kernel<UNITS>), dim3((unsigned)(wanted < fill ? wanted : fill), p.c.Hkv, p.c.B), dim3(kMoveNT), 0, st, p);
    return OJASX_OK;
}
}  // namespace

}  // namespace ojx

extern "C" {

OJASX_API long ojasx_kve_evict_workspace(const OjasxKVECache *cache, int budget, int max_held) {
    using namespace ojx;
    KveView v{};
    KveEvictPlan pl{};
    int rc = kve_view(cache, &v);
    if (!rc) rc = evict_plan(v, budget, 0, 0, max_held, &pl);
    return rc ? rc : pl.bytes;
}

OJASX_API int ojasx_kve_evict_device(const OjasxKVECache *cache, const int *held, int budget, int sink_tokens,
                                     int recent_tokens, int max_held, void *workspace, long workspace_bytes,
                                     void *stream) {
    using namespace ojx;
    KveEvictParams p{};
    KveEvictPlan pl{};
    int rc = kve_view(cache, &p.c);
    if (!rc) rc = evict_plan(p.c, budget, sink_tokens, recent_tokens, max_held, &pl);
    if (rc) return rc;
    if (!held) return OJASX_ERR_NULL;
    if (!pl.most_moves) return OJASX_OK;         // no sequence can hold more than the budget
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < pl.bytes) {
        set_error("KV eviction: the workspace has to be 16-byte aligned and of %ld bytes, got %ld", pl.bytes,
                  workspace_bytes);
        return OJASX_ERR_INVALID;
    }
    p.held = held;
    p.counts = static_cast<int *>(workspace);
    p.moves = p.counts + (long)p.c.B * p.c.Hkv;
    p.budget = budget, p.sink = sink_tokens, p.recent = recent_tokens;
    p.most = pl.most, p.most_moves = pl.most_moves, p.in_lds = pl.most <= kRanksInLds;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (p.c.D * (p.c.dtype == OJASX_DTYPE_F32 ? 4 : 2) / 16) {
        case 8: rc = evict<8>(p, st); break;
        case 16: rc = evict<16>(p, st); break;
        case 32: rc = evict<32>(p, st); break;
        default: rc = evict<64>(p, st);
    }
    if (rc) return rc;
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

}  // extern "C"
