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
//
// One workgroup for a (sequence, head), since every pass of the selection needs all of its ranks and
// those of 32768 tokens fit LDS (of more they lie in the workspace).  What is read is small (8 bytes
// a token and head; of a moved token its rows besides), so the time is that of a chain of steps that
// wait for each other: block table, positions and weights, four counts, two walks with ballots.
// 11-bit digits, in three passes, took as long as four of 8 bits.  Up to kMoveInPlace moves the workgroup does itself, four units of
// a thread in flight; more are a second launch over the whole card, one unit of a thread in flight
// (16.8 us against 23.0 for four, for 8 sequences of 4096 that leave 1024).
//
// Measured, bf16, 8 heads of 128, the launches without the append: 64 sequences of 2064 tokens that
// leave 2048: 18 us (1 sequence of 1008 fp32 tokens: 10 us); 8 sequences of 4096 that leave 1024: 18 us and
// 17 us for their moves; a sequence of 65536, whose ranks lie in the workspace: 138 us (formed anew
// in each pass: 272).
#include <climits>

#include "kve.h"

namespace ojx {

namespace {
constexpr int kDigitBits = 8;            // of a rank's 32: four passes
constexpr int kDigits = 1 << kDigitBits;
constexpr int kCopies = 8;               // counters of a digit, so that equal digits of a wave's lanes collide less
constexpr int kRanksInLds = 32768;       // tokens whose ranks lie in LDS (128 KB); those of more in the workspace
constexpr int kMoveInPlace = 256;        // moves that the selecting workgroup does itself
// Threads of a selecting workgroup.  One that has a CU of its own takes kWideNT (8 sequences of 4096 tokens, 8
// heads: 21 us against 29 with 512); where a CU takes several, each is faster with fewer, which leave fewer
// idle in its scans (64 sequences of 2064: 19.5 us against 24; 256 of 1016: 26 with 256 threads, 32 with 512).
constexpr int kWideNT = 1024, kManyNT = 512, kShortNT = 256;
constexpr int kWidePairs = 256, kShortTokens = 1024;
constexpr int kMoveNT = 256;
constexpr size_t kSelectLds = kDigits * kCopies * 4 + 4096;   // static LDS of the selecting kernel, rounded up

struct KveEvictParams {
    KveView c;
    const int *held;
    int *moves;                 // [B][Hkv][2][most_moves]: places, tokens for them
    int *counts;                // [B][Hkv]
    uint32_t *ranks;            // [B][Hkv][most], where they are too many for LDS
    int budget, sink, recent, most, most_moves, in_lds;
};

template <int NT>
__device__ __forceinline__ int block_max(int v, int *sh) {
    v = ~wave_min_i(~v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = sh[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s = max(s, sh[i]);
    return s;
}

// The moves first, first + threads, ... of the n of a (sequence, kv head): keys, values, weights and
// positions of the slots of[m] to the slots to[m].  A thread has kUnits 16-byte units under way at a time.
template <int UNITS, int kUnits, typename L>
__device__ __forceinline__ void move_rows(const KveEvictParams &p, int b, int h, L to, L of, int n, int thread, int threads) {
    const long hrow = (long)h << p.c.pshift, all = (long)n * (2 * UNITS);
    for (long i0 = thread; i0 < all; i0 += (long)kUnits * threads) {
        long d[kUnits], s[kUnits];
        u4_t x[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const long i = i0 + (long)j * threads;
            const int m = (int)((i < all ? i : i0) / (2 * UNITS));
            d[j] = kve_row(p.c, b, to[m]), s[j] = kve_row(p.c, b, of[m]);
            if (i >= all || d[j] < 0) s[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int u = (int)((i0 + (long)j * threads) % (2 * UNITS));
            if (s[j] < 0) continue;
            x[j] = *reinterpret_cast<const u4_t *>((u < UNITS ? p.c.k : p.c.v) + (s[j] + hrow) * (UNITS * 16) + (u % UNITS) * 16);
        }
#pragma unroll
        for (int j = 0; j < kUnits; ++j) {
            const int u = (int)((i0 + (long)j * threads) % (2 * UNITS));
            if (s[j] < 0) continue;
            *reinterpret_cast<u4_t *>((u < UNITS ? p.c.k : p.c.v) + (d[j] + hrow) * (UNITS * 16) + (u % UNITS) * 16) = x[j];
            if (u == 0) p.c.w[d[j] + hrow] = p.c.w[s[j] + hrow];
            if (u == 1) p.c.pos[d[j] + hrow] = p.c.pos[s[j] + hrow];
        }
    }
}
}  // namespace

// Workgroup (kv head, sequence).  UNITS: 16-byte units of a row; MOVES: it moves the rows too.
template <int UNITS, bool MOVES, int NT>
__global__ __launch_bounds__(NT) void kve_select_kernel(KveEvictParams p) {
    constexpr int kNT = NT, kNW = NT / 64;
    constexpr int kBatch = NT == kManyNT ? 8 : 4;          // tokens of a thread whose loads are in flight together
    extern __shared__ uint32_t ranks[];
    __shared__ int counts[kDigits * kCopies], sh[kNW], sh2[kNW], picked[2], places_of[MOVES ? 2 * kMoveInPlace : 1];
    __shared__ int4 parts[kNW];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = min(max(p.held[b], 0), p.most);
    int *number = p.counts + (long)b * p.c.Hkv + h;
    if (n <= p.budget) {
        if (!MOVES && tid == 0) *number = 0;
        return;
    }
    const long hrow = (long)h << p.c.pshift;
    auto rank_of = [&](long row, int pos, float w, int newest) -> uint32_t {
        if (row < 0) return 0;
        if (pos < p.sink || (long)pos > (long)newest - p.recent) return 0xffffffffu;
        w += 0.f;                                // -0: 0
        if (w != w) return 1;
        const uint32_t u = __float_as_uint(w);
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    // kBatch tokens from t0 on, kNT apart
    long row[kBatch];
    int pos[kBatch];
    float w[kBatch];
    auto load = [&](int t0, bool weights) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) row[i] = t0 + i * kNT < n ? kve_row(p.c, b, t0 + i * kNT) : -1;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            pos[i] = row[i] < 0 ? INT_MIN : p.c.pos[row[i] + hrow];
            if (weights) w[i] = row[i] < 0 ? 0.f : p.c.w[row[i] + hrow];
        }
    };
    int newest = INT_MIN;
    const bool once = n <= kNT * kBatch;         // all tokens at once: they stay in registers
    for (int t0 = tid; t0 - tid < n; t0 += kNT * kBatch) {
        load(t0, once);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) newest = max(newest, pos[i]);
    }
    for (int i = tid; i < kDigits * kCopies; i += kNT) counts[i] = 0;
    newest = block_max<NT>(newest, sh);
    uint32_t *far = p.ranks + ((long)b * p.c.Hkv + h) * p.most;
    for (int t0 = tid; t0 - tid < n; t0 += kNT * kBatch) {
        if (!once) load(t0, true);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int t = t0 + i * kNT;
            if (t >= n) continue;
            const uint32_t r = rank_of(row[i], pos[i], w[i], newest);
            if (p.in_lds) ranks[t] = r;
            else far[t] = r;
        }
    }
    // The counts below read the ranks of the thread's own tokens; others' are read behind their barriers.
    // f(t, rank of t) for t = first, first + apart, ... by whole waves while any lane's is before `end`; four
    // ranks under way at a time, where a thread has that many.  At or past the end f gets some rank.
    auto walk = [&](int first, int end, int apart, auto f) {
        constexpr int kAtOnce = 4;
        if (once && p.in_lds) {                  // a few tokens under a bound past LDS have their ranks in the workspace
            for (int t = first; t - lane < end; t += apart) f(t, ranks[min(t, n - 1)]);
            return;
        }
        for (int t0 = first; t0 - lane < end; t0 += kAtOnce * apart) {
            uint32_t r[kAtOnce];
            if (p.in_lds) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) r[i] = ranks[min(t0 + i * apart, n - 1)];
            } else {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) r[i] = far[min(t0 + i * apart, n - 1)];
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) f(t0 + i * apart, r[i]);
        }
    };
    // the rank of the budget-th largest: `above` are larger
    uint32_t last = 0;
    int above = 0;
    uint32_t high = 0;                           // the bits of `last` that are known
    for (int shift = 32 - kDigitBits;; shift -= kDigitBits) {
        walk(tid, n, kNT, [&](int t, uint32_t r) {
            if (t < n && ((r ^ last) & high) == 0) atomicAdd(&counts[((r & ~high) >> shift) * kCopies + lane % kCopies], 1);
        });
        __syncthreads();
        // a digit for each of the first threads, the largest first
        const int d = kDigits - 1 - tid;
        int c = 0, upto = 0;
        if (tid < kDigits) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) c += counts[d * kCopies + i], counts[d * kCopies + i] = 0;
            upto = wave_scan_i(c);
            if (lane == 63) sh2[wv] = upto;
        }
        __syncthreads();
        if (tid < kDigits) {
            int before = above + upto - c;
#pragma unroll
            for (int i = 0; i < kDigits / 64; ++i) before += i < wv ? sh2[i] : 0;
            if (before < p.budget && before + c >= p.budget) picked[0] = d, picked[1] = before;
        }
        __syncthreads();
        last |= (uint32_t)picked[0] << shift;
        above = picked[1];
        high = 0xffffffffu << shift;
        if (shift == 0) break;
    }
    const int ties = p.budget - above;           // tokens of rank `last` that stay, the lowest slots
    // wave w has slots [w * span, (w + 1) * span)
    const int span = ((n + kNW - 1) / kNW + 63) & ~63, s0 = min(n, wv * span), s1 = min(n, s0 + span);
    // tokens of rank `last` and of larger ones, among the wave's slots below the budget and the others
    int4 mine = {0, 0, 0, 0};
    walk(s0 + lane, s1, 64, [&](int t, uint32_t r) {
        const unsigned long same = __ballot(t < s1 && r == last), more = __ballot(t < s1 && r > last), low = __ballot(t < p.budget);
        mine.x += __popcll(same & low), mine.y += __popcll(same & ~low);
        mine.z += __popcll(more & low), mine.w += __popcll(more & ~low);
    });
    if (lane == 0) parts[wv] = mine;
    __syncthreads();
    // of wave `lane`: ties before its slots, then the places and tokens for them that it has
    const int4 of_wave = lane < kNW ? parts[lane] : int4{0, 0, 0, 0};
    const int w0 = min(n, lane * span), w1 = lane < kNW ? min(n, w0 + span) : w0;
    const int tie_sum = wave_scan_i(of_wave.x + of_wave.y), tie_before = tie_sum - of_wave.x - of_wave.y;
    const int stay = ties - tie_before;          // of them that stay from the wave's first on
    const int places = min(w1, p.budget) - min(w0, p.budget) - of_wave.z - min(max(stay, 0), of_wave.x);
    const int tokens = of_wave.w + min(max(stay - of_wave.x, 0), of_wave.y);
    const int place_sum = wave_scan_i(places), token_sum = wave_scan_i(tokens);
    const int n_moves = __builtin_amdgcn_readlane(token_sum, 63);
    int tie = __builtin_amdgcn_readlane(tie_before, wv);
    int place = __builtin_amdgcn_readlane(place_sum - places, wv), token = __builtin_amdgcn_readlane(token_sum - tokens, wv);
    const unsigned long below = (1ul << lane) - 1;
    int *to = MOVES ? places_of : p.moves + ((long)b * p.c.Hkv + h) * 2 * p.most_moves, *of = to + p.most_moves;
    walk(s0 + lane, s1, 64, [&](int t, uint32_t r) {
        const unsigned long same = __ballot(t < s1 && r == last);
        const bool keep = r > last || (r == last && tie + __popcll(same & below) < ties);
        tie += __popcll(same);
        const unsigned long a = __ballot(t < s1 && t < p.budget && !keep), c = __ballot(t < s1 && t >= p.budget && keep);
        if (a >> lane & 1) to[min(place + (int)__popcll(a & below), p.most_moves - 1)] = t;
        if (c >> lane & 1) of[min(token + (int)__popcll(c & below), p.most_moves - 1)] = t;
        place += __popcll(a);
        token += __popcll(c);
    });
    if (!MOVES) {
        if (tid == 0) *number = n_moves;
        return;
    }
    __syncthreads();
    const int *from = places_of;
    move_rows<UNITS, 4>(p, b, h, from, from + p.most_moves, min(n_moves, p.most_moves), tid, kNT);
}

// The moves of the selecting launch: workgroup (part, kv head, sequence).
template <int UNITS>
__global__ __launch_bounds__(kMoveNT) void kve_move_kernel(KveEvictParams p) {
    const int h = blockIdx.y, b = blockIdx.z;
    const long at = (long)b * p.c.Hkv + h;
    const int *to = p.moves + at * 2 * p.most_moves;
    move_rows<UNITS, 1>(p, b, h, to, to + p.most_moves, min(p.counts[at], p.most_moves), blockIdx.x * kMoveNT + threadIdx.x,
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
    // moves and their numbers; ranks
    const long words = 2L * p->most_moves + 1 + (p->most > kRanksInLds ? p->most : 0);
    p->bytes = p->most_moves ? ((long)v.B * v.Hkv * words * 4 + 15) / 16 * 16 : 0;
    return OJASX_OK;
}

template <int UNITS, bool MOVES, int NT>
int select(const KveEvictParams &p, dim3 grid, size_t lds, hipStream_t st) {
    static DynLds granted;
    if (lds + kSelectLds > 65536)
        OJX_HIP(raise_dyn_lds(reinterpret_cast<const void *>(&kve_select_kernel<UNITS, MOVES, NT>), lds, &granted));
    OJX_LAUNCH((kve_select_kernel<UNITS, MOVES, NT>), grid, dim3(NT), lds, st, p);
    return OJASX_OK;
}
template <int UNITS>
int evict(const KveEvictParams &p, hipStream_t st) {
    const dim3 grid(p.c.Hkv, p.c.B);
    const size_t lds = p.in_lds ? round_up((size_t)p.most * 4, 16) : 0;
    const bool wide = (long)p.c.B * p.c.Hkv <= kWidePairs, brief = p.most <= kShortTokens;
    if (p.most_moves <= kMoveInPlace)
        return wide    ? select<UNITS, true, kWideNT>(p, grid, lds, st)
               : brief ? select<UNITS, true, kShortNT>(p, grid, lds, st)
                       : select<UNITS, true, kManyNT>(p, grid, lds, st);
    const int rc = wide    ? select<UNITS, false, kWideNT>(p, grid, lds, st)
                   : brief ? select<UNITS, false, kShortNT>(p, grid, lds, st)
                           : select<UNITS, false, kManyNT>(p, grid, lds, st);
    if (rc) return rc;
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
    p.ranks = reinterpret_cast<uint32_t *>(p.moves + (long)p.c.B * p.c.Hkv * 2 * pl.most_moves);
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
