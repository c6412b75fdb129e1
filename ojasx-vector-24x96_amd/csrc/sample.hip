// sample.hip -- one token of every row of logits, drawn with a given random number.
//
//   e_i = exp((l_i - max l) / T); the tokens in order of falling l, equal ones of rising index;
//   top-k: the first k of them; top-p: of those the shortest beginning whose sum of e is at least
//   p times all of theirs; min-p: of those the ones with e_i >= m; token: the first of the kept
//   ones, in the vocabulary's order, at which the running sum of e passes u times their sum.
//
// All three cuts keep a beginning of one order, so together they are one logit kappa and a count:
// kept is what lies above kappa, and of the tokens that equal it the first `ties`.  No sort, and
// no token is looked at more than three times:
//   1. by slices of the vocabulary, counts of tokens and sums of e in 255 bins of the logit (width
//      T / 7, on one grid for all slices, from the slice's largest down to where e is below 2^-51
//      of it and is not drawn);
//   2. by slices again, with the slices' bins added up: the tokens of the bins that the cuts fall
//      into go to a list of the row;
//   3. by rows: the cuts themselves, selected among the list's tokens digit by digit of their
//      logits' order; then the slice that the draw falls into, from the slices' kept sums, and the
//      token within it.
// A row without cuts needs of 1. its slices' sums alone, and nothing of 2.
//
// A drawn token is a whole number: it has to be the definition's own.  So e is fp64 to about
// 2^-50, sums are fp64, or in LDS, where they are added in any order, 64-bit integers: a fixed
// number of bits behind the point, the same result in every order.  A slice's sums have 50 bits, relative
// to its largest e: 8192 equal logits that round alike are off by 2^-38 of it, 3.6e-12.  A bin's sums are
// relative to the bin's largest.  What is not drawn and lies in a bin that is counted shifts a border by
// 2^-51 for each such token.
//
// What is read is small (2 or 4 bytes a logit), and the fp64 products of the exponentials issue in no more
// than a third of the cycles.  With cuts 1. is bound by its one or two additions in LDS for each token (half of
// the LDS cycles are conflicts), 2. by adding the row's bins in every workgroup; the rest, and few rows, by the
// latency of the launches' chains.  Measured: 256 rows of 32000 fp16 logits without cuts 11 + 10 us (1. and
// 3.), 64 rows of 151936 bf16 ones with settings of their own 19 + 18 + 20 us, 256 such rows with top-k 50 and
// top-p 0.9 54 + 42 + 15, one row of 151936 fp32 ones with the same 7 + 9 + 16.5 us.  Keeping a row's
// workgroups on one die's L2 took 3 % off rows that all have cuts and cost as much where only some have.
#include <cfloat>
#include <climits>
#include <cmath>

#include "sample.h"

namespace ojx {

namespace {
constexpr int kNT = 1024;                // threads of a row's workgroup
constexpr int kNW = kNT / 64;
constexpr int kPer = 8;                  // tokens that a thread takes at a time
constexpr int kSlice = kNT * kPer;
// Threads of a slice's workgroup, each with four times kPer tokens: what a wave does once, its settings,
// maxima and sums, is as much as the work on 8 tokens a lane (256 rows of 32000: 15.5 us with 1024 threads).
constexpr int kSliceNT = 256;
constexpr int kSliceNW = kSliceNT / 64;
constexpr int kSteps = kSlice / (kSliceNT * kPer);
constexpr int kBins = 256;               // the last: e below kLeast
constexpr int kCopies = 8;               // of the bins' counters, so that a wave's lanes collide less
constexpr double kBinsPerE = 7.0;        // 255 / 7 = 36.4 > 51 ln 2
constexpr int kFrac = 50;                // bits behind the point of a slice's sums (8192 of them: 2^63)
constexpr int kList = 8192;              // tokens that are selected among in LDS; more: in memory
constexpr int kMostSlices = 512;
constexpr int kDigitBits = 9;            // of a selection's pass: two passes over an fp32 bin's keys
constexpr int kDigits = 1 << kDigitBits;
constexpr double kLeast = 0x1p-51;       // tokens of a smaller e are not drawn

typedef unsigned long long u64;

struct SliceHead {
    double total;                        // rows without cuts: the slice's sum of e, relative to its largest
    float most;
    int at;                              // index of the largest logit
    int top;                             // its bin
    int bad;                             // a NaN or +inf among the logits
};
struct Bin {
    u64 sum;
    unsigned count, pad;                 // of rows with a top-k cut
};
struct SliceBins {
    Bin upto[kBins];                     // sums and counts up to and with the bin; the last two alike
};
struct RowBins {                         // of the whole row, up to and with the bin
    double sum[kBins];                   // the last two alike
    int count[kBins];
    int cut[6];                          // CutBins
    unsigned listed;                     // tokens in the row's list
    int pad;
};
struct Work {
    SliceBins *bins;                     // [row][slice]
    SliceHead *heads;                    // [row][slice]
    RowBins *rows;                       // [row]
    uint2 *list;                         // [row][vocab]: key, index and in the high byte the bin
};

// A constant held in scalar registers: one instruction adds its multiple, where the compiler would
// copy it to two vector registers first.
__device__ __forceinline__ double held(double c) {
    asm("" : "+s"(c));
    return c;
}
// 2^(x c), -1020 < x c <= 60, to about 2^-51.5: 2^f, |f| <= 1/2, by the polynomial of degree 10
// through its values at the 11 Chebyshev nodes (off by 3e-16), scaled by the exponent.
__device__ __forceinline__ double exp2_f64(double x, double c) {
    const double whole = held(0x1.8p52);         // the sum's last bits are x c rounded to whole numbers
    const double t = fma(x, c, whole), f = fma(x, c, whole - t);
    double p = fma(held(0x1.e6063f7217bc6p-28), f, held(0x1.b675bca4eeebbp-24));
    p = fma(p, f, held(0x1.62bfd47773353p-20));
    p = fma(p, f, held(0x1.ffcb54062e698p-17));
    p = fma(p, f, held(0x1.430913096fd9fp-13));
    p = fma(p, f, held(0x1.5d87fe9d7a584p-10));
    p = fma(p, f, held(0x1.3b2ab6fba1ddap-7));
    p = fma(p, f, held(0x1.c6b08d703ce49p-5));
    p = fma(p, f, held(0x1.ebfbdff82c598p-3));
    p = fma(p, f, held(0x1.62e42fefa3a19p-1));
    p = fma(p, f, 1.0);                          // 0.7 .. 1.42
    return __longlong_as_double(__double_as_longlong(p) + (__double_as_longlong(t) << 52));
}
// Bits of e in [0, 1] behind the point, rounded: e + 2^(52 - frac) has its last bit there.
__device__ __forceinline__ u64 fixed(double e, int frac) {
    const double one = __longlong_as_double((long long)(1023 + 52 - frac) << 52);
    return (u64)(__double_as_longlong(e + one) - __double_as_longlong(one));
}

// Numbers in the order of the floats (no NaN; -0 as 0), and back.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Row {
    double c;                            // log2(e) / T
    double bins;                         // bins per unit of the logit
    double width;                        // a bin's
    float limit;                         // logits past it are one bin: 2^29 bins from 0
    double depth;                        // e of a logit further below the largest is that of this distance
    double p, m;
    int k;
    bool greedy, bad, k_cut, p_cut, m_cut;
    __device__ __forceinline__ bool cuts() const { return k_cut || p_cut || m_cut; }
    // A logit's bin on the grid of all slices: its product rounded to the nearest whole number, so that
    // larger logits have no smaller one.
    __device__ __forceinline__ int bin(float x) const {
        return __double2loint(fma((double)__builtin_amdgcn_fmed3f(x, -limit, limit), bins, 0x1.8p52));
    }
    // Bins behind bin `top`, at most the last.
    __device__ __forceinline__ int behind(int top, float x) const {
        const int b = min(top - bin(x), kBins - 1);
        return x == -INFINITY ? kBins - 1 : b;
    }
    // A logit that none of bin b is above, nor further below than the bin's width unless the bin is one of all
    // beyond the limit; top, most: the row's first bin and largest logit.  Sums of the bin are of e relative to
    // it: relative to the row's largest, the step of a fixed point is as much as the e of a far bin's tokens, and
    // equal logits all round the same way.
    __device__ __forceinline__ double bin_top(int b, int top, float most) const {
        return b ? ((double)(top - b) + 0.5) * width : (double)most;
    }
    __device__ __forceinline__ double e(double x, double most) const { return exp2_f64(fmax(x - most, -depth), c); }
};
__device__ __forceinline__ Row row_of(const SampleParams &a, int r) {
    Row s;
    const double given = a.temperatures ? (double)a.temperatures[r] : a.temperature;
    const double T = fmax(given, 0x1p-300);      // as any below: of two fp32 logits the smaller's e is 0, and 1 / T is finite
    s.k = a.top_ks ? a.top_ks[r] : a.top_k;
    s.p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
    s.m = fmin(a.min_ps ? (double)a.min_ps[r] : a.min_p, 1.0);
    s.bad = !(given >= 0.0) || given > (double)FLT_MAX || s.p != s.p || (a.min_ps && a.min_ps[r] != a.min_ps[r]);
    s.greedy = given == 0.0;
    const double inv = 1.0 / T;                  // the others are its multiples or T's: a division costs 20 products
    s.c = 1.4426950408889634074 * inv;
    s.bins = kBinsPerE * inv;
    s.width = 1.0 / kBinsPerE * T;
    s.limit = (float)fmin(0x1p29 / kBinsPerE * T, (double)FLT_MAX);
    s.depth = 1000.0 / 1.4426950408889634074 * T;
    s.k_cut = s.k > 0 && s.k < a.vocab;
    s.p_cut = s.p < 1.0;
    s.m_cut = s.m > 0.0;
    return s;
}

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }

// Eight logits from i on, -inf past the vocabulary's end.  Rows begin anywhere: global loads need no
// alignment, only the compiler has to know.
template <typename T>
__device__ __forceinline__ void load_logits(const T *row, int i, int V, float (&x)[kPer]) {
    if (i + kPer <= V) {
        typedef unsigned int u4_any __attribute__((ext_vector_type(4), aligned(2)));
        T raw[kPer];
#pragma unroll
        for (unsigned j = 0; j < sizeof(T) / 2; ++j)
            reinterpret_cast<u4_any *>(raw)[j] = reinterpret_cast<const u4_any *>(row + i)[j];
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = as_f32(raw[e]);
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = i + e < V ? as_f32(row[i + e]) : -INFINITY;
    }
}

// A thread's tokens of a slice that begins at s0, all loads of a slice within the vocabulary under way together.
template <typename T>
__device__ __forceinline__ void load_slice(const T *row, int s0, int V, float (&x)[kSteps][kPer]) {
    typedef unsigned int u4_any __attribute__((ext_vector_type(4), aligned(2)));
    constexpr int kVecs = sizeof(T) / 2;
    const int i0 = s0 + (int)threadIdx.x * kPer;
    if (s0 + kSlice <= V) {
        u4_any raw[kSteps][kVecs];
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int j = 0; j < kVecs; ++j)
                raw[i][j] = reinterpret_cast<const u4_any *>(row + i0 + i * (kSliceNT * kPer))[j];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            T part[kPer];
            __builtin_memcpy(part, raw[i], sizeof(part));
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[i][e] = as_f32(part[e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) load_logits(row, i0 + i * (kSliceNT * kPer), V, x[i]);
    }
}

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
__device__ __forceinline__ double lane_d(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                            __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum_d(double v) {
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    v += dpp_d<0x141>(v);
    v += dpp_d<0x140>(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp0_u(u64 v) {
    return (u64)(unsigned)dpp0_i<CTRL, ROWS>((int)(v >> 32)) << 32 | (unsigned)dpp0_i<CTRL, ROWS>((int)v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp0_d(double v) {
    return __longlong_as_double((long long)dpp0_u<CTRL, ROWS>((u64)__double_as_longlong(v)));
}
// As wave_scan_i.
#define OJX_WAVE_SCAN(NAME, T, DPP)                     \
    __device__ __forceinline__ T NAME(T v) {            \
        v += DPP<0x111, 0xF>(v);                        \
        v += DPP<0x112, 0xF>(v);                        \
        v += DPP<0x114, 0xF>(v);                        \
        v += DPP<0x118, 0xF>(v);                        \
        v += DPP<0x142, 0xA>(v);                        \
        v += DPP<0x143, 0xC>(v);                        \
        return v;                                       \
    }
OJX_WAVE_SCAN(wave_scan_u, u64, dpp0_u)
OJX_WAVE_SCAN(wave_scan_d, double, dpp0_d)
#undef OJX_WAVE_SCAN

// What the slices' heads say of the row; mine: the head of slice number lane.
struct RowHead {
    float most;
    int at, top, bad;
    SliceHead mine;
};
__device__ __forceinline__ RowHead row_head(const Row &row, const SliceHead *heads, int S) {
    const int lane = threadIdx.x & 63;           // by every wave
    RowHead h;
    h.mine = heads[min(lane, S - 1)];
    h.most = h.mine.most, h.at = h.mine.at, h.bad = h.mine.bad;
    for (int s = 64 + lane; s < S; s += 64) {
        const SliceHead x = heads[s];
        if (x.most > h.most) h.most = x.most, h.at = x.at;
        h.bad |= x.bad;
    }
    const float most = wave_max_f(h.most);
    h.at = wave_min_i(h.most == most ? h.at : INT_MAX);
    h.bad = __any(h.bad);
    h.most = most;
    h.top = row.bin(most);
    return h;
}
// Bins that a slice's first one is behind the row's.
__device__ __forceinline__ int slice_off(const SliceHead &h, int top) {
    return h.most == -INFINITY ? kBins : min(max(top - h.top, 0), kBins);
}
}  // namespace

// Workgroup row * slices + slice.
template <typename T>
__global__ __launch_bounds__(kSliceNT) void sample_slice_kernel(SampleParams a, Work wk) {
    __shared__ u64 sum[kBins * kCopies];
    __shared__ unsigned count[kBins * kCopies];
    __shared__ float wm[kSliceNW];
    __shared__ int wi[kSliceNW], wbad[kSliceNW];
    __shared__ double wt[kSliceNW];
    __shared__ u64 wsum[kSliceNW];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
    float x[kSteps][kPer];
    const int i0 = s * kSlice + tid * kPer;
    load_slice(static_cast<const T *>(a.logits) + (long)r * a.stride, s * kSlice, a.vocab, x);
    const Row row = row_of(a, r);
    if (row.cuts())
        for (int i = tid; i < kBins * kCopies; i += kSliceNT) sum[i] = 0, count[i] = 0;
    float most = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            bad |= !(x[i][e] < INFINITY);
            most = fmaxf(most, x[i][e]);
        }
    most = wave_max_f(most);
    const bool any = __any(bad);
    int at = INT_MAX;
    if (row.greedy) {
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i)
#pragma unroll
            for (int e = kPer - 1; e >= 0; --e)
                if (x[i][e] == most) at = i0 + i * (kSliceNT * kPer) + e;
        at = wave_min_i(at);
    }
    if (lane == 0) wm[wv] = most, wi[wv] = at, wbad[wv] = any;
    __syncthreads();
    most = wm[0], at = wi[0];
    int bads = wbad[0];
#pragma unroll
    for (int w = 1; w < kSliceNW; ++w) {
        if (wm[w] > most) at = wi[w];
        else if (wm[w] == most) at = min(at, wi[w]);
        most = fmaxf(most, wm[w]);
        bads |= wbad[w];
    }
    SliceHead h{0.0, most, at, 0, bads || row.bad};
    if (s == 0 && tid == 0) wk.rows[r].listed = 0;
    if (row.greedy || h.bad || most == -INFINITY) {
        if (tid == 0) wk.heads[blockIdx.x] = h;
        return;
    }
    if (!row.cuts()) {
        double t = 0.0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
            for (int e = 0; e < kPer; ++e) t += row.e(x[i][e], most);   // of -inf 2^-1000: nothing beside the largest's 1
        t = wave_sum_d(t);
        if (lane == 0) wt[wv] = t;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kSliceNW; ++w) h.total += wt[w];
            wk.heads[blockIdx.x] = h;
        }
        return;
    }
    h.top = row.bin(most);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {           // eight chains of products at once; what is not drawn to the last bin
        int b[kPer];
        u64 q[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            b[e] = row.behind(h.top, x[i][e]) * kCopies + (lane & (kCopies - 1));
            q[e] = fixed(row.e(x[i][e], most), kFrac);
        }
#pragma unroll
        for (int e = 0; e < kPer; ++e) atomicAdd(&sum[b[e]], q[e]);
        if (row.k_cut)
#pragma unroll
            for (int e = 0; e < kPer; ++e) atomicAdd(&count[b[e]], 1u);
    }
    __syncthreads();
    static_assert(kSliceNT == kBins, "a thread for each bin");
    u64 t = 0;
    int n = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {          // each lane begins at a copy of its own: other banks
        const int i = tid * kCopies + ((c + tid) & (kCopies - 1));
        t += sum[i], n += (int)count[i];
    }
    if (tid == kBins - 1) t = 0, n = 0;
    t = wave_scan_u(t);
    n = wave_scan_i(n);
    if (lane == 63) wsum[wv] = t, wi[wv] = n;
    __syncthreads();
    for (int w = 0; w < wv; ++w) t += wsum[w], n += wi[w];
    wk.bins[blockIdx.x].upto[tid] = Bin{t, (unsigned)n, 0};
    if (tid == 0) wk.heads[blockIdx.x] = h;
}

namespace {
struct CutLds {
    double scale[kMostSlices];           // e of a slice's largest logit
    int off[kMostSlices];                // bins that the slice's first one is behind the row's
    double wsum[kBins];                  // the row's bins: sums and counts up to and with the bin
    int wcount[kBins];
    unsigned key;
};
// scale and off of all slices.
__device__ __forceinline__ void load_slices(CutLds &L, const Row &row, const RowHead &h, const SliceHead *heads, int S) {
    for (int s = threadIdx.x; s < S; s += blockDim.x) {
        const SliceHead x = s < 64 ? h.mine : heads[s];    // of the first wave
        L.scale[s] = x.most == -INFINITY ? 0.0 : row.e(x.most, h.most);
        L.off[s] = slice_off(x, h.top);
    }
    __syncthreads();
}
// The row's bins, a thread for each, the slices in order; the last as the one before it, as a slice's are: a
// slice whose first bin is behind the row's has tokens there, and they are not drawn.
__device__ __forceinline__ void add_bins(CutLds &L, const SliceBins *bins, int S) {
    constexpr int kAtOnce = 20;                  // slices' loads in flight
    const int j = min((int)threadIdx.x, kBins - 2);
    double w = 0.0;
    int n = 0;
    for (int s0 = 0; s0 < S; s0 += kAtOnce) {
        u4_t t[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int s = min(s0 + i, S - 1);
            t[i] = *reinterpret_cast<const u4_t *>(&bins[s].upto[max(j - L.off[s], 0)]);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int s = min(s0 + i, S - 1);
            const bool in = (s0 + i < S) & (j >= L.off[s]);
            const double sum = (double)((u64)t[i][1] << 32 | t[i][0]) * L.scale[s];
            w += in ? sum : 0.0;
            n += in ? (int)t[i][2] : 0;
        }
    }
    L.wsum[threadIdx.x] = w * 0x1p-50, L.wcount[threadIdx.x] = n;
    __syncthreads();
}
// The first bin that reaches `need`, or kBins: none does; sums and counts never fall from bin to bin.
// Every wave finds it by itself.
__device__ __forceinline__ int reaches(const CutLds &L, bool by_sum, double need) {
    int before = 0;
#pragma unroll
    for (int i = 0; i < kBins; i += 64) {
        const int j = i + (threadIdx.x & 63);
        before += __popcll(__ballot((by_sum ? L.wsum[j] : (double)L.wcount[j]) < need));
    }
    return before;
}
// The lowest finite key up to the largest logit's with e >= m, by one wave (e rises with the logit).
__device__ __forceinline__ unsigned key_of_e(const Row &row, float most) {
    const int lane = threadIdx.x & 63;
    unsigned lo = key_of(-FLT_MAX), hi = key_of(most);
    while (lo < hi) {                            // 64 probes at once, six or seven times
        const unsigned step = (hi - lo) / 64 + 1, probe = min(lo + lane * step, hi);
        const u64 yes = __ballot(row.e(of_key(probe), most) >= row.m);
        const int f = yes ? __ffsll(yes) - 1 : 64;
        if (f < 64) hi = min(lo + f * step, hi);
        if (f > 0) lo = min(lo + (f - 1) * step + 1, hi);
    }
    return lo;
}
// Which bins the cuts fall into: top-k's, those that top-p's may (its sum is known only between two
// bounds while top-k's cut is not selected), min-p's; kBins: no cut there.
struct CutBins {
    int k, p0, p1, m;
    unsigned m_key;
    int pad;
    // Bits 32 w .. 32 w + 31 of the set of them.
    __device__ __forceinline__ unsigned word(int w) const {
        unsigned bits = 0;
        for (int i = 0; i < 32; ++i) {
            const int b = w * 32 + i;
            bits |= (unsigned)((b < kBins - 1) & ((b == k) | ((b >= p0) & (b <= p1)) | (b == m))) << i;
        }
        return bits;
    }
};
__device__ __forceinline__ CutBins cut_bins(CutLds &L, const Row &row, const RowHead &h) {
    CutBins c{kBins, kBins, kBins - 1, kBins, 0, 0};
    double low = L.wsum[kBins - 1], high = low;
    if (row.m_cut) {
        if (threadIdx.x < 64) {
            const unsigned key = key_of_e(row, h.most);
            if (threadIdx.x == 0) L.key = key;
        }
        __syncthreads();
        c.m_key = L.key;
        c.m = h.top - row.bin(of_key(c.m_key));
        if (c.m >= kBins - 1) c.m = kBins;
    }
    if (row.k_cut && L.wcount[kBins - 1] > row.k) {
        c.k = reaches(L, false, row.k);
        low = c.k ? L.wsum[c.k - 1] : 0.0, high = L.wsum[c.k];
    }
    if (row.p_cut) {
        c.p0 = reaches(L, true, row.p * low);
        c.p1 = min(reaches(L, true, row.p * high), kBins - 1);
    }
    return c;
}
}  // namespace

// Workgroup row * slices + slice: its tokens of the cuts' bins to the row's list; the first slice's
// leaves the row's bins too.
template <typename T>
__global__ __launch_bounds__(kSliceNT) void sample_list_kernel(SampleParams a, Work wk) {
    __shared__ CutLds L;
    __shared__ unsigned found, base, words[kBins / 32];
    const int tid = threadIdx.x, r = blockIdx.x / a.slices, s = blockIdx.x % a.slices, S = a.slices;
    const SliceHead *heads = wk.heads + (long)r * S;
    const Row row = row_of(a, r);
    if (!row.cuts() || row.greedy || row.bad) return;
    const RowHead h = row_head(row, heads, S);
    if (h.bad || h.most == -INFINITY) return;
    if (tid == 0) found = 0;
    load_slices(L, row, h, heads, S);
    add_bins(L, wk.bins + (long)r * S, S);
    if (s == 0) wk.rows[r].sum[tid] = L.wsum[tid], wk.rows[r].count[tid] = L.wcount[tid];
    // loaded no earlier: the registers that they take leave room for fewer waves beside this one
    float x[kSteps][kPer];
    const int i0 = s * kSlice + tid * kPer;
    load_slice(static_cast<const T *>(a.logits) + (long)r * a.stride, s * kSlice, a.vocab, x);
    const CutBins cut = cut_bins(L, row, h);
    if (s == 0 && tid == 0) *reinterpret_cast<CutBins *>(wk.rows[r].cut) = cut;
    if (L.off[s] >= kBins) return;
    if (tid < kBins / 32) words[tid] = cut.word(tid);
    __syncthreads();
    // No logit below it is in the cuts' bins, so that few need the product that finds a logit's bin (256 rows of
    // 151936 with top-k 50 and top-p 0.9: 55 to 45 us; a cut that keeps most tokens takes 0.3 us more).
    const int lowest = max(max(cut.k < kBins - 1 ? cut.k : 0, cut.m < kBins - 1 ? cut.m : 0), cut.p0 <= cut.p1 ? cut.p1 : 0);
    const double under = ((double)(h.top - lowest) - 1.0) / row.bins;
    const float least = under > -(double)row.limit ? (float)(under - fabs(under) * 0x1p-20) : -INFINITY;
    float most[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        most[i] = x[i][0];
#pragma unroll
        for (int e = 1; e < kPer; ++e) most[i] = fmaxf(most[i], x[i][e]);
    }
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        if (!__any(most[i] >= least)) continue;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int b = row.behind(h.top, x[i][e]);
            mine |= (words[b >> 5] >> (b & 31) & 1) << (i * kPer + e);
        }
    }
    // places in the list: of the wave's tokens, of the workgroup's, of the row's
    const int n = __popc(mine), upto = wave_scan_i(n), all = __builtin_amdgcn_readlane(upto, 63);
    unsigned at = 0;
    if ((tid & 63) == 0 && all) at = atomicAdd(&found, (unsigned)all);
    at = __builtin_amdgcn_readfirstlane(at) + (unsigned)(upto - n);
    __syncthreads();
    if (found == 0) return;
    if (tid == 0) base = atomicAdd(&wk.rows[r].listed, found);
    __syncthreads();
    uint2 *to = wk.list + (long)r * a.vocab + base + at;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            if (mine >> (i * kPer + e) & 1)
                *to++ = make_uint2(key_of(x[i][e]), (unsigned)(i0 + i * (kSliceNT * kPer) + e) |
                                                        (unsigned)(h.top - row.bin(x[i][e])) << 24);
}

namespace {
struct Found {                           // a digit, the sum and count of what lies above it, its own count
    u64 above;
    int digit, counts, count, pad;
};
struct RowLds {
    CutLds c;
    u64 hsum[2][kDigits];                // a digit's sums, counts: one set in use, the other cleared
    unsigned hcount[2][kDigits];
    uint2 list[kList];
    double kept[kMostSlices];
    u64 csum[kMostSlices];               // of the cut's bin: sum of e above kappa, tokens at kappa
    int cties[kMostSlices];
    double dw[kNW], rest;
    unsigned kmin[2], kmax[2];
    u64 uw[kDigits / 64];
    Found found[kDigits / 64];
    int iw[kNW], hit, last, slice, before;
};

// The selection among the row's listed tokens.
template <typename T>
struct Chosen {
    // low bits of a key that T's values have alike: of bf16 16, of fp16 13
    static constexpr int kLow = sizeof(T) == 4 ? 0 : __is_same(T, __half) ? 13 : 16;
    const Row &row;
    RowLds &L;
    const RowHead &h;
    const uint2 *list;
    int n;                               // tokens of the list; in LDS if kList of them are enough
    int frac;                            // bits behind the point of a bin's sums
    int set;                             // of the digits' sums and counts, the one that is clear

    // f(index, key, e relative to the logit `top`) for the listed tokens of bin b; with_e: e is formed, for four
    // tokens at once
    template <bool with_e, typename F>
    __device__ __forceinline__ void each(int b, double top, F f) const {
        constexpr int kAtOnce = 4;
        for (int i0 = threadIdx.x; i0 < n; i0 += kAtOnce * kNT) {
            uint2 t[kAtOnce];
            double e[kAtOnce];
            if (n <= kList) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) t[i] = L.list[min(i0 + i * kNT, n - 1)];
            } else {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) t[i] = list[min(i0 + i * kNT, n - 1)];
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) e[i] = with_e ? row.e(of_key(t[i].x), top) : 0.0;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (i0 + i * kNT < n && (int)(t[i].y >> 24) == b) f((int)(t[i].y & 0xffffffu), t[i].x, e[i]);
        }
    }
    // The key of T's values whose high bits they are.
    static __device__ __forceinline__ unsigned whole_key(unsigned high) {
        const unsigned k = high << kLow;
        return kLow && k < 0x80000000u ? k | ((1u << kLow) - 1) : k;       // a negative value's low bits are ones
    }
    // Of the tokens of bin b, in falling order: the key at which `need` of them (by_sum: of their sum of
    // e) are reached, and how many of that key it takes; *sum: their sum of e up to there.  Digit by digit
    // of the key's distance to the bin's lowest, without the bits that T's values never use.  call: 0, 1.
    __device__ void select(int call, int b, bool by_sum, double need, unsigned *kappa, int *ties, double *sum) {
        unsigned kmin = 0xffffffffu, kmax = 0;
        each<false>(b, 0.0, [&](int, unsigned k, double) { kmin = min(kmin, k), kmax = max(kmax, k); });
        kmin = (unsigned)wave_min_i((int)(kmin ^ 0x80000000u)) ^ 0x80000000u;
        kmax = ~((unsigned)wave_min_i((int)(~kmax ^ 0x80000000u)) ^ 0x80000000u);
        if ((threadIdx.x & 63) == 0 && kmin <= kmax) atomicMin(&L.kmin[call], kmin), atomicMax(&L.kmax[call], kmax);
        __syncthreads();
        const double top = row.bin_top(b, h.top, h.most);
        if (by_sum) need *= row.e(h.most, top);
        kmin = L.kmin[call] >> kLow, kmax = L.kmax[call] >> kLow;
        unsigned prefix = 0;
        // all in whole numbers, sums with frac bits behind the point: exactly one digit is the first to reach
        u64 above = 0;                   // sum of what lies above the prefix
        int counts = 0, last_count = 0;  // tokens above it, tokens of it
        // of one key alone this is one pass, of no token none
        for (int shift = kmin <= kmax ? (31 - __clz((kmax - kmin) | 1u)) / kDigitBits * kDigitBits : -1; shift >= 0;
             shift -= kDigitBits) {
            u64 *hsum = L.hsum[set];
            unsigned *hcount = L.hcount[set];
            set ^= 1;
            auto add = [&](int, unsigned k, double e) {
                const unsigned q = (k >> kLow) - kmin;
                if ((u64)(q ^ prefix) >> (shift + kDigitBits)) return;
                if (shift) atomicAdd(&hsum[q >> shift & (kDigits - 1)], fixed(e, frac));
                atomicAdd(&hcount[q >> shift & (kDigits - 1)], 1u);
            };
            // the last digit's tokens have one key each: their sum is a multiple of its e
            if (shift) each<true>(b, top, add);
            else each<false>(b, top, add);
            __syncthreads();
            // a digit for each of the first threads, the largest first
            const int d = kDigits - 1 - (int)threadIdx.x, w = threadIdx.x / 64;
            u64 mine = 0, upto = 0;
            int c = 0, n_upto = 0;
            if (threadIdx.x < kDigits) {
                c = (int)hcount[d];
                const double e = row.e(fmin((double)of_key(whole_key((prefix | (unsigned)d) + kmin)), top), top);
                mine = shift ? hsum[d] : c ? c * fixed(e, frac) : 0;                // no token: e of any key
                upto = wave_scan_u(mine), n_upto = wave_scan_i(c);
                if ((threadIdx.x & 63) == 63) L.uw[w] = upto, L.iw[w] = n_upto;
                L.hsum[set][d] = 0, L.hcount[set][d] = 0;
            }
            __syncthreads();
            if (threadIdx.x < kDigits) {
                u64 before = above, all = above;
                int n_before = counts;
#pragma unroll
                for (int i = 0; i < kDigits / 64; ++i) {
                    if (i < w) before += L.uw[i], n_before += L.iw[i];
                    all += L.uw[i];
                }
                // what rounding leaves unreached is all of it
                const u64 goal = by_sum ? min((u64)ceil(fmax(ldexp(need, frac), 0.0)), all) : 0;
                const bool there = c && (by_sum ? before + upto >= goal : n_before + n_upto >= (int)need);
                const u64 who = __ballot(there);
                if ((threadIdx.x & 63) == 0) L.found[w].digit = -1;
                if (there && (threadIdx.x & 63) == __ffsll(who) - 1)
                    L.found[w] = Found{before + (upto - mine), d, n_before + n_upto - c, c, 0};
            }
            __syncthreads();
            Found f = L.found[0];
#pragma unroll
            for (int i = 1; i < kDigits / 64; ++i)
                if (f.digit < 0) f = L.found[i];
            prefix |= (unsigned)f.digit << shift;
            above = f.above, counts = f.counts, last_count = f.count;
        }
        const double sums = (double)above * ldexp(1.0, -frac);
        prefix = whole_key(prefix + kmin);
        const double e = row.e(of_key(prefix), top);
        double t = by_sum ? ceil((need - sums) / e) : need - counts;
        t = fmin(fmax(t, 1.0), (double)last_count);
        *kappa = prefix;
        *ties = (int)t;
        *sum = (sums + t * e) * row.e(top, h.most);
    }
};
}  // namespace

// Workgroup = row.
template <typename T>
__global__ __launch_bounds__(kNT) void sample_row_kernel(SampleParams a, Work wk) {
    __shared__ RowLds L;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = blockIdx.x, S = a.slices;
    const SliceHead *heads = wk.heads + (long)r * S;
    const SliceBins *bins = wk.bins + (long)r * S;
    const Row row = row_of(a, r);
    const RowHead h = row_head(row, heads, S);
    if (h.bad || row.bad || h.most == -INFINITY || row.greedy) {
        if (tid == 0) a.tokens[r] = h.bad || row.bad || h.most == -INFINITY ? -1 : h.at;
        return;
    }
    for (int s = tid; s < S; s += kNT) L.csum[s] = 0, L.cties[s] = 0;
    if (tid < 2) L.kmin[tid] = 0xffffffffu, L.kmax[tid] = 0;
    if (tid < kDigits) L.hsum[0][tid] = 0, L.hcount[0][tid] = 0;
    if (tid == 0) L.hit = INT_MAX, L.last = -1;
    unsigned kappa = 0;
    int ties = INT_MAX, jc = kBins - 1;
    const int frac = min(kFrac, 62 - (32 - __clz(a.vocab)));   // a sum of e of all tokens fits
    if (row.cuts()) {
        const RowBins &of = wk.rows[r];
        Chosen<T> d{row, L, h, wk.list + (long)r * a.vocab, (int)of.listed, frac, 0};
        const CutBins cut = *reinterpret_cast<const CutBins *>(of.cut);
        if (tid < kBins) L.c.wsum[tid] = of.sum[tid], L.c.wcount[tid] = of.count[tid];
        if (d.n <= kList)
            for (int i = tid; i < d.n; i += kNT) L.list[i] = d.list[i];
        load_slices(L.c, row, h, heads, S);
        double all = L.c.wsum[kBins - 1];
        if (cut.k < kBins) {
            const int j = cut.k;
            double sum;
            d.select(0, j, false, (double)row.k - (j ? L.c.wcount[j - 1] : 0), &kappa, &ties, &sum);
            all = (j ? L.c.wsum[j - 1] : 0.0) + sum;
        }
        if (row.p_cut) {
            const double need = row.p * all;
            const int j = min(max(reaches(L.c, true, need), cut.p0), cut.p1);
            if (j < kBins - 1) {
                unsigned key;
                int n;
                double sum;
                d.select(1, j, true, need - (j ? L.c.wsum[j - 1] : 0.0), &key, &n, &sum);
                if (key > kappa) kappa = key, ties = n;
                else if (key == kappa) ties = min(ties, n);
            }
        }
        if (row.m_cut && cut.m_key > kappa) kappa = cut.m_key, ties = INT_MAX;
        // the bin of the cut; a slice keeps its bins before that, and of its tokens in that bin those above kappa
        if (kappa) jc = min(max(h.top - row.bin(of_key(kappa)), 0), kBins - 1);
        d.template each<true>(jc, row.bin_top(jc, h.top, h.most), [&](int i, unsigned k, double e) {
            if (k > kappa) atomicAdd(&L.csum[i / kSlice], fixed(e, kFrac));      // a slice's, as its bins'
            if (k == kappa) atomicAdd(&L.cties[i / kSlice], 1);
        });
        __syncthreads();
    } else {
        load_slices(L.c, row, h, heads, S);
    }
    // the slice that the draw falls into
    if (wv == 0) {
        const int per = (S + 63) / 64, s0 = min(S, lane * per), s1 = min(S, s0 + per);
        int before = 0;
        for (int s = s0; s < s1; ++s) before += L.cties[s];
        before = wave_scan_i(before) - before;   // ties of the slices before
        const int ties0 = before;
        const double e = kappa ? row.e(of_key(kappa), h.most) : 0.0;
        const double unit = row.e(row.bin_top(jc, h.top, h.most), h.most) * 0x1p-50;     // of csum
        double mine = 0.0;
        for (int s = s0; s < s1; ++s) {
            const int b = jc - 1 - L.c.off[s];
            const double w = !row.cuts() ? heads[s].total : b >= 0 ? (double)bins[s].upto[b].sum * 0x1p-50 : 0.0;
            L.kept[s] = w * L.c.scale[s] + (double)L.csum[s] * unit + (double)min(max(ties - before, 0), L.cties[s]) * e;
            before += L.cties[s];
            mine += L.kept[s];
        }
        const double incl = wave_scan_d(mine), total = lane_d(incl, 63);
        double u = (double)a.uniform[a.step ? *a.step : r];
        u = u >= 0.0 ? fmin(u, 1.0) : 0.0;       // NaN: 0
        const double t = u * total;
        double run = incl - mine, rest = 0.0;
        int pick = INT_MAX, last = -1, pick_ties = 0, last_ties = 0;
        before = ties0;
        for (int s = s0; s < s1; ++s) {
            // a slice that keeps any token keeps its largest
            const bool some = L.kept[s] > 0.0 && L.c.scale[s] >= kLeast;
            if (some) last = s, last_ties = before;
            if (pick == INT_MAX && some && run + L.kept[s] > t) pick = s, pick_ties = before, rest = t - run;
            run += L.kept[s];
            before += L.cties[s];
        }
        const int slice = wave_min_i(pick), end = -wave_min_i(-last);
        if (slice != INT_MAX && pick == slice) L.slice = slice, L.rest = rest, L.before = pick_ties;
        // u = 1, or a rounding at the end: the last token
        if (slice == INT_MAX && last == end) L.slice = end, L.rest = INFINITY, L.before = last_ties;
    }
    __syncthreads();
    const int s = L.slice, i0 = s * kSlice + tid * kPer;
    const double rest = L.rest;
    float x[kPer];
    load_logits(static_cast<const T *>(a.logits) + (long)r * a.stride, i0, a.vocab, x);
    // ties before the thread's tokens
    int mine = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += kappa && i0 + e < a.vocab && key_of(x[e]) == kappa;
    const int incl = wave_scan_i(mine);
    if (lane == 63) L.iw[wv] = incl;
    __syncthreads();
    int before = L.before + incl - mine;
    for (int w = 0; w < wv; ++w) before += L.iw[w];
    double e[kPer], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const unsigned k = key_of(x[i]);         // kappa 0: below every key
        const bool same = k == kappa, keep = (k > kappa) | (same & (before < ties));
        before += same;
        e[i] = 0.0;
        const bool some = keep & (x[i] > -INFINITY);       // not past the end
        if (__any(some)) {                       // few of a cut's tokens are kept
            const double v = row.e(x[i], h.most);
            e[i] = some ? v : 0.0;
        }
        sum += e[i];
    }
    const double scan = wave_scan_d(sum);
    if (lane == 63) L.dw[wv] = scan;
    __syncthreads();
    double run = scan - sum;
    {
        double w0 = 0.0;
        for (int w = 0; w < wv; ++w) w0 += L.dw[w];
        run += w0;
    }
    int hit = INT_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        run += e[i];
        if (e[i] >= kLeast) {
            last = i0 + i;
            if (hit == INT_MAX && run > rest) hit = i0 + i;
        }
    }
    const int whit = wave_min_i(hit), wlast = -wave_min_i(-last);
    if (lane == 0) {
        atomicMin(&L.hit, whit);
        atomicMax(&L.last, wlast);
    }
    __syncthreads();
    if (tid == 0) a.tokens[r] = L.hit == INT_MAX ? L.last : L.hit;
}

namespace {
template <typename T>
void sample(const SampleParams &a, const Work &wk, hipStream_t st) {
    const dim3 slices((unsigned)a.rows * a.slices);
    OJX_LAUNCH((sample_slice_kernel<T>), slices, dim3(kSliceNT), 0, st, a, wk);
    // no row can have a cut: nothing to list
    if (a.top_ks || a.top_ps || a.min_ps || (a.top_k > 0 && a.top_k < a.vocab) || a.top_p < 1.0 || a.min_p > 0.0)
        OJX_LAUNCH((sample_list_kernel<T>), slices, dim3(kSliceNT), 0, st, a, wk);
    OJX_LAUNCH((sample_row_kernel<T>), dim3(a.rows), dim3(kNT), 0, st, a, wk);
}
}  // namespace

long sample_workspace(int rows, int vocab) {
    if (rows < 0 || vocab <= 0 || vocab > kMostSlices * kSlice) {
        set_error("sampling: %d rows of %d logits (1 to 2^22)", rows, vocab);
        return OJASX_ERR_INVALID;
    }
    const long slices = ((long)vocab + kSlice - 1) / kSlice;
    if (rows * slices > 0x3fffffL) {             // a grid has fewer than 2^32 threads
        set_error("sampling: %d rows of %d logits are more than a launch takes", rows, vocab);
        return OJASX_ERR_INVALID;
    }
    return rows * (slices * (long)(sizeof(SliceHead) + sizeof(SliceBins)) + (long)sizeof(RowBins) +
                   (long)round_up((size_t)vocab * sizeof(uint2), 16));
}

int launch_sample(SampleParams a, int dtype, void *workspace, hipStream_t st) {
    a.slices = (a.vocab + kSlice - 1) / kSlice;
    Work wk;
    const long n = (long)a.rows * a.slices;
    wk.bins = static_cast<SliceBins *>(workspace);
    wk.heads = reinterpret_cast<SliceHead *>(wk.bins + n);
    wk.rows = reinterpret_cast<RowBins *>(wk.heads + n);
    wk.list = reinterpret_cast<uint2 *>(wk.rows + a.rows);
    if (dtype == OJASX_DTYPE_F32) sample<float>(a, wk, st);
    else if (dtype == OJASX_DTYPE_BF16) sample<__hip_bfloat16>(a, wk, st);
    else sample<__half>(a, wk, st);
    OJX_HIP(hipGetLastError());
    return OJASX_OK;
}

int check_sampling(double temperature, double top_p, double min_p) {
    if (!(temperature >= 0.0 && temperature <= (double)FLT_MAX) || !(top_p >= 0.0) || !(min_p >= 0.0 && min_p <= 1.0)) {
        set_error("sampling: temperature %g, top_p %g, min_p %g", temperature, top_p, min_p);
        return OJASX_ERR_INVALID;
    }
    return OJASX_OK;
}

}  // namespace ojx

extern "C" {

OJASX_API long ojasx_sample_workspace(int num_rows, int vocab) { return ojx::sample_workspace(num_rows, vocab); }

OJASX_API int ojasx_sample_device(const void *logits, int dtype, int num_rows, int vocab, long row_stride,
                                  const float *uniform, const OjasxSampling *settings, int *tokens, void *workspace,
                                  long workspace_bytes, void *stream) {
    using namespace ojx;
    const long need = sample_workspace(num_rows, vocab);
    if (need < 0) return (int)need;
    if (dtype != OJASX_DTYPE_F32 && dtype != OJASX_DTYPE_BF16 && dtype != OJASX_DTYPE_F16) {
        set_error("unsupported dtype %d", dtype);
        return OJASX_ERR_INVALID;
    }
    if (!settings) return OJASX_ERR_NULL;
    // a value that an array replaces is not looked at
    const OjasxSampling &s = *settings;
    int rc = check_sampling(s.temperatures ? 1.0 : s.temperature, s.top_ps ? 1.0 : s.top_p, s.min_ps ? 0.0 : s.min_p);
    if (rc) return rc;
    if (num_rows == 0) return OJASX_OK;
    if (!logits || !uniform || !tokens) return OJASX_ERR_NULL;
    if (row_stride < 0 || (reinterpret_cast<uintptr_t>(logits) & (dtype == OJASX_DTYPE_F32 ? 3 : 1))) {
        set_error("sampling: row stride %ld, or logits that are not aligned", row_stride);
        return OJASX_ERR_INVALID;
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need) {
        set_error("sampling: the workspace has to be 16-byte aligned and of %ld bytes, got %ld", need, workspace_bytes);
        return OJASX_ERR_INVALID;
    }
    SampleParams a{};
    a.logits = logits, a.stride = row_stride, a.rows = num_rows, a.vocab = vocab;
    a.uniform = uniform, a.tokens = tokens;
    a.temperature = s.temperature, a.temperatures = s.temperatures;
    a.top_k = s.top_k, a.top_ks = s.top_ks;
    a.top_p = s.top_p, a.top_ps = s.top_ps;
    a.min_p = s.min_p, a.min_ps = s.min_ps;
    return launch_sample(a, dtype, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
