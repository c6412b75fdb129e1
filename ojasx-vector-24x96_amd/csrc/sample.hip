// sample.hip -- one token of every row of logits, drawn with a given random number.
//
//   e_i = exp((l_i - max l) / T); the tokens in order of falling l, equal ones of rising index;
//   top-k: the first k of them; top-p: of those the shortest beginning whose sum of e is at least
//   p times all of theirs; min-p: of those the ones with e_i >= m; token: the first of the kept
//   ones, in the vocabulary's order, at which the running sum of e passes u times their sum.
//
// All three cuts keep a beginning of one order, so together they are one logit kappa and a count:
// kept is what lies above kappa, and of the tokens that equal it the first `ties`.  No sort: the
// first kernel counts, by slices of the vocabulary, tokens and sums of e in 255 bins of the logit
// (width T / 7, on one grid for all slices, from the slice's largest down to where e is
// below 2^-51 of it and is not drawn); the second, a workgroup per row, adds the slices' bins,
// finds the bin that a cut falls into, takes that bin's tokens from the row and selects among
// them byte by byte of their logits' order; then it finds the slice that the draw falls into from
// the slices' kept sums, and the token within it.
//
// A drawn token is a whole number: it has to be the definition's own.  So e is fp64 to about
// 2^-50, sums are fp64, or in LDS, where they are added in any order, 64-bit integers: a fixed
// number of bits behind the point, the same result in every order.
#include <cfloat>
#include <climits>
#include <cmath>

#include "sample.h"

namespace ojx {

namespace {
constexpr int kNT = 1024;
constexpr int kNW = kNT / 64;
constexpr int kPer = 8;                  // tokens of a thread
constexpr int kSlice = kNT * kPer;
constexpr int kBins = 256;               // the last: e below kLeast
constexpr int kCopies = 4;               // of the bins' counters, so that a wave's lanes collide less
constexpr double kBinsPerE = 7.0;        // 255 / 7 = 36.4 > 51 ln 2
constexpr int kFrac = 50;                // bits behind the point of a slice's sums (8192 of them: 2^63)
constexpr int kList = 8192;              // tokens of a bin that are selected among in LDS
constexpr int kMostSlices = 512;
constexpr double kLeast = 0x1p-51;       // tokens of a smaller e are not drawn

typedef unsigned long long u64;

struct SliceHead {
    double top;                          // bin of the slice's largest logit
    double total;                        // rows without cuts: the slice's sum of e, relative to its largest
    float most;
    int at;                              // index of the largest logit
    int bad;                             // a NaN or +inf among the logits
    int pad;
};
struct SliceBins {
    u64 sum[kBins];
    unsigned count[kBins];
};

// 2^x for x <= 0, to about 2^-52: 2^f as its Taylor polynomial of degree 12, |f| <= 1/2 (the next
// term is below 2^-52), scaled by the exponent; below 2^-1000: that.
__device__ __forceinline__ double exp2_f64(double x) {
    x = fmax(x, -1000.0);
    const double n = rint(x), f = x - n;
    constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4,
                     c5 = c4 * c1 / 5, c6 = c5 * c1 / 6, c7 = c6 * c1 / 7, c8 = c7 * c1 / 8, c9 = c8 * c1 / 9,
                     c10 = c9 * c1 / 10, c11 = c10 * c1 / 11, c12 = c11 * c1 / 12;
    double p = fma(c12, f, c11);
    p = fma(p, f, c10);
    p = fma(p, f, c9);
    p = fma(p, f, c8);
    p = fma(p, f, c7);
    p = fma(p, f, c6);
    p = fma(p, f, c5);
    p = fma(p, f, c4);
    p = fma(p, f, c3);
    p = fma(p, f, c2);
    p = fma(p, f, c1);
    return ldexp(fma(p, f, 1.0), (int)n);
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
    double c, bins;                      // log2(e) / T, bins per unit of the logit
    double p, m;
    int k;
    bool greedy, bad, k_cut, p_cut, m_cut;
    __device__ __forceinline__ bool cuts() const { return k_cut || p_cut || m_cut; }
};
__device__ __forceinline__ Row row_of(const SampleParams &a, int r) {
    Row s;
    const double T = a.temperatures ? (double)a.temperatures[r] : a.temperature;
    s.k = a.top_ks ? a.top_ks[r] : a.top_k;
    s.p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
    s.m = fmin(a.min_ps ? (double)a.min_ps[r] : a.min_p, 1.0);
    s.bad = !(T >= 0.0) || T > (double)FLT_MAX;
    s.greedy = T == 0.0;
    s.c = 1.4426950408889634074 / T;
    s.bins = kBinsPerE / T;
    s.k_cut = s.k > 0 && s.k < a.vocab;
    s.p_cut = s.p < 1.0;
    s.m_cut = s.m > 0.0;
    return s;
}

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }

// Eight logits from i on (i a multiple of 8), -inf past the vocabulary's end.
template <typename T>
__device__ __forceinline__ void load_logits(const T *row, int i, int V, float (&x)[kPer]) {
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && i + kPer <= V) {
        load8(row + i, x);
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[e] = i + e < V ? as_f32(row[i + e]) : -INFINITY;
    }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double wave_scan_d(double v) {       // with this lane's
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(v, o);
        if ((threadIdx.x & 63) >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ int wave_scan_i(int v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(v, o);
        if ((threadIdx.x & 63) >= o) v += x;
    }
    return v;
}
}  // namespace

// Workgroup row * slices + slice.
template <typename T>
__global__ __launch_bounds__(kNT) void sample_slice_kernel(SampleParams a, SliceHead *heads, SliceBins *bins) {
    __shared__ u64 sum[kBins * kCopies];
    __shared__ unsigned count[kBins * kCopies];
    __shared__ float wm[kNW];
    __shared__ int wi[kNW], wbad[kNW];
    __shared__ double wt[kNW];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int r = blockIdx.x / a.slices, s = blockIdx.x % a.slices;
    const Row row = row_of(a, r);
    float x[kPer];
    const int i0 = s * kSlice + tid * kPer;
    load_logits(static_cast<const T *>(a.logits) + (long)r * a.stride, i0, a.vocab, x);
    float most = -INFINITY;
    int at = INT_MAX;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        bad |= !(x[e] < INFINITY);
        if (x[e] > most) most = x[e], at = i0 + e;
    }
    const float wmost = wave_max_f(most);
    const int wat = wave_min_i(most == wmost ? at : INT_MAX);
    const bool any = __any(bad);
    if (lane == 0) wm[wv] = wmost, wi[wv] = wat, wbad[wv] = any;
    for (int i = tid; i < kBins * kCopies; i += kNT) sum[i] = 0, count[i] = 0;
    __syncthreads();
    most = wm[0], at = wi[0];
    int bads = wbad[0];
#pragma unroll
    for (int w = 1; w < kNW; ++w) {
        if (wm[w] > most || (wm[w] == most && wi[w] < at)) at = wi[w];
        most = fmaxf(most, wm[w]);
        bads |= wbad[w];
    }
    SliceHead *head = heads + blockIdx.x;
    SliceHead h{0.0, 0.0, most, at, bads || row.bad, 0};
    if (row.greedy || h.bad || most == -INFINITY) {
        if (tid == 0) *head = h;
        // a slice of -inf: empty bins, which the second kernel adds
        if (!row.greedy && !h.bad && row.cuts())
            for (int i = tid; i < kBins; i += kNT) bins[blockIdx.x].sum[i] = 0, bins[blockIdx.x].count[i] = 0;
        return;
    }
    if (!row.cuts()) {
        double t = 0.0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) t += x[e] == -INFINITY ? 0.0 : exp2_f64(((double)x[e] - (double)most) * row.c);
        t = wave_sum_d(t);
        if (lane == 0) wt[wv] = t;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < kNW; ++w) h.total += wt[w];
            *head = h;
        }
        return;
    }
    h.top = floor((double)most * row.bins);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const double d = h.top - floor((double)x[e] * row.bins);
        if (d < kBins - 1) {                     // of -inf: no
            const int b = (int)d * kCopies + (lane & (kCopies - 1));
            atomicAdd(&sum[b], fixed(exp2_f64(((double)x[e] - (double)most) * row.c), kFrac));
            atomicAdd(&count[b], 1u);
        }
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kNT) {
        u64 t = 0;
        unsigned n = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) t += sum[i * kCopies + c], n += count[i * kCopies + c];
        bins[blockIdx.x].sum[i] = t;
        bins[blockIdx.x].count[i] = n;
    }
    if (tid == 0) *head = h;
}

namespace {
struct RowLds {
    u64 hsum[kBins];                     // a digit's sums, counts
    unsigned hcount[kBins];
    double wsum[kBins];                  // the row's bins: sums and counts up to and with the bin
    int wcount[kBins];
    double gsum[4][kBins];
    int gcount[4][kBins];
    unsigned lkey[kList];
    int lidx[kList];
    double scale[kMostSlices];           // e of a slice's largest logit
    double kept[kMostSlices];
    int off[kMostSlices];                // bins that the slice's first one is behind the row's
    u64 csum[kMostSlices];               // of the cut's bin: sum of e above kappa, tokens at kappa
    int cties[kMostSlices];
    double dw[kNW];
    int iw[kNW], jw[kNW];
    double picked_sum, target, rest;
    int picked, listed, hit, last, slice;
    unsigned klo, khi;
};

// What the second kernel's parts share.
template <typename T>
struct Draw {
    const SampleParams &a;
    const Row &row;
    RowLds &L;
    const T *logits;
    float most;
    double top;
    int frac;                            // bits behind the point of sums over the row
    unsigned klo, khi;                   // the tokens in view: keys from .. to
    bool in_lds;                         // and whether they are listed

    __device__ __forceinline__ double e_of(float x) const { return exp2_f64(((double)x - (double)most) * row.c); }
    // Bins of a logit behind the row's first one.
    __device__ __forceinline__ double bin_of(float x) const { return top - floor((double)x * row.bins); }
    // The lowest finite key up to the largest logit's with in(its logit), which is false below some
    // key and true from there on, and for the largest; by one wave.
    template <typename F>
    __device__ unsigned first_key(F in) const {
        const int lane = threadIdx.x & 63;
        unsigned lo = key_of(-FLT_MAX), hi = key_of(most);
        while (lo < hi) {                        // 64 probes at once, six or seven times
            const unsigned step = (hi - lo) / 64 + 1, probe = min(lo + lane * step, hi);
            const u64 yes = __ballot(in(of_key(probe)));
            const int f = yes ? __ffsll(yes) - 1 : 64;
            if (f < 64) hi = min(lo + f * step, hi);
            if (f > 0) lo = min(lo + (f - 1) * step + 1, hi);
        }
        return lo;
    }
    // f(index, key) for the row's tokens with klo <= key <= khi, from memory
    template <typename F>
    __device__ __forceinline__ void scan(F f) const {
        const float lo = of_key(klo), hi = of_key(khi);
        for (int i = threadIdx.x * kPer; i < a.vocab; i += kSlice) {
            float x[kPer];
            load_logits(logits, i, a.vocab, x);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (x[e] >= lo && x[e] <= hi && i + e < a.vocab) f(i + e, key_of(x[e]));
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        if (in_lds)
            for (int i = threadIdx.x; i < L.listed; i += kNT) f(L.lidx[i], L.lkey[i]);
        else
            scan(f);
    }
    // Brings the tokens of bin j into view.
    __device__ void view_bin(int j) {
        __syncthreads();
        if (threadIdx.x < 64) {
            const unsigned lo = first_key([&](float x) { return bin_of(x) <= j; });
            if (threadIdx.x == 0) L.klo = lo, L.listed = 0;
        } else if (threadIdx.x < 128) {
            const unsigned above = j ? first_key([&](float x) { return bin_of(x) <= j - 1; }) : key_of(most) + 1;
            if (threadIdx.x == 64) L.khi = above - 1;
        }
        __syncthreads();
        klo = L.klo, khi = L.khi;
        scan([&](int i, unsigned k) {
            const int at = atomicAdd(&L.listed, 1);
            if (at < kList) L.lidx[at] = i, L.lkey[at] = k;
        });
        __syncthreads();
        in_lds = L.listed <= kList;
    }
    // Of the tokens in view, in falling order: the key at which `need` of them (by_sum: of their sum
    // of e) are reached, and how many of that key it takes; *sum: their sum of e up to there.
    __device__ void select(bool by_sum, double need, unsigned *kappa, int *ties, double *sum) {
        unsigned prefix = 0;
        double sums = 0.0;               // above the prefix
        int counts = 0, last_count = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            const unsigned high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            if (((klo ^ khi) >> shift) == 0) {   // one digit for all of them
                prefix = khi & (0xffffffffu << shift);
                if (shift == 0) last_count = INT_MAX;
                continue;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < kBins; i += kNT) L.hsum[i] = 0, L.hcount[i] = 0;
            __syncthreads();
            each([&](int, unsigned k) {
                if ((k & high) != (prefix & high)) return;
                atomicAdd(&L.hsum[k >> shift & 255], fixed(e_of(of_key(k)), frac));
                atomicAdd(&L.hcount[k >> shift & 255], 1u);
            });
            __syncthreads();
            if (threadIdx.x < 64) {      // four digits a lane, the largest first
                const int lane = threadIdx.x;
                const double unit = ldexp(1.0, -frac);
                double s = 0.0;
                int n = 0, last = -1;
                for (int i = 0; i < 4; ++i) {
                    const int d = 255 - (lane * 4 + i);
                    s += (double)L.hsum[d] * unit;
                    n += L.hcount[d];
                    if (L.hcount[d]) last = d;
                }
                double s0 = sums + (wave_scan_d(s) - s);
                int n0 = counts + (wave_scan_i(n) - n);
                // the lowest digit that has tokens: where rounding leaves the need unreached
                const int lowest = wave_min_i(last < 0 ? INT_MAX : last);
                if (lane == 0) L.picked = -1;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                for (int i = 0; i < 4; ++i) {
                    const int d = 255 - (lane * 4 + i), c = L.hcount[d];
                    const double ds = (double)L.hsum[d] * unit;
                    const bool there = by_sum ? c && s0 < need && (s0 + ds >= need || d == lowest)
                                              : (double)n0 < need && (double)(n0 + c) >= need;
                    const bool first = by_sum && need <= s0 && n0 == counts && c;   // nothing needed: the largest
                    if (there || first) L.picked = d, L.iw[0] = n0, L.iw[1] = c, L.picked_sum = s0;
                    s0 += ds, n0 += c;
                }
            }
            __syncthreads();
            if (L.picked < 0) break;     // nothing in view
            prefix |= (unsigned)L.picked << shift;
            sums = L.picked_sum, counts = L.iw[0], last_count = L.iw[1];
        }
        const double e = e_of(of_key(prefix));
        double n = by_sum ? ceil((need - sums) / e) : need - counts;
        n = fmin(fmax(n, 1.0), (double)last_count);
        *kappa = prefix;
        *ties = (int)n;
        *sum = sums + n * e;
    }
};
}  // namespace

// Workgroup = row.
template <typename T>
__global__ __launch_bounds__(kNT) void sample_row_kernel(SampleParams a, const SliceHead *heads, const SliceBins *bins) {
    __shared__ RowLds L;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, r = blockIdx.x, S = a.slices;
    const Row row = row_of(a, r);
    heads += (long)r * S, bins += (long)r * S;
    float most = -INFINITY;
    int at = INT_MAX, bad = 0;
    for (int s = 0; s < S; ++s) {                // the same for every thread
        const float m = heads[s].most;
        if (m > most) most = m, at = heads[s].at;
        bad |= heads[s].bad;
    }
    if (bad || row.bad || most == -INFINITY || row.greedy) {
        if (tid == 0) a.tokens[(long)r * a.token_stride] = bad || row.bad || most == -INFINITY ? -1 : at;
        return;
    }
    Draw<T> d{a, row, L, static_cast<const T *>(a.logits) + (long)r * a.stride, most, floor((double)most * row.bins),
              min(kFrac, 62 - (32 - __clz(a.vocab))), 0, 0, false};
    for (int s = tid; s < S; s += kNT) {
        const SliceHead h = heads[s];
        const double f = h.most == -INFINITY ? 0.0 : exp2_f64(((double)h.most - (double)most) * row.c);
        L.scale[s] = f;
        L.off[s] = h.most == -INFINITY ? kBins : (int)fmin(d.top - h.top, (double)kBins);
        L.kept[s] = h.total * f;                 // without cuts
        L.csum[s] = 0, L.cties[s] = 0;
    }
    __syncthreads();
    unsigned kappa = 0;
    int ties = INT_MAX;
    if (row.cuts()) {
        {   // the row's bins: four shares of the slices, then the shares in order
            const int j = tid & (kBins - 1), g = tid / kBins;
            double w = 0.0;
            int n = 0;
            for (int s = g; s < S; s += kNT / kBins) {
                const int b = j - L.off[s];
                if (b >= 0 && b < kBins - 1) w += (double)bins[s].sum[b] * L.scale[s], n += bins[s].count[b];
            }
            L.gsum[g][j] = w * ldexp(1.0, -kFrac), L.gcount[g][j] = n;
        }
        __syncthreads();
        if (wv == 0) {
            double w[4], t = 0.0;
            int n[4], m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = lane * 4 + i;
                t += w[i] = ((L.gsum[0][j] + L.gsum[1][j]) + L.gsum[2][j]) + L.gsum[3][j];
                m += n[i] = L.gcount[0][j] + L.gcount[1][j] + L.gcount[2][j] + L.gcount[3][j];
            }
            double t0 = wave_scan_d(t) - t;
            int m0 = wave_scan_i(m) - m;
#pragma unroll
            for (int i = 0; i < 4; ++i) t0 += w[i], m0 += n[i], L.wsum[lane * 4 + i] = t0, L.wcount[lane * 4 + i] = m0;
        }
        __syncthreads();
        int viewed = -1;
        double all = L.wsum[kBins - 1];
        // the first bin that reaches `need`, or kBins: none does
        auto bin_of = [&](bool by_sum, double need) {
            __syncthreads();
            if (tid == 0) L.picked = kBins;
            __syncthreads();
            if (tid < kBins && (by_sum ? L.wsum[tid] >= need : (double)L.wcount[tid] >= need) &&
                (tid == 0 ? L.wcount[0] > 0 || !by_sum : L.wcount[tid] > L.wcount[tid - 1]))
                atomicMin(&L.picked, tid);
            __syncthreads();
            return L.picked;
        };
        if (row.k_cut && L.wcount[kBins - 1] > row.k) {
            const int j = bin_of(false, row.k);
            d.view_bin(viewed = j);
            double sum;
            d.select(false, (double)row.k - (j ? L.wcount[j - 1] : 0), &kappa, &ties, &sum);
            all = (j ? L.wsum[j - 1] : 0.0) + sum;
        }
        if (row.p_cut) {
            const double need = row.p * all;
            const int j = bin_of(true, need);
            if (j < kBins) {
                if (j != viewed) d.view_bin(viewed = j);
                unsigned key;
                int n;
                double sum;
                d.select(true, need - (j ? L.wsum[j - 1] : 0.0), &key, &n, &sum);
                if (key > kappa) kappa = key, ties = n;
                else if (key == kappa) ties = min(ties, n);
            }
        }
        if (row.m_cut) {
            __syncthreads();
            if (wv == 0) {
                const unsigned key = d.first_key([&](float x) { return d.e_of(x) >= row.m; });
                if (lane == 0) L.klo = key;
            }
            __syncthreads();
            if (L.klo > kappa) kappa = L.klo, ties = INT_MAX;
        }
        // the bin of the cut; a slice keeps its bins before that, and of its tokens in that bin those above kappa
        int jc = kBins - 1;
        if (kappa) jc = (int)fmin(fmax(d.bin_of(of_key(kappa)), 0.0), kBins - 1.0);
        if (jc < kBins - 1 && jc != viewed) d.view_bin(jc);
        __syncthreads();
        if (jc < kBins - 1) {
            d.each([&](int i, unsigned k) {
                if (k > kappa) atomicAdd(&L.csum[i / kSlice], fixed(d.e_of(of_key(k)), d.frac));
                if (k == kappa) atomicAdd(&L.cties[i / kSlice], 1);
            });
            __syncthreads();
        }
        const double e = kappa ? d.e_of(of_key(kappa)) : 0.0;
        for (int s = wv; s < S; s += kNW) {
            double w = 0.0;
            for (int b = lane; b < min(jc - L.off[s], kBins - 1); b += 64) w += (double)bins[s].sum[b];
            w = wave_sum_d(w);
            int before = 0;
            for (int q = lane; q < s; q += 64) before += L.cties[q];
#pragma unroll
            for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o);
            if (lane == 0)
                L.kept[s] = w * ldexp(1.0, -kFrac) * L.scale[s] + (double)L.csum[s] * ldexp(1.0, -d.frac) +
                            (double)min(max(ties - before, 0), L.cties[s]) * e;
        }
        __syncthreads();
    }
    // the slice that the draw falls into
    if (wv == 0) {
        double mine = 0.0;
        const int per = (S + 63) / 64, s0 = min(S, lane * per), s1 = min(S, s0 + per);
        for (int s = s0; s < s1; ++s) mine += L.kept[s];
        const double incl = wave_scan_d(mine);
        const double total = __shfl(incl, 63);
        double u = (double)a.uniform[a.step ? *a.step : r];
        u = u >= 0.0 ? fmin(u, 1.0) : 0.0;       // NaN: 0
        const double t = u * total;
        double run = incl - mine;
        int pick = INT_MAX, last = -1;
        double rest = 0.0;
        for (int s = s0; s < s1; ++s) {
            // a slice that keeps any token keeps its largest
            const bool some = L.kept[s] > 0.0 && L.scale[s] >= kLeast;
            if (some) last = s;
            if (pick == INT_MAX && some && run + L.kept[s] > t) pick = s, rest = t - run;
            run += L.kept[s];
        }
        const int slice = wave_min_i(pick), end = -wave_min_i(-last);
        if (slice == INT_MAX) {                  // u = 1, or a rounding at the end: the last token
            if (lane == 0) L.slice = end, L.rest = INFINITY;
        } else if (pick == slice) {
            L.slice = slice, L.rest = rest;
        }
    }
    if (tid == 0) L.hit = INT_MAX, L.last = -1;
    __syncthreads();
    const int s = L.slice, i0 = s * kSlice + tid * kPer;
    const double rest = L.rest;
    float x[kPer];
    load_logits(d.logits, i0, a.vocab, x);
    // ties before the slice, and before the thread's tokens within it
    int mine = 0, before = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += kappa && i0 + e < a.vocab && key_of(x[e]) == kappa;
    for (int q = lane; q < s; q += 64) before += L.cties[q];
#pragma unroll
    for (int o = 32; o; o >>= 1) before += __shfl_xor(before, o);
    const int incl = wave_scan_i(mine);
    if (lane == 63) L.iw[wv] = incl;
    __syncthreads();
    before += incl - mine;
    for (int w = 0; w < wv; ++w) before += L.iw[w];
    double e[kPer], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        bool keep = x[i] > -INFINITY;            // also false past the end
        if (kappa && keep) {
            const unsigned k = key_of(x[i]);
            keep = k > kappa || (k == kappa && before++ < ties);
        }
        e[i] = keep ? d.e_of(x[i]) : 0.0;
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
    if (tid == 0) a.tokens[(long)r * a.token_stride] = L.hit == INT_MAX ? L.last : L.hit;
}

namespace {
template <typename T>
void sample(const SampleParams &a, SliceHead *heads, SliceBins *bins, hipStream_t st) {
    OJX_LAUNCH((sample_slice_kernel<T>), dim3((unsigned)a.rows * a.slices), dim3(kNT), 0, st, a, heads, bins);
    OJX_LAUNCH((sample_row_kernel<T>), dim3(a.rows), dim3(kNT), 0, st, a, heads, bins);
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
    return rows * slices * (long)(sizeof(SliceHead) + sizeof(SliceBins));
}

int launch_sample(SampleParams a, int dtype, void *workspace, hipStream_t st) {
    a.slices = (a.vocab + kSlice - 1) / kSlice;
    SliceBins *bins = static_cast<SliceBins *>(workspace);
    SliceHead *heads = reinterpret_cast<SliceHead *>(bins + (long)a.rows * a.slices);
    if (dtype == OJASX_DTYPE_F32) sample<float>(a, heads, bins, st);
    else if (dtype == OJASX_DTYPE_BF16) sample<__hip_bfloat16>(a, heads, bins, st);
    else sample<__half>(a, heads, bins, st);
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
    a.uniform = uniform, a.tokens = tokens, a.token_stride = 1;
    a.temperature = s.temperature, a.temperatures = s.temperatures;
    a.top_k = s.top_k, a.top_ks = s.top_ks;
    a.top_p = s.top_p, a.top_ps = s.top_ps;
    a.min_p = s.min_p, a.min_ps = s.min_ps;
    return launch_sample(a, dtype, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
