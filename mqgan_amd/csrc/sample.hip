// Drawing a code per row of scores: temperature, top-k, top-p, min-p, from given uniform numbers.
//
//   order the codes by (score descending, index ascending); w = exp((z - max) / T)
//   top-k: the first k;  top-p: of those, every code before which less than top_p of their mass lies (the first always);
//   min-p: of those, w >= min_p (of the largest's weight 1)
//   drawn: the first code in INDEX order with (mass of the kept codes up to and with it) > u * (mass of all kept codes)
// T <= 0: the largest score, lowest index.  -inf and NaN are never drawn; a row of nothing else gives -1; where +inf occurs, the
// +inf codes share the draw evenly.
//
// Masses are whole numbers: w rounded to units of 2^-min(51, 62 - ceil(log2 V)), exp in f64.  Their sums are exact whatever the order of
// the additions, so histograms by atomics, scans and tree sums all agree to the last bit, and a cut or a draw next to a border falls the
// same way on every run.  With f32 masses a row of 8192 codes would be drawn next to a border about once in 1000 rows.  A weight under
// the unit counts as one unit (2^-49 at V = 8192) unless exp gives 0.
//
// Both cuts are a place in the order, (score, index): everything at or before it stays.  A block has one row; where it fits (48 KiB) the row is
// read once, into LDS.  A cut is found without sorting: a histogram over the distance from the maximum (bins of equal RATIO, so neither the
// scores' scale nor masks of the type's lowest value matter) tells the bin that the cut falls into, a second one over that bin's lower bits
// narrows it, and the few codes left are put into a list and counted against each other.  Where that list overflows (hundreds of equal scores
// across the cut) radix selection over the bits of the score finds the cut instead.  Once a cut leaves few codes they are put
// into a list in index order that takes the row's place: after a top-k the f64 exponentials are those of the codes it keeps.
// A wave covers a contiguous part of the row, so that sums up to a code need one number per wave.
#include "common.h"

namespace mq {

struct SampleArgs {
    const void *z;
    int64_t ld;
    int V, shift;                        // weights are w 2^shift
    const float *u;
    const float *temperature, *top_p, *min_p;        // per row, or NULL
    const int32_t *top_k;
    double t0, p0, m0;
    int k0;
    const uint8_t *padded;
    int64_t *idx;
    float *logp;
};
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }      // NaN is never drawn; -0 and +0 are one score
template <int DT> struct Score;                                      // 0 f32, 1 bf16, 2 f16, as they lie in memory
template <> struct Score<0> {
    typedef float Raw;
    typedef f32x4u Raw4;
    static __device__ __forceinline__ float widen(Raw v) { return v; }
    static __device__ __forceinline__ Raw narrow(float v) { return v; }
};
template <> struct Score<1> {
    typedef uint16_t Raw;
    typedef u16x4u Raw4;
    static __device__ __forceinline__ float widen(Raw v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ Raw narrow(float v) { return (Raw)(__float_as_uint(v) >> 16); }      // of a value that is one
};
template <> struct Score<2> {
    typedef uint16_t Raw;
    typedef u16x4u Raw4;
    static __device__ __forceinline__ float widen(Raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ Raw narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// The scores of a row, from LDS (cleaned, padded to a multiple of 4 with -inf) or from memory.
template <int DT, bool STAGED>
struct View {
    typedef Score<DT> S;
    const typename S::Raw *p;
    int n;                               // codes
    bool inf;                            // from memory: the row has +inf scores, which become 0, the others -inf
    __device__ __forceinline__ float one(int c) const
    {
        if (STAGED) return S::widen(p[c]);
        const float v = clean(S::widen(p[c]));
        return inf ? (v == INFINITY ? 0.f : -INFINITY) : v;
    }
    __device__ __forceinline__ void four(int c, float (&x)[4]) const      // c is a multiple of 4 below n
    {
        if (STAGED || c + 4 <= n) {
            const typename S::Raw4 q = *reinterpret_cast<const typename S::Raw4 *>(p + c);
            const typename S::Raw v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = S::widen(v[i]);
                if (!STAGED) {
                    x[i] = clean(x[i]);
                    if (inf) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = c + i < n ? one(c + i) : -INFINITY;
        }
    }
};

// exp(d), -746 <= d <= 0, in f64: d = n ln 2 + r, |r| <= 0.35, Taylor's series of exp(r) to r^11 (the rest is under 1e-14).
constexpr double LN2_HI = 2977044472.0 / 4294967296.0, LN2_LO = -4.2009150726810846e-11;    // ln 2 2^32 to the nearest whole number, and the rest
__device__ __forceinline__ double exp_neg(double d)
{
    const double n = rint(d * 1.4426950408889634074);
    double r = fma(n, -LN2_HI, d);                                  // exact: LN2_HI has 32 bits, n 11
    r = fma(n, -LN2_LO, r);
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// What of a row's settings the weights need; max is finite (rows with +inf are remapped to scores 0 and -inf before)
struct Row {
    double max, per_t;                   // 1 / T; 0 for T = inf
    double scale;                        // 2^shift
    double min_p;                        // <= 1
    // Units of a code with a score above -inf: w 2^shift to the nearest whole number, at least 1 - the bits of w 2^shift + 2^52 (shift <= 51,
    // w <= 1); 0 where w would underflow and, with FILTER, where it is under min_p.
    template <bool FILTER>
    __device__ __forceinline__ uint64_t units(float x) const
    {
        const double d = ((double)x - max) * per_t, w = exp_neg(fmax(d, -746.0));
        const uint64_t q = (uint64_t)__double_as_longlong(fma(w, scale, 4503599627370496.0)) & 0xfffffffffffffull;
        return d < -745.0 || (FILTER && w < min_p) ? 0 : q > 1 ? q : 1;
    }
    // log of a weight's share of Z units
    __device__ __forceinline__ float logp(float x, uint64_t Z) const { return (float)(((double)x - max) * per_t - log((double)Z / scale)); }
};

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
    return v;
}
template <typename U>
__device__ __forceinline__ U wave_scan(U v)                          // inclusive
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const U t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}
// over a block of W waves; red: W entries of its own, free again when the call returns
template <int W>
__device__ __forceinline__ uint64_t block_sum_u64(uint64_t v, unsigned long long *red)
{
    v = wave_sum_u64(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) t += red[i];
    __syncthreads();
    return t;
}
template <int W>
__device__ __forceinline__ float block_max_f32(float v, float *red)
{
    v = wave_max(v);
    if (W == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
#pragma unroll
    for (int i = 1; i < W; ++i) t = fmaxf(t, red[i]);
    __syncthreads();
    return t;
}

// The first bin up to and with which at least `goal` lies, and what lies before it; by the first wave, in LDS for the block.  FROM_TOP: the
// bins are ordered by the score instead of by the distance from the maximum, so they are walked from the last.
struct Found {
    unsigned long long before, total;
    int bin;
};
template <int BINS, bool FROM_TOP, typename U>
__device__ __forceinline__ void find_bin(const U *hist, uint64_t goal, Found *out)
{
    if (threadIdx.x < 64) {
        constexpr int PER = BINS / 64;
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += hist[FROM_TOP ? BINS - 1 - ((int)threadIdx.x * PER + i) : (int)threadIdx.x * PER + i];
        const uint64_t upto = wave_scan<unsigned long long>(mine);
        if (threadIdx.x == 63) out->total = upto;
        if (upto >= goal && upto - mine < goal) {
            uint64_t before = upto - mine;
            int i = 0;
            for (; i < PER - 1; ++i) {
                const uint64_t h = hist[FROM_TOP ? BINS - 1 - ((int)threadIdx.x * PER + i) : (int)threadIdx.x * PER + i];
                if (before + h >= goal) break;
                before += h;
            }
            out->before = before;
            out->bin = FROM_TOP ? BINS - 1 - ((int)threadIdx.x * PER + i) : (int)threadIdx.x * PER + i;
        }
    }
    __syncthreads();
}

// order-preserving key of a score
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

// ----------------------------------------------------------------------------- bins
// Bins of a distance from the maximum: 2^(23 - SH) to an octave over 32 octaves from 2^-12 up, what lies outside in the first and the last.
// An inner bin holds distances that differ in their lower SH bits only; its own bins are the highest of those.
template <int BINS>
struct Bins {
    static constexpr int LOG = BINS == 512 ? 9 : 8, SH = 28 - LOG;
    static __device__ __forceinline__ int of(float d)
    {
        const int b = (int)(__float_as_uint(d) >> SH) - ((127 - 12) << (23 - SH));
        return min(max(b, 0), BINS - 1);
    }
    static __device__ __forceinline__ int inner(float d) { return (int)(__float_as_uint(d) >> (SH - LOG)) & (BINS - 1); }
};

// (x, i) stands before (y, j) in the order
__device__ __forceinline__ bool ahead_of(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

struct Entry {
    float x;
    int i;
    unsigned long long w;
};
template <int DT, int W>
struct Lds {
    static constexpr int BINS = W <= 2 ? 256 : 512, LIST = BINS / 2, KEPT = BINS;
    unsigned long long hist[BINS];
    Entry list[LIST];                                               // codes of the bin that a cut falls into
    alignas(16) typename Score<DT>::Raw kept_x[KEPT];               // the kept codes in index order, once they are few
    int kept_i[KEPT];
    unsigned long long red[W];
    float redf[W], cut_x;
    int redi[W], cut_i, length;
    Found found;
};

template <int DT, bool STAGED, int W>
struct Draw {
    static constexpr int NT = 64 * W, FEW = 40;
    typedef Lds<DT, W> L;
    typedef Bins<L::BINS> B;
    L &s;
    View<DT, STAGED> row;
    float cut_x;                                                    // kept: at or before (cut_x, cut_i) in the order
    int cut_i;

    __device__ __forceinline__ Draw(L &s_) : s(s_) {}
    // The wave's part of the row: codes [from, to), a multiple of 256 from the last one's
    __device__ __forceinline__ int from(int wave) const { return wave * part(); }
    __device__ __forceinline__ int part() const { return (row.n + 256 * W - 1) / (256 * W) * 256; }
    __device__ __forceinline__ bool kept(float x, int c) const { return x > cut_x || (x == cut_x && c <= cut_i); }
    // f(x, c) for the kept codes of the block
    template <typename F>
    __device__ __forceinline__ void each(F f) const
    {
        const int c0 = from(threadIdx.x >> 6), c1 = min(c0 + part(), row.n);
#pragma unroll 1
        for (int c = c0 + (threadIdx.x & 63) * 4; c < c1; c += 256) {
            float x[4];
            row.four(c, x);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (kept(x[i], c + i)) f(x[i], c + i);
        }
    }
    // Sum of q(x) over the kept codes of the lane, four at a time without branches between them
    template <typename Q>
    __device__ __forceinline__ uint64_t sum(Q q) const
    {
        uint64_t t = 0;
        const int c0 = from(threadIdx.x >> 6), c1 = min(c0 + part(), row.n);
#pragma unroll 1
        for (int c = c0 + (threadIdx.x & 63) * 4; c < c1; c += 256) {
            float x[4];
            row.four(c, x);
            bool in[4], any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= in[i] = kept(x[i], c + i);
            if (!any) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t u = q(in[i] ? x[i] : (float)-INFINITY);
                t += in[i] ? u : 0;
            }
        }
        return t;
    }
    // The same cut by radix selection over the bits of the score, for borders that hundreds of equal or nearly equal scores lie at.
    template <typename Q>
    __device__ __forceinline__ void find_cut_by_bits(uint64_t goal, Q q)
    {
        uint32_t prefix = 0;
        uint64_t above = 0;
#pragma unroll 1
        for (int sh = 24; sh >= 0; sh -= 8) {
            __syncthreads();
            for (int b = threadIdx.x; b < 256; b += NT) s.hist[b] = 0;
            __syncthreads();
            each([&](float v, int) {
                const uint32_t key = key_of(v);
                if (sh == 24 || key >> (sh + 8) == prefix) atomicAdd(&s.hist[(key >> sh) & 255u], (unsigned long long)q(v));
            });
            __syncthreads();
            find_bin<256, true>(s.hist, goal - above, &s.found);
            prefix = prefix << 8 | (uint32_t)s.found.bin;
            above += s.found.before;
        }
        // codes with the border's score are kept while above + j w < goal: the last of them by its index
        const float border = score_of(prefix);
        const uint64_t w = q(border);
        const int need = (int)((goal - above + w - 1) / w);
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int c0 = from(wave), c1 = min(c0 + part(), row.n);
        int count = 0;
        each([&](float v, int) { count += v == border; });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o, 64);
        if (lane == 0) s.redi[wave] = count;
        __syncthreads();
        int before = 0;
        for (int v = 0; v < wave; ++v) before += s.redi[v];
        if (before < need && before + count >= need) {
#pragma unroll 1
            for (int c = c0; c < c1; c += 256) {                    // the wave's lanes go round together
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                const int at = c + lane * 4;
                if (at < c1) row.four(at, x);
                int mine = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) mine += x[i] == border && kept(x[i], at + i);
                int upto = wave_scan(mine) + before;
                before = __shfl(upto, 63, 64);
                upto -= mine;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (x[i] == border && kept(x[i], at + i) && ++upto == need) s.cut_i = at + i;
            }
        }
        __syncthreads();
        cut_x = border;
        cut_i = s.cut_i;
    }
    // Moves the cut to the code with which the mass of the kept codes, in their order, reaches `goal` (leaves it if it does not).  q(x): a code's
    // mass.  limit: a bin that the cut is believed not to lie behind; codes behind it take no part (they do if the belief was wrong).
    template <typename Q>
    __device__ __forceinline__ void find_cut(float mx, uint64_t goal, int limit, Q q)
    {
        const int tid = threadIdx.x;
        int bin = 0, sub = -1;
        uint64_t above = 0;
#pragma unroll 1
        for (int level = 0; level < 2; ++level) {
            __syncthreads();
#pragma unroll 1
            for (int b = tid; b < L::BINS; b += NT) s.hist[b] = 0;
            if (tid == 0) s.length = 0;
            __syncthreads();
            each([&](float v, int) {
                const float d = mx - v;
                const int b = B::of(d);
                if (level == 0 ? b <= limit : b == bin) atomicAdd(&s.hist[level == 0 ? b : B::inner(d)], (unsigned long long)q(v));
            });
            __syncthreads();
            find_bin<L::BINS, false>(s.hist, goal - above, &s.found);
            if (level == 0) {
                if (s.found.total < goal) {
                    if (limit == L::BINS - 1) return;
                    limit = L::BINS - 1;
                    level = -1;
                    continue;
                }
                bin = s.found.bin;
            } else {
                sub = s.found.bin;
            }
            above += s.found.before;
            each([&](float v, int c) {
                const float d = mx - v;
                if (B::of(d) != bin || (sub >= 0 && B::inner(d) != sub)) return;
                const int e = atomicAdd(&s.length, 1);
                if (e < L::LIST) s.list[e] = Entry{v, c, (unsigned long long)q(v)};
            });
            __syncthreads();
            if (s.length <= FEW || bin == 0 || bin == L::BINS - 1) break;
        }
        const int many = s.length;
        if (many > L::LIST) {
            find_cut_by_bits(goal, q);
            return;
        }
#pragma unroll 1
        for (int e = tid; e < many; e += NT) {
            const Entry me = s.list[e];
            uint64_t before = above;
#pragma unroll 4
            for (int o = 0; o < many; ++o) {
                const Entry t = s.list[o];
                before += ahead_of(t.x, t.i, me.x, me.i) ? t.w : 0;
            }
            if (before < goal && before + me.w >= goal) {
                s.cut_x = me.x;
                s.cut_i = me.i;
            }
        }
        __syncthreads();
        cut_x = s.cut_x;
        cut_i = s.cut_i;
    }
    // A bin that at least `goal` codes lie up to: the one that `goal` of the threads' own maxima do.  One number a thread instead of its codes.
    __device__ __forceinline__ int limit_of(float mx, float own, int goal)
    {
        if (goal > NT) return L::BINS - 1;
        for (int b = threadIdx.x; b < L::BINS; b += NT) s.hist[b] = 0;
        __syncthreads();
        if (own > -INFINITY) atomicAdd(&s.hist[B::of(mx - own)], 1ull);
        __syncthreads();
        find_bin<L::BINS, false>(s.hist, (uint64_t)goal, &s.found);
        return s.found.total < (uint64_t)goal ? L::BINS - 1 : s.found.bin;
    }
    // Where at most KEPT codes are kept: they take the row's place (a row in LDS only), in index order.  Whether they did.
    __device__ __forceinline__ bool compact()
    {
        if (!STAGED) return false;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const uint64_t below = (1ull << lane) - 1;
        const int c0 = from(wave), c1 = min(c0 + part(), row.n);
        int count = 0;
#pragma unroll 1
        for (int c = c0; c < c1; c += 256) {                        // all lanes of a wave go round together
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (c + lane * 4 < c1) row.four(c + lane * 4, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) count += __popcll(__builtin_amdgcn_ballot_w64(kept(x[i], c + lane * 4 + i)));
        }
        if (lane == 0) s.redi[wave] = count;
        __syncthreads();
        int at = 0, many = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            at += w < wave ? s.redi[w] : 0;
            many += s.redi[w];
        }
        __syncthreads();
        if (many > L::KEPT) return false;
#pragma unroll 1
        for (int c = c0; c < c1; c += 256) {
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (c + lane * 4 < c1) row.four(c + lane * 4, x);
            int place = at;
            bool in[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                in[i] = kept(x[i], c + lane * 4 + i);
                const uint64_t m = __builtin_amdgcn_ballot_w64(in[i]);
                place += __popcll(m & below);
                at += __popcll(m);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (in[i]) {
                    s.kept_x[place] = Score<DT>::narrow(x[i]);
                    s.kept_i[place++] = c + lane * 4 + i;
                }
        }
        if (threadIdx.x < (unsigned)(-many & 3)) s.kept_x[many + threadIdx.x] = Score<DT>::narrow(-INFINITY);      // to whole quads
        __syncthreads();
        row.p = s.kept_x;
        row.n = many;
        cut_x = -INFINITY;
        cut_i = -1;
        return true;
    }
};

template <int DT, bool STAGED, int W>
__global__ __launch_bounds__(64 * W, 6) void sample_kernel(const SampleArgs a)
{
    typedef Score<DT> S;
    constexpr int NT = 64 * W;
    extern __shared__ __attribute__((aligned(16))) char staged[];
    __shared__ Lds<DT, W> s;
    const int64_t n = blockIdx.x;
    const int V = a.V, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const auto answer = [&](int64_t i, float lp) {
        a.idx[n] = i;
        if (a.logp) a.logp[n] = lp;
    };
    if (a.padded && a.padded[n]) {
        if (tid == 0) answer(-1, 0.f);
        return;
    }
    const typename S::Raw *z = reinterpret_cast<const typename S::Raw *>(a.z) + n * a.ld;
    typename S::Raw *lds = reinterpret_cast<typename S::Raw *>(staged);
    Draw<DT, STAGED, W> d(s);
    d.row = {z, V, false};
    d.cut_x = -INFINITY;
    d.cut_i = -1;                                                   // nothing with a score of -inf
    float mx = -INFINITY;
    if (STAGED) {
        const View<DT, false> from{z, V, false};
#pragma unroll 4
        for (int c = tid * 4; c < V; c += NT * 4) {
            float x[4];
            from.four(c, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mx = fmaxf(mx, x[i]);
                lds[c + i] = S::narrow(x[i]);
            }
        }
        d.row.p = lds;
    } else {
        d.each([&](float v, int) { mx = fmaxf(mx, v); });
    }
    const double T = a.temperature ? (double)a.temperature[n] : a.t0, P = a.top_p ? (double)a.top_p[n] : a.p0;
    const double mp = a.min_p ? (double)a.min_p[n] : a.m0;
    const int k = a.top_k ? a.top_k[n] : a.k0;
    const float u = a.u[n];
    float own = mx;
    mx = block_max_f32<W>(mx, s.redf);
    if (mx == -INFINITY) {
        if (tid == 0) answer(-1, 0.f);
        return;
    }
    if (mx == INFINITY) {
        mx = 0.f;
        own = own == INFINITY ? 0.f : -INFINITY;
        if (STAGED) {
            for (int c = tid; c < (V + 3) / 4 * 4; c += NT) lds[c] = S::narrow(S::widen(lds[c]) == INFINITY ? 0.f : -INFINITY);
        } else {
            d.row.inf = true;
        }
    }
    __syncthreads();
    if (!(T > 0.0)) {                                               // the lowest index that has the maximum
        int first = INT32_MAX;
        d.each([&](float v, int c) { first = v == mx && c < first ? c : first; });
        const float lowest = block_max_f32<W>(-(float)first, s.redf);  // indices are below 2^24
        if (tid == 0) answer((int64_t)-lowest, 0.f);
        return;
    }
    const Row r{(double)mx, fmin(1.0 / T, 1e300), ldexp(1.0, a.shift), mp > 1.0 ? 1.0 : mp};
    const auto units = [&](float v) { return r.template units<false>(v); };
    bool listed = false;
    if (k > 0 && k < V) {
        d.find_cut(mx, (uint64_t)k, d.limit_of(mx, own, k), [](float) { return (uint64_t)1; });
        if (k <= Lds<DT, W>::KEPT) listed = d.compact();
    }
    if (P < 1.0) {
        const double Z = (double)block_sum_u64<W>(d.sum(units), s.red), g = ceil(P * Z);
        // codes further than D from the maximum have at most n exp(-D / T) = (1 - P) Z together
        const float D = (float)(T * 1.0001 * log((double)d.row.n * r.scale / ((1.0 - P) * Z)));
        d.find_cut(mx, g > 1.0 ? (uint64_t)g : 1, D > 0.f ? Bins<Lds<DT, W>::BINS>::of(D) : 0, units);      // kept while less than that lies before them
        if (!listed) listed = d.compact();
    }
    // the draw: the waves' sums, then the wave that it falls to goes over its part again
    // (NaN min_p: nothing is under it)
    const auto drawn = [&](float v) { return r.min_p > 0.0 ? r.template units<true>(v) : r.template units<false>(v); };
    uint64_t part = d.sum(drawn);
    part = wave_sum_u64(part);
    if (lane == 0) s.red[wave] = part;
    __syncthreads();
    uint64_t Z = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) Z += s.red[w];
    const double t = floor((double)(u > 0.f ? u : 0.f) * (double)Z);
    uint64_t target = t < (double)Z ? (uint64_t)t : Z - 1;
    if (target >= Z) target = Z - 1;
    uint64_t before = 0;
    int mine = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const uint64_t here = s.red[w];
        if (before + here <= target) {
            before += here;
            mine = w + 1;
        } else {
            break;
        }
    }
    if (wave != mine) return;
    const int c0 = d.from(wave), c1 = min(c0 + d.part(), d.row.n);
#pragma unroll 1
    for (int c = c0; c < c1; c += 256) {                            // the wave's lanes go round together
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const int at = c + lane * 4;
        if (at < c1) d.row.four(at, x);
        uint64_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = d.kept(x[i], at + i) ? drawn(x[i]) : 0;
        const uint64_t sum = (q[0] + q[1]) + (q[2] + q[3]), upto = wave_scan<unsigned long long>(sum) + before;
        if (upto > target && upto - sum <= target) {
            uint64_t b = upto - sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (b <= target && b + q[i] > target) answer(listed ? s.kept_i[at + i] : at + i, a.logp ? r.logp(x[i], Z) : 0.f);
                b += q[i];
            }
        }
        before = __shfl((unsigned long long)upto, 63, 64);
        if (before > target) return;
    }
}

}  // namespace mq

using namespace mq;

// Waves a row: with many rows as few as keep a compute unit's 32 waves busy next to the rows' LDS, with too few rows to fill the chip as many
// as the row has quads for, up to 16.
template <int DT>
static void sample_launch(const SampleArgs &a, int64_t rows, hipStream_t s)
{
    const dim3 grid((unsigned)rows);
    const size_t bytes = ((size_t)a.V + 3) / 4 * 4 * sizeof(typename Score<DT>::Raw);
#define GO(W) hipLaunchKernelGGL((sample_kernel<DT, true, W>), grid, dim3(64 * W), bytes, s, a)
    if (bytes > 48 * 1024) hipLaunchKernelGGL((sample_kernel<DT, false, 8>), grid, dim3(512), 0, s, a);
    else if (rows < 256) {
        if (a.V <= 1024) GO(4);
        else if (a.V <= 2048) GO(8);
        else GO(16);
    } else if (a.V <= 1024) GO(2);
    else if (a.V <= 4096) GO(4);
    else GO(8);
#undef GO
}

extern "C" int mq_sample_codes(const mqSampleDesc *d, const void *logits, const float *uniform, const float *temperature, const int32_t *top_k,
                               const float *top_p, const float *min_p, const uint8_t *padded, int64_t *idx, float *logp, mqStream stream)
{
    MQ_REQUIRE(d && logits && uniform && idx, "mq_sample_codes: NULL argument");
    MQ_REQUIRE(d->dtype >= 0 && d->dtype <= 2, "mq_sample_codes: dtype %d (0 f32, 1 bf16, 2 f16)", d->dtype);
    MQ_REQUIRE(d->rows > 0 && d->rows < INT32_MAX && d->codes > 0 && d->codes <= (1 << 20) && d->row_stride >= d->codes,
               "mq_sample_codes: bad sizes (rows %lld, codes %d of at most 2^20, row stride %lld)", (long long)d->rows, d->codes, (long long)d->row_stride);
    MQ_REQUIRE(temperature || d->temperature >= 0.0, "mq_sample_codes: temperature %g", d->temperature);
    MQ_REQUIRE(top_k || d->top_k >= 0, "mq_sample_codes: top_k %d", d->top_k);
    MQ_REQUIRE(top_p || (d->top_p >= 0.0 && d->top_p <= 1.0), "mq_sample_codes: top_p %g is not in [0, 1]", d->top_p);
    MQ_REQUIRE(min_p || (d->min_p >= 0.0 && d->min_p <= 1.0), "mq_sample_codes: min_p %g is not in [0, 1]", d->min_p);
    int bits = 0;
    while ((1ll << bits) < d->codes) ++bits;
    const int shift = 62 - bits < 51 ? 62 - bits : 51;
    const SampleArgs a{logits, d->row_stride, d->codes, shift, uniform, temperature, top_p, min_p, top_k, d->temperature, d->top_p, d->min_p, d->top_k, padded, idx, logp};
    if (d->dtype == 0) sample_launch<0>(a, d->rows, S(stream));
    else if (d->dtype == 1) sample_launch<1>(a, d->rows, S(stream));
    else sample_launch<2>(a, d->rows, S(stream));
    MQ_LAUNCH_CHECK("mq_sample_codes");
    return 0;
}
