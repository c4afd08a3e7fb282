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
// the unit counts as one unit (2^-49 at V = 8192) unless exp gives 0.  All roundings of a row together stay under V units of the largest weight: 2^-36
// at 8192 codes, 2^-24 at 2^19, which is one step of the uniform numbers next to 1.  Past that whole units of codes that weigh nothing would be
// drawn (at 2^20 by the three largest numbers under 1), so 2^19 codes is what a row may have.
//
// Both cuts are a place in the order, (score, index): everything at or before it stays.  A block has one row, which is read once, into LDS, where
// it fits (up to 9896 f32 or 14848 two-byte scores; past that each pass reads memory); each wave has a contiguous part, reads back what it wrote itself and needs no barrier
// for that, and sums up to a code need one number per wave.  The codes that can be before a cut are found by a bound first - k of the threads'
// own maxima are at least so large; codes beyond some distance hold less mass than top_p leaves out - and packed, in index order.
// A cut is found without sorting: a histogram over the distance from the maximum (bins of equal RATIO, so neither the scores' scale nor masks of
// the type's lowest value matter) tells the bin that it falls into, a second one over that bin's lower bits narrows it, and the few codes left
// are put into a list and counted against each other.  Where that list overflows (dozens of equal scores across the cut) radix selection over
// the bits of the score finds the cut instead.
//
// What bounds it: 16384 x 8192 f32 read once are 76 us at the 7.1 TB/s that loads alone reach here.  The maximum alone (temperature 0) takes 105
// us, top-k 20 145, top-k 100 with top-p 0.95 195-205: the vector units are busy 74 % of the latter (35 instructions a code), the rest is waits of the
// lists' waves.  Without top-k the masses of all codes are needed, 15 sums, products and FMAs in f64 each beside scaling, rounding, conversion and
// comparison: 16384 x 8192 without a filter 263-280 us (52 instructions a code, busy 76 %), top-p 0.95 530-590 (132, busy 90 %); 16384 x 1024 with
// top-p 0.9 57-61 (floor 9.5; 99 a code, busy 85 %), of which reading and the first masses are 32, the cut 20 and the draw 7.  Small calls are latency,
// a chain of some thirty dependent LDS accesses and barriers: one row of 1000 codes with all filters 10 us, 48 of 8003 with top-p 0.95 25, 64 of 32000
// with top-k 100 and top-p 0.9 27.  Selection by the bits of the scores over a row in memory took 2688 us where the lists take 200; a row in
// registers needs 215 of them.
#include <algorithm>

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
    int64_t row0, rows;                                              // those of a launch: [row0, rows)
    int squeezes;                                                    // there is a cut: the rows' LDS has room for V indices
    __device__ __forceinline__ double T(int64_t n) const { return temperature ? (double)temperature[n] : t0; }
    __device__ __forceinline__ double P(int64_t n) const { return top_p ? (double)top_p[n] : p0; }
    __device__ __forceinline__ double min(int64_t n) const { return min_p ? (double)min_p[n] : m0; }
    __device__ __forceinline__ int k(int64_t n) const
    {
        const int v = top_k ? top_k[n] : k0;
        return v < V ? v : 0;                                        // 0 and below: all
    }
};
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4a __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4a __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY); }      // NaN is never drawn
template <int DT> struct Score;                                      // 0 f32, 1 bf16, 2 f16, as they lie in memory
template <> struct Score<0> {
    typedef float Raw;
    typedef f32x4u Raw4;
    typedef f32x4a Quad;                                             // in LDS
    static __device__ __forceinline__ float widen(Raw v) { return v; }
    static __device__ __forceinline__ Raw narrow(float v) { return v; }
};
template <> struct Score<1> {
    typedef uint16_t Raw;
    typedef u16x4u Raw4;
    typedef u16x4a Quad;
    static __device__ __forceinline__ float widen(Raw v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ Raw narrow(float v) { return (Raw)(__float_as_uint(v) >> 16); }      // of a value that is one
};
template <> struct Score<2> {
    typedef uint16_t Raw;
    typedef u16x4u Raw4;
    typedef u16x4a Quad;
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
        if (STAGED) {
            const typename S::Quad q = *reinterpret_cast<const typename S::Quad *>(p + c);
            const typename S::Raw v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = S::widen(v[i]);
        } else if (c + 4 <= n) {
            const typename S::Raw4 q = *reinterpret_cast<const typename S::Raw4 *>(p + c);
            const typename S::Raw v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = clean(S::widen(v[i]));
                if (inf) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = c + i < n ? one(c + i) : -INFINITY;
        }
    }
};

// 2^r, |r| <= 1/2, in f64: 1 + r q(r), q by interpolation at Chebyshev's points; relative error under 4e-14, 1 at 0.  (Taylor's series needs two
// more terms, and the masses are what limits the filters of a whole row: about 25 operations in f64 a code, at the rate of f32.)
__device__ __forceinline__ double exp2_half(double r)
{
    double q = 1.0203121063391729e-07;
    q = fma(q, r, 1.3255224878668817e-06);
    q = fma(q, r, 1.525268684626772e-05);
    q = fma(q, r, 1.5403455852453838e-04);
    q = fma(q, r, 1.3333558179043112e-03);
    q = fma(q, r, 9.618129159402558e-03);
    q = fma(q, r, 5.5504108664760424e-02);
    q = fma(q, r, 2.402265069581299e-01);
    q = fma(q, r, 6.931471805599453e-01);
    return fma(q, r, 1.0);
}
// ln x, 1 <= x < 2^64, to 1e-13: the f32 instruction's log2, corrected by how far 2 to its power is from x
__device__ __forceinline__ double ln(double x)
{
    const double y = (double)__builtin_amdgcn_logf((float)x), n = rint(y);
    const double off = ldexp(x * exp2_half(n - y), -(int)n) - 1.0;  // about 1e-6 at most
    return fma(y, 0.6931471805599453, off * fma(off, -0.5, 1.0));
}
// What of a row's settings the weights need; max is finite (rows with +inf are remapped to scores 0 and -inf before)
struct Row {
    double max, per_t;                   // 1 / T; 0 for T = inf
    double per2;                         // log2(e) / T
    int shift;                           // weights are w 2^shift
    double tiny, least;                  // 2^shift times the smallest weight above 0, and times min_p where that is more (min_p <= 1)
    __device__ __forceinline__ Row(float max_, double T, double min_p, int shift_)
        : max((double)max_), per_t(fmin(1.0 / T, 1e300)), per2(per_t * 1.4426950408889634074), shift(shift_), tiny(ldexp(1.15, shift_ - 1075)),
          least(fmax(ldexp(min_p > 1.0 ? 1.0 : min_p, shift_), tiny))
    {
    }
    // Units of a code: w 2^shift to the nearest whole number, at least 1 - the bits of w 2^shift + 2^52 (shift <= 51, w <= 1); 0 where w would
    // underflow in f64 (where d is past f64, as for a score of -inf, w is a NaN) and where w 2^shift is under `limit`.
    __device__ __forceinline__ uint64_t units(float x, double limit) const
    {
        const double d = ((double)x - max) * per2, n = rint(d);
        const double w = ldexp(exp2_half(d - n), (int)n + shift);
        const uint64_t q = (uint64_t)__double_as_longlong(fmax(w, 1.0) + 4503599627370496.0) & 0xfffffffffffffull;
        return w >= limit ? q : 0;
    }
    __device__ __forceinline__ uint64_t units(float x) const { return units(x, tiny); }
    // log of a weight's share of Z units
    __device__ __forceinline__ float logp(float x, uint64_t Z) const { return (float)(((double)x - max) * per_t - ln(ldexp((double)Z, -shift))); }
};

// Inclusive scans over the 64 lanes by DPP (row shifts, then the rows' last lanes broadcast): a tenth of the latency of the LDS crossbar's.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t v)             // 0 where there is no lane to read
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_from(uint64_t v)
{
    return (uint64_t)dpp_from<CTRL, ROWS>((uint32_t)v) | (uint64_t)dpp_from<CTRL, ROWS>((uint32_t)(v >> 32)) << 32;
}
template <typename U>
__device__ __forceinline__ U wave_scan(U v)
{
    v += dpp_from<0x111, 0xf>(v);                                    // row_shr 1, 2, 4, 8
    v += dpp_from<0x112, 0xf>(v);
    v += dpp_from<0x114, 0xf>(v);
    v += dpp_from<0x118, 0xf>(v);
    v += dpp_from<0x142, 0xa>(v);                                    // row_bcast 15 into rows 1 and 3
    v += dpp_from<0x143, 0xc>(v);                                    // row_bcast 31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ uint32_t from_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }      // lane: the same in all
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane)
{
    return (uint64_t)from_lane((uint32_t)v, lane) | (uint64_t)from_lane((uint32_t)(v >> 32), lane) << 32;
}
template <typename U>
__device__ __forceinline__ U wave_total(U v) { return from_lane(wave_scan(v), 63); }
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
template <int W> __device__ __forceinline__ void together();
template <int BINS, bool FROM_TOP, int W, typename U>
__device__ __forceinline__ void find_bin(const U *hist, uint64_t goal, Found *out)
{
    const int lane = W > 1 ? (int)threadIdx.x : (int)threadIdx.x & 63;
    if (lane < 64) {
        constexpr int PER = BINS / 64;
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) mine += hist[FROM_TOP ? BINS - 1 - (lane * PER + i) : lane * PER + i];
        const uint64_t upto = wave_scan(mine);
        if (lane == 63) out->total = upto;
        if (upto >= goal && upto - mine < goal) {
            uint64_t before = upto - mine;
            int i = 0;
            for (; i < PER - 1; ++i) {
                const uint64_t h = hist[FROM_TOP ? BINS - 1 - (lane * PER + i) : lane * PER + i];
                if (before + h >= goal) break;
                before += h;
            }
            out->before = before;
            out->bin = FROM_TOP ? BINS - 1 - (lane * PER + i) : lane * PER + i;
        }
    }
    together<W>();
}

// order-preserving key of a score
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __float_as_uint(x + 0.0f);                   // -0 and +0 are one score
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

// ----------------------------------------------------------------------------- bins
// Bins of a distance from the maximum: 2^(23 - SH) to an octave over 32 octaves from 2^-12 up, what lies outside in the first and the last.
// An inner bin holds distances that differ in their lower SH bits only; its own bins are the highest of those.
template <int BINS>
struct Bins {
    static constexpr int LOG = BINS == 512 ? 9 : BINS == 256 ? 8 : 7, SH = 28 - LOG;
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
// What a cut is found with
template <int NBINS>
struct Search {
    static constexpr int BINS = NBINS, LIST = 64;
    unsigned long long hist[BINS];
    Entry list[LIST];                                               // codes of the bin that a cut falls into
    float cut_x;
    int cut_i, length;
    unsigned long long cut_mass;                                    // up to and with the cut
    Found found;
};
// The codes kept of a row, in index order, once they are few, and the row's settings
template <int DT, int KEPT>
struct Few {
    alignas(16) typename Score<DT>::Raw x[KEPT];
    uint16_t i[KEPT];                                               // a row in LDS has at most 14848
    double T, P, min_p;
    int k, padded;
    float u;
    float max;
    int state;                                                      // the number of codes kept, or
    enum { DONE = -1, WHOLE = -2 };                                 // answered; to be worked on by the whole block
};
// A block's LDS next to the row
template <int W, int NBINS>
struct Shared {
    static constexpr int BINS = NBINS;
    Search<BINS> search;
    unsigned long long red[W];
    float redf[W];
    int redi[W], counts[W];
};

// W waves of a block work together on a row; with W = 1 one wave works on by itself, the others have left.
template <int W>
__device__ __forceinline__ void together()
{
    if (W > 1) __syncthreads();
    else {                                                           // a wave's LDS accesses are carried out in its order
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}
template <int DT, bool STAGED, int W, int BINS>
struct Draw {
    static constexpr int NT = 64 * W, FEW = 24;
    typedef Bins<BINS> B;
    Search<BINS> &s;
    unsigned long long *red;                                        // W each
    int *redi;
    View<DT, STAGED> row;
    float cut_x;                                                    // kept: at or before (cut_x, cut_i) in the order
    int cut_i;
    int begin, end, full;                                           // the wave's part; how many waves have a whole one, at least 1

    __device__ __forceinline__ Draw(Search<BINS> &s_, unsigned long long *red_, int *redi_, const View<DT, STAGED> &v) : s(s_), red(red_), redi(redi_), row(v), cut_x(-INFINITY), cut_i(-1)
    {                                                               // nothing with a score of -inf
        const int part = (row.n + 256 * W - 1) / (256 * W) * 256;
        begin = wave() * part;
        end = min(begin + part, row.n);
        full = max(row.n / part, 1);
    }
    // The wave's part of the row: codes [begin, end), a multiple of 256 up to the last one's
    __device__ __forceinline__ int wave() const { return W > 1 ? (int)(threadIdx.x >> 6) : 0; }
    __device__ __forceinline__ bool kept(float x, int c) const { return x > cut_x || (x == cut_x && c <= cut_i); }
    // all codes with scores from x up may be kept
    __device__ __forceinline__ void from_score(float x)
    {
        cut_x = x;
        cut_i = x > -INFINITY ? INT32_MAX : -1;
    }
    // f(x, c) for the kept codes, one at a time: a small loop, there are several of them and the instruction cache is shared
    template <typename F>
    __device__ __forceinline__ void each(F f) const
    {
        const int c1 = end;
#pragma unroll 1
        for (int c = begin + (threadIdx.x & 63); c < c1; c += 64) {
            const float x = row.one(c);
            if (kept(x, c)) f(x, c);
        }
    }
    // Sum of q(x) over the kept codes of the lane, four at a time without branches between them
    template <typename Q>
    __device__ __forceinline__ uint64_t sum(Q q) const
    {
        uint64_t t = 0;
        const int c1 = end;
#pragma unroll 1
        for (int c = begin + (threadIdx.x & 63) * 4; c < c1; c += 256) {
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
    // Sum of q(x) over all of the lane's codes; q(-inf) is 0
    template <typename Q>
    __device__ __forceinline__ uint64_t sum_all(Q q) const
    {
        uint64_t t = 0;
        const int c1 = end;
#pragma unroll 1
        for (int c = begin + (threadIdx.x & 63) * 4; c < c1; c += 256) {
            float x[4];
            row.four(c, x);
            t += (q(x[0]) + q(x[1])) + (q(x[2]) + q(x[3]));
        }
        return t;
    }
    // The same cut by radix selection over the bits of the score, for borders that hundreds of equal or nearly equal scores lie at.
    template <typename Q>
    __device__ __forceinline__ void find_cut_by_bits(uint64_t goal, Q q)
    {
        uint64_t prefix = 0, above = 0;
#pragma unroll 1
        for (int sh = 32; sh > 0;) {
            const int bits = min(B::LOG, sh);
            sh -= bits;
            together<W>();
            for (int b = (W > 1 ? (int)threadIdx.x : (int)threadIdx.x & 63); b < BINS; b += NT) s.hist[b] = 0;
            together<W>();
            each([&](float v, int) {
                const uint32_t key = key_of(v);
                if ((uint64_t)key >> (sh + bits) == prefix) atomicAdd(&s.hist[(key >> sh) & ((1u << bits) - 1u)], (unsigned long long)q(v));
            });
            together<W>();
            find_bin<BINS, true, W>(s.hist, goal - above, &s.found);
            prefix = prefix << bits | (uint64_t)s.found.bin;
            above += s.found.before;
        }
        // codes with the border's score are kept while above + j w < goal: the last of them by its index
        const float border = score_of((uint32_t)prefix);
        const uint64_t w = q(border);
        const int need = (int)((goal - above + w - 1) / w);
        if (threadIdx.x % NT == 0) s.cut_mass = above + (uint64_t)need * w;
        const int lane = threadIdx.x & 63, c0 = begin, c1 = end;
        uint32_t mine = 0;
        each([&](float v, int) { mine += v == border; });
        const int count = (int)wave_total(mine);
        if (lane == 0) redi[wave()] = count;
        together<W>();
        int before = 0;
        for (int v = 0; v < wave(); ++v) before += redi[v];
        if (before < need && before + count >= need) {
#pragma unroll 1
            for (int c = c0; c < c1; c += 256) {                    // the wave's lanes go round together
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                const int at = c + lane * 4;
                if (at < c1) row.four(at, x);
                uint32_t here = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) here += x[i] == border && kept(x[i], at + i);
                const uint32_t scan = wave_scan(here);
                int upto = before + (int)(scan - here);
                before += (int)from_lane(scan, 63);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (x[i] == border && kept(x[i], at + i) && ++upto == need) s.cut_i = at + i;
            }
        }
        together<W>();
        cut_x = border;
        cut_i = s.cut_i;
    }
    // Moves the cut to the code with which the mass of the kept codes, in their order, reaches `goal`.  q(x): a code's mass.  False: they have
    // less than that, the cut is where it was.
    template <typename Q>
    __device__ __forceinline__ bool find_cut(float mx, uint64_t goal, Q q)
    {
        const int tid = (W > 1 ? (int)threadIdx.x : (int)threadIdx.x & 63);
        int bin = 0, sub = -1;
        uint64_t above = 0;
#pragma unroll 1
        for (int level = 0; level < 2; ++level) {
            together<W>();
#pragma unroll 1
            for (int b = tid; b < BINS; b += NT) s.hist[b] = 0;
            if (tid == 0) s.length = 0;
            together<W>();
            each([&](float v, int) {
                const float d = mx - v;
                const int b = B::of(d);
                if (level == 0 || b == bin) atomicAdd(&s.hist[level == 0 ? b : B::inner(d)], (unsigned long long)q(v));
            });
            together<W>();
            find_bin<BINS, false, W>(s.hist, goal - above, &s.found);
            if (level == 0) {
                if (s.found.total < goal) return false;
                bin = s.found.bin;
            } else {
                sub = s.found.bin;
            }
            above += s.found.before;
            each([&](float v, int c) {
                const float d = mx - v;
                if (B::of(d) != bin || (sub >= 0 && B::inner(d) != sub)) return;
                const int e = atomicAdd(&s.length, 1);
                if (e < s.LIST) s.list[e] = Entry{v, c, (unsigned long long)q(v)};
            });
            together<W>();
            if (s.length <= FEW || bin == 0 || bin == BINS - 1) break;
        }
        const int many = s.length;
        if (many > s.LIST) {
            find_cut_by_bits(goal, q);
            return true;
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
                s.cut_mass = before + me.w;
            }
        }
        together<W>();
        cut_x = s.cut_x;
        cut_i = s.cut_i;
        return true;
    }
    // The cuts among the row's codes, and the draw.  Z: the mass of all codes if it is known (they may be more than this row's), else 0.
    template <typename A>
    __device__ __forceinline__ void finish(const Row &r, float mx, int k, double P, float u, uint64_t Z, A answer)
    {
        const int lane = threadIdx.x & 63;
        bool known = false;                                         // whether cut_mass is the kept mass
#pragma unroll 1
        for (int stage = 0; stage < 2; ++stage) {                   // one copy of find_cut for both: the code has to stay in the instruction cache
            uint64_t goal = (uint64_t)k;
            if (stage == 0) {
                if (k <= 0) continue;
            } else {
                if (!(P < 1.0)) continue;
                if (!Z) Z = total(sum([&](float v) { return r.units(v); }));
                goal = goal_of(P, Z);
            }
            const bool found = find_cut(mx, goal, [&](float v) { return stage == 0 ? (uint64_t)1 : r.units(v); });
            known = stage == 1 && found;
        }
        // the waves' sums, then the wave that the draw falls to goes over its part again (NaN min_p: nothing is under it); a wave by itself has
        // the sum from the cut already
        const uint64_t own = W == 1 && known && r.least == r.tiny ? s.cut_mass : wave_total(sum([&](float v) { return r.units(v, r.least); }));
        together<W>();
        if (lane == 0) red[wave()] = own;
        together<W>();
        uint64_t mass = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) mass += red[w];
        const double t = floor((double)(u > 0.f ? u : 0.f) * (double)mass);
        uint64_t target = t < (double)mass ? (uint64_t)t : mass - 1;
        if (target >= mass) target = mass - 1;
        uint64_t before = 0;
        int mine = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint64_t here = red[w];
            if (before + here <= target) {
                before += here;
                mine = w + 1;
            } else {
                break;
            }
        }
        if (wave() != mine) return;
        const int c1 = end;
#pragma unroll 1
        for (int c = begin; c < c1; c += 256) {                    // the wave's lanes go round together
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            const int at = c + lane * 4;
            if (at < c1) row.four(at, x);
            uint64_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = kept(x[i], at + i) ? r.units(x[i], r.least) : 0;
            const uint64_t four = (q[0] + q[1]) + (q[2] + q[3]), upto = wave_scan(four) + before;
            if (upto > target && upto - four <= target) {
                uint64_t b = upto - four;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (b <= target && b + q[i] > target) answer(at + i, x[i], mass);
                    b += q[i];
                }
            }
            before = from_lane(upto, 63);
            if (before > target) return;
        }
    }
    // over the waves
    __device__ __forceinline__ uint64_t total(uint64_t v) const
    {
        v = wave_total(v);
        if (W == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        uint64_t t = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) t += red[w];
        return t;
    }
    // codes are kept while less than this lies before them
    static __device__ __forceinline__ uint64_t goal_of(double P, uint64_t Z)
    {
        const double g = ceil(P * (double)Z);
        return g > 1.0 ? (uint64_t)g : 1;
    }
    // Puts the codes with x >= floor (> -inf) into the list of kept codes, in index order, where they are at most KEPT.  How many they are.  For
    // parts of at most 64 SLOTS codes: one comparison a code, and where none of 64 is kept nothing else.
    template <int SLOTS, int KEPT>
    __device__ __forceinline__ int compact(float floor, Few<DT, KEPT> &few)
    {
        const int lane = threadIdx.x & 63;
        float x[SLOTS];
        uint64_t m[SLOTS];
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
            const int c = begin + j * 64 + lane;
            x[j] = c < end ? row.one(c) : (float)-INFINITY;
        }
        int count = 0;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
            m[j] = __builtin_amdgcn_ballot_w64(x[j] >= floor);
            count += __popcll(m[j]);
        }
        if (lane == 0) redi[wave()] = count;
        together<W>();
        int at = 0, many = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            at += w < wave() ? redi[w] : 0;
            many += redi[w];
        }
        if (many <= KEPT) {
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int j = 0; j < SLOTS; ++j) {
                if (m[j]) {                                          // the same in all lanes
                    const int place = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m[j], (uint32_t)at));
                    if (x[j] >= floor) {
                        few.x[place] = Score<DT>::narrow(x[j]);
                        few.i[place] = (uint16_t)(begin + j * 64 + lane);
                    }
                    at += __popcll(m[j]);
                }
            }
            if (threadIdx.x < (unsigned)(-many & 3)) few.x[many + threadIdx.x] = Score<DT>::narrow(-INFINITY);      // to whole quads
        }
        return many;
    }
    // Puts the codes with x >= floor (> -inf) into x_ and index, in index order, where they are at most `room`.  How many they are.
    __device__ __forceinline__ int gather(float floor, typename Score<DT>::Raw *x_, int *index, int room)
    {
        const int lane = threadIdx.x & 63;
        int count = 0, at = 0, many = 0;
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            for (int c = begin + lane * 4; c < begin + (end - begin + 255) / 256 * 256 + lane * 4; c += 256) {      // all lanes go round together
                float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (c < end) row.four(c, x);
                uint64_t m[4];
                int place = at;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m[i] = __builtin_amdgcn_ballot_w64(x[i] >= floor);
                    place += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m[i], 0u));
                }
                const int here = __popcll(m[0]) + __popcll(m[1]) + __popcll(m[2]) + __popcll(m[3]);
                if (pass == 0) {
                    count += here;
                } else if (here) {
                    at += here;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (x[i] >= floor) {
                            x_[place] = Score<DT>::narrow(x[i]);
                            index[place++] = c + i;
                        }
                }
            }
            if (pass) break;
            if (lane == 0) redi[wave()] = count;
            together<W>();
#pragma unroll
            for (int w = 0; w < W; ++w) {
                at += w < wave() ? redi[w] : 0;
                many += redi[w];
            }
            if (many > room) return many;
        }
        if (threadIdx.x < (unsigned)(-many & 3)) x_[many + threadIdx.x] = Score<DT>::narrow(-INFINITY);      // to whole quads
        together<W>();
        return many;
    }
    // Leaves the codes with x >= floor (> -inf) only, each wave in its part of the row: packed in index order, index[place] the code.  How many a
    // wave's are.
    __device__ __forceinline__ int squeeze(typename Score<DT>::Raw *x_, uint16_t *index, float floor)
    {
        const int lane = threadIdx.x & 63;
        int at = begin;
#pragma unroll 1
        for (int c = begin + lane; c < begin + (end - begin + 255) / 256 * 256; c += 256) {      // all lanes go round together
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = c + j * 64 < end ? row.one(c + j * 64) : (float)-INFINITY;
            together<1>();                                           // they write at or before what they have read
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t m = __builtin_amdgcn_ballot_w64(x[j] >= floor);
                const int place = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, (uint32_t)at));
                if (x[j] >= floor) {
                    x_[place] = Score<DT>::narrow(x[j]);
                    index[place] = (uint16_t)(c + j * 64);
                }
                at += __popcll(m);
            }
        }
        if (lane < (-at & 3)) x_[at + lane] = Score<DT>::narrow(-INFINITY);      // to whole quads
        end = at;
        together<1>();
        return at - begin;
    }
};

// The lower end (a score's key, its low 16 bits cleared) of what at least `need` of the wave's values have: bit by bit from the top.
template <int G>
__device__ __forceinline__ uint32_t values_above(const uint32_t (&key)[G], int need)
{
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 16; --b) {
        const uint32_t with = t | 1u << b;
        int many = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) many += __popcll(__builtin_amdgcn_ballot_w64(key[g] >= with));
        if (many >= need) t = with;
    }
    return t;
}

// The block's maximum, and a score that at least `need` own maxima of each of the first `full` waves reach (the other waves' parts are shorter or
// empty); need 0: none.  With need = k / full at least k codes reach it.  own: maxima of G groups of the thread's codes.  Four groups cost 200
// instructions more than one, so only a wave that has a whole row by itself takes them.
template <int W, int G>
__device__ __forceinline__ float maximum(const float (&own)[G], int need, int full, float *redf, int *redi, float *floor)
{
    const int wave = W > 1 ? threadIdx.x >> 6 : 0;
    float most = own[0];
    uint32_t key[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        most = fmaxf(most, own[g]);
        key[g] = key_of(own[g]);
    }
    const float wmax = wave_max(most);
    uint32_t low = need ? (wave < full ? values_above(key, need) : 0xffffffffu) : 0;
    float mx = wmax;
    if (W > 1) {
        if ((threadIdx.x & 63) == 0) {
            redf[wave] = wmax;
            redi[wave] = (int)low;
        }
        __syncthreads();
        mx = redf[0];
        low = (uint32_t)redi[0];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            mx = fmaxf(mx, redf[w]);
            low = min(low, (uint32_t)redi[w]);
        }
    }
    *floor = low >= key_of(-INFINITY) ? score_of(low) : -INFINITY;
    return mx;
}
// The lowest index with the maximum
template <int DT, bool STAGED, int W>
__device__ __forceinline__ int first_of(float mx, float own, const View<DT, STAGED> &row, int c0, int c1, float *redf)
{
    int first = 1 << 24;                                            // indices are below
    if (own == mx) {
#pragma unroll 1
        for (int c = c0; c < c1 && first == 1 << 24; c += 256) {
            float y[4];
            row.four(c, y);
#pragma unroll
            for (int i = 3; i >= 0; --i) first = y[i] == mx ? c + i : first;
        }
    }
    together<W>();
    return (int)-block_max_f32<W>(-(float)first, redf);
}

constexpr int LISTED = 6144;             // codes of a row that does not fit the LDS
// One row by a block of W waves.  HELD: it is read once, into LDS (at `lds`), each wave's part by itself; else each time from memory, and what a
// bound leaves of it goes into LDS (LISTED scores and their indices).  index:
// NULL, or where V codes' indices may go, and few a list of the codes to keep.
template <int DT, bool HELD, int W, typename H, int KEPT>
__device__ __forceinline__ void draw_row(const SampleArgs &a, int64_t n, typename Score<DT>::Raw *lds, H &s, uint16_t *index, Few<DT, KEPT> *few)
{
    typedef Score<DT> S;
    constexpr int G = W == 1 ? 4 : 1;
    const int V = a.V, tid = threadIdx.x, lane = tid & 63;
    const auto answer = [&](int64_t i, float lp) {
        a.idx[n] = i;
        if (a.logp) a.logp[n] = lp;
    };
    if (a.padded && a.padded[n]) {
        if (tid == 0) answer(-1, 0.f);
        return;
    }
    const double T = a.T(n), P = a.P(n);
    const int k = a.k(n);
    const typename S::Raw *z = reinterpret_cast<const typename S::Raw *>(a.z) + n * a.ld;
    Draw<DT, HELD, W, H::BINS> d(s.search, s.red, s.counts, View<DT, HELD>{HELD ? lds : z, V, false});
    const View<DT, false> from{z, V, false};
    const int c0 = d.begin + lane * 4, c1 = d.end;
    float own[G], most = -INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g) own[g] = -INFINITY;
    for (int c = c0; c < c1; c += 1024) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = c + q * 256;
            if (at >= c1) continue;
            float x[4];
            from.four(at, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) own[q % G] = fmaxf(own[q % G], x[i]);
            if (HELD) *reinterpret_cast<typename S::Quad *>(lds + at) = typename S::Quad{S::narrow(x[0]), S::narrow(x[1]), S::narrow(x[2]), S::narrow(x[3])};
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) most = fmaxf(most, own[g]);
    float floor;
    float mx = maximum<W, G>(own, k > 0 && k <= 64 * G * d.full ? (k + d.full - 1) / d.full : 0, d.full, s.redf, s.redi, &floor);
    if (mx == -INFINITY) {
        if (tid == 0) answer(-1, 0.f);
        return;
    }
    if (!(T > 0.0)) {
        const int first = first_of<DT, HELD, W>(mx, most, d.row, c0, c1, s.redf);
        if (tid == 0) answer(first, 0.f);
        return;
    }
    if (mx == INFINITY) {                                           // the codes that have it share the draw
        mx = 0.f;
        floor = -INFINITY;
        if (HELD) {
            for (int c = d.begin + lane; c < c1; c += 64) lds[c] = S::narrow(S::widen(lds[c]) == INFINITY ? 0.f : -INFINITY);
        } else {
            d.row.inf = true;
        }
    }
    const Row row(mx, T, a.min(n), a.shift);
    uint64_t Z = 0;
    if (k <= 0 && P < 1.0) {
        Z = d.total(d.sum_all([&](float v) { return row.units(v); }));
        // The codes further than D from the maximum have at most V (exp(-D / T) 2^shift + 1) units.  That much may be missing of (1 - P) Z, less
        // what rounding P Z and Z to f64 takes.
        const double spare = (1.0 - P) * (double)Z * 0.999 - (double)V - 4096.0;
        if (spare > 0.0) {
            const double D = T * ln(fmax(ldexp((double)V, a.shift) / spare, 1.0));
            if (D < 1e30) floor = (float)((double)mx - fmax(D, 0.0) - fabs((double)mx) * 1e-6 - 1e-30);
        }
    }
    const bool squeezed = HELD && index && floor > -INFINITY;
    if (squeezed) {
        const int count = d.squeeze(lds, index, floor);
        if (W > 1) {
            if (lane == 0) s.counts[tid >> 6] = count;
            __syncthreads();
            int at = 0, many = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                at += w < tid >> 6 ? s.counts[w] : 0;
                many += s.counts[w];
            }
            if (many <= KEPT) {                                     // one wave does the rest, without barriers; the others make room
                for (int c = lane; c < count; c += 64) {
                    few->x[at + c] = lds[d.begin + c];
                    few->i[at + c] = index[d.begin + c];
                }
                if (tid < (-many & 3)) few->x[many + tid] = S::narrow(-INFINITY);
                __syncthreads();
                if (tid >= 64) return;
                Draw<DT, true, 1, H::BINS> l(s.search, s.red, s.counts, View<DT, true>{few->x, many, false});
                l.finish(row, mx, k, P, a.u[n], Z, [&](int c, float x, uint64_t mass) { answer(few->i[c], a.logp ? row.logp(x, mass) : 0.f); });
                return;
            }
        }
    }
    if (!HELD && floor > -INFINITY) {                               // the codes that a bound leaves, where they fit
        int *which = reinterpret_cast<int *>(lds + LISTED);
        const int many = d.gather(floor, lds, which, LISTED);
        if (many <= LISTED) {
            Draw<DT, true, W, H::BINS> l(s.search, s.red, s.counts, View<DT, true>{lds, many, false});
            l.finish(row, mx, k, P, a.u[n], Z, [&](int c, float x, uint64_t mass) { answer(which[c], a.logp ? row.logp(x, mass) : 0.f); });
            return;
        }
    }
    d.from_score(floor);
    d.finish(row, mx, k, P, a.u[n], Z, [&](int c, float x, uint64_t mass) { answer(squeezed ? index[c] : c, a.logp ? row.logp(x, mass) : 0.f); });
}
template <int DT, bool HELD, int W>
__global__ __launch_bounds__(64 * W, W == 8 ? 6 : W == 1 ? 5 : 4) void sample_kernel(const SampleArgs a)
{
    constexpr int KEPT = !HELD || W == 1 ? 4 : 192;                 // a whole row's wave needs no list beside it; three rows of 8192 to a compute unit
    typedef typename Score<DT>::Raw Raw;
    extern __shared__ __attribute__((aligned(16))) char staged[];
    __shared__ Shared<W, W == 1 ? 128 : 256> s;
    __shared__ Few<DT, KEPT> few;
    Raw *lds = reinterpret_cast<Raw *>(staged);
    draw_row<DT, HELD, W>(a, a.row0 + blockIdx.x, lds, s, a.squeezes ? reinterpret_cast<uint16_t *>(lds + (a.V + 3) / 4 * 4) : nullptr, &few);
}

// For many rows with top-k: a block takes W of them, one after the other as far as it needs the whole row - the next one is on its way
// meanwhile - and what is done on a short list of codes is left to the end, where each wave has a row's.  Rows without such a list
// come last, by the whole block.  One row a block and its list by one wave took 334 us where this takes 200 (16384 x 8192, top-k 100 and
// top-p 0.95): the row's 32 KB of LDS were held while seven of eight waves had nothing to do.
template <int DT, int W>
__global__ __launch_bounds__(64 * W, W == 8 ? 6 : 4) void sample_many_kernel(const SampleArgs a)
{
    typedef Score<DT> S;
    constexpr int KEPT = 256, QUADS = 4, BINS = 256;                // BINS: for a list's cuts
    typedef Few<DT, KEPT> F;
    extern __shared__ __attribute__((aligned(16))) char staged[];
    __shared__ Shared<W, 256> s;
    __shared__ F few[W];
    const int V = a.V, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t n0 = a.row0 + (int64_t)blockIdx.x * W;
    const int rows = (int)min((int64_t)W, a.rows - n0);
    typename S::Raw *lds = reinterpret_cast<typename S::Raw *>(staged);
    const auto answer = [&](int r, int64_t i, float lp) {
        a.idx[n0 + r] = i;
        if (a.logp) a.logp[n0 + r] = lp;
    };
    if (tid < rows) {
        F &f = few[tid];
        f.T = a.T(n0 + tid);
        f.P = a.P(n0 + tid);
        f.min_p = a.min(n0 + tid);
        f.k = a.k(n0 + tid);
        f.u = a.u[n0 + tid];
        f.padded = a.padded && a.padded[n0 + tid];
        f.state = F::DONE;
    }
    Draw<DT, true, W, 256> d(s.search, s.red, s.counts, View<DT, true>{lds, V, false});
    const int c0 = d.begin + lane * 4, c1 = d.end;                // a lane has at most QUADS quads
    typename S::Raw4 raw[QUADS];
    const auto load = [&](int r) {
        const typename S::Raw *z = reinterpret_cast<const typename S::Raw *>(a.z) + (n0 + r) * a.ld;
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int c = c0 + q * 256;
            if (c + 4 <= c1) {
                raw[q] = *reinterpret_cast<const typename S::Raw4 *>(z + c);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[q][i] = c + i < c1 ? z[c + i] : S::narrow(-INFINITY);
            }
        }
    };
    load(0);
    const int need = a.k0 > 0 && a.k0 <= 64 * d.full ? (a.k0 + d.full - 1) / d.full : 0;      // k is one for all rows here
    __syncthreads();
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
        const bool greedy = !(few[r].T > 0.0), padded = few[r].padded;
        float own[1] = {-INFINITY};                                 // the thread's maximum
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {                           // each wave reads what it wrote itself: no barrier
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = clean(S::widen(raw[q][i]));
                own[0] = fmaxf(own[0], x[i]);
            }
            if (c0 + q * 256 < c1)
                *reinterpret_cast<typename S::Quad *>(lds + c0 + q * 256) = typename S::Quad{S::narrow(x[0]), S::narrow(x[1]), S::narrow(x[2]), S::narrow(x[3])};
        }
        if (r + 1 < rows && !few[r + 1].padded) load(r + 1);
        float floor;
        const float mx = maximum<W, 1>(own, greedy ? 0 : need, d.full, s.redf, s.redi, &floor);
        int state = F::DONE;
        if (padded || mx == -INFINITY) {
            if (tid == 0) answer(r, -1, 0.f);
        } else if (greedy) {
            const int first = first_of<DT, true, W>(mx, own[0], d.row, c0, c1, s.redf);
            if (tid == 0) answer(r, first, 0.f);
        } else {
            state = F::WHOLE;
            if (floor > -INFINITY && mx < INFINITY) {
                const int many = d.template compact<4 * QUADS>(floor, few[r]);
                if (many <= KEPT) state = many;
            }
        }
        if (tid == 0) {
            few[r].max = mx;
            few[r].state = state;
        }
        __syncthreads();
    }
    if (wave < rows && few[wave].state >= 0) {
        const F &f = few[wave];
        const Row row(f.max, f.T, f.min_p, a.shift);
        Search<BINS> &there = reinterpret_cast<Search<BINS> *>(staged)[wave];      // in the place of the rows
        Draw<DT, true, 1, BINS> l(there, s.red + wave, s.counts + wave, View<DT, true>{f.x, f.state, false});
        l.finish(row, f.max, f.k, f.P, f.u, 0, [&](int c, float x, uint64_t mass) { answer(wave, f.i[c], a.logp ? row.logp(x, mass) : 0.f); });
    }
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
        if (few[r].state != F::WHOLE) continue;
        __syncthreads();
        SampleArgs b = a;
        asm volatile("" : "+s"(b.V));                               // nothing of the body is worked out before the loop: it would be spilled
        draw_row<DT, true, W>(b, n0 + r, lds, s, nullptr, (F *)nullptr);
    }
}

}  // namespace mq

using namespace mq;

// Waves a row: with many rows as few as keep a compute unit's 32 waves busy next to the rows' LDS, with too few rows to fill the chip as many
// as the row has quads for, up to 16.
constexpr size_t ROOM = 58 * 1024;       // for a row and its indices: LDS that needs no leave from the runtime, less the kernels' own
template <int DT>
static size_t row_bytes(int V) { return ((size_t)V + 3) / 4 * 4 * sizeof(typename Score<DT>::Raw); }
template <int DT, int W>
static void sample_go(SampleArgs a, hipStream_t s)
{
    const size_t row = row_bytes<DT>(a.V), index = (size_t)a.V * sizeof(uint16_t);
    a.squeezes = a.top_k || a.k0 > 0 || a.top_p || a.p0 < 1.0;
    hipLaunchKernelGGL((sample_kernel<DT, true, W>), dim3((unsigned)(a.rows - a.row0)), dim3(64 * W), row + (a.squeezes ? index : 0), s, a);
}
template <int DT, int W>
static void sample_many(const SampleArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((sample_many_kernel<DT, W>), dim3((unsigned)((a.rows - a.row0 + W - 1) / W)), dim3(64 * W), std::max(row_bytes<DT>(a.V), W * sizeof(Search<256>)), s, a);
}
// Waves a row: fewer with more rows, whose waves fill the chip without barriers between them.  Measured (f32, normal scores with deviation 3;
// us without a filter / top-p 0.95 / top-k 100 and top-p 0.95):
//   1000 codes: 1024 rows 7.0 / 16.0 / 17.5 with four waves, 8.0 / 19.0 / 19.3 with one; 4096 rows 17.6 / 41.6 / 31.9, 14.8 / 29.2 / 27.7
//   4096 codes: 256 rows 6.8 / 13.8 / 17.0 with eight, 8.3 / 17.5 / 17.8 with four; 1024 rows 13.5 / 29.1 / 24.0, 13.7 / 26.9 / 20.1
//   8192 codes: 256 rows 8.7 / 18.5 / 20.1 with sixteen, 9.4 / 19.9 / 17.8 with eight; 512 rows 14.1 / 33.6 / 36.0, 12.4 / 26.0 / 19.7
// The kernel for many rows wants enough of them for every compute unit (top-k 100 and top-p 0.95: 8192 codes, 2048 rows 71 against 55 us, 4096 87
// against 100; 4096 codes, 2048 rows 33 against 36, 4096 43 against 66; 2048 codes never pays) and a k whose list is short (8192 codes, 16384
// rows: k = 128 199 us, k = 160 436 against 263; 4096 codes, 4096 rows: k = 100 43 against 66, k = 128 47 against 45).
template <int DT>
static void sample_launch(const SampleArgs &a, hipStream_t s)
{
    const int64_t n = a.rows - a.row0;
    const int k = a.top_k ? 0 : a.k0;
    const bool greedy = !a.temperature && a.t0 == 0.0;
    if (row_bytes<DT>(a.V) + a.V * sizeof(uint16_t) > ROOM) {
        const size_t room = LISTED * (sizeof(typename Score<DT>::Raw) + sizeof(int));
        if (n <= 256) hipLaunchKernelGGL((sample_kernel<DT, false, 16>), dim3((unsigned)n), dim3(1024), room, s, a);
        else hipLaunchKernelGGL((sample_kernel<DT, false, 8>), dim3((unsigned)n), dim3(512), room, s, a);
    }
    else if (a.V <= 1024) n < 2048 ? sample_go<DT, 4>(a, s) : sample_go<DT, 1>(a, s);
    else if (a.V <= 4096) n <= 512 ? sample_go<DT, 8>(a, s) : n >= 4096 && a.V > 2048 && k > 0 && k <= 100 ? sample_many<DT, 4>(a, s) : sample_go<DT, 4>(a, s);
    else if (a.V <= 8192) n <= 256 && k <= 0 ? sample_go<DT, 16>(a, s) : n >= 4096 && (greedy || (k > 0 && k <= 128)) ? sample_many<DT, 8>(a, s) : sample_go<DT, 8>(a, s);
    else sample_go<DT, 16>(a, s);
}

extern "C" int mq_sample_codes(const mqSampleDesc *d, const void *logits, const float *uniform, const float *temperature, const int32_t *top_k,
                               const float *top_p, const float *min_p, const uint8_t *padded, int64_t *idx, float *logp, mqStream stream)
{
    MQ_REQUIRE(d && logits && uniform && idx, "mq_sample_codes: NULL argument");
    MQ_REQUIRE(d->dtype >= 0 && d->dtype <= 2, "mq_sample_codes: dtype %d (0 f32, 1 bf16, 2 f16)", d->dtype);
    MQ_REQUIRE(d->rows > 0 && d->rows < INT32_MAX && d->codes > 0 && d->codes <= (1 << 19) && d->row_stride >= d->codes,
               "mq_sample_codes: bad sizes (rows %lld, codes %d of at most 2^19, row stride %lld)", (long long)d->rows, d->codes, (long long)d->row_stride);
    MQ_REQUIRE(temperature || d->temperature >= 0.0, "mq_sample_codes: temperature %g", d->temperature);
    MQ_REQUIRE(top_k || d->top_k >= 0, "mq_sample_codes: top_k %d", d->top_k);
    MQ_REQUIRE(top_p || (d->top_p >= 0.0 && d->top_p <= 1.0), "mq_sample_codes: top_p %g is not in [0, 1]", d->top_p);
    MQ_REQUIRE(min_p || (d->min_p >= 0.0 && d->min_p <= 1.0), "mq_sample_codes: min_p %g is not in [0, 1]", d->min_p);
    int bits = 0;
    while ((1ll << bits) < d->codes) ++bits;
    const int shift = 62 - bits < 51 ? 62 - bits : 51;
    SampleArgs a{logits, d->row_stride, d->codes, shift, uniform, temperature, top_p, min_p, top_k, d->temperature, d->top_p, d->min_p, d->top_k, padded, idx, logp, 0, 0, 0};
    constexpr int64_t MOST = 1 << 21;                               // rows a launch: one holds under 2^32 threads
    for (a.row0 = 0; a.row0 < d->rows; a.row0 = a.rows) {
        a.rows = std::min(a.row0 + MOST, d->rows);
        if (d->dtype == 0) sample_launch<0>(a, S(stream));
        else if (d->dtype == 1) sample_launch<1>(a, S(stream));
        else sample_launch<2>(a, S(stream));
    }
    MQ_LAUNCH_CHECK("mq_sample_codes");
    return 0;
}
