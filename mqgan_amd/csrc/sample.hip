// Drawing a code per row of scores: temperature, top-k, top-p, min-p, from given uniform numbers.
//
//   order the codes by (score descending, index ascending); w = exp((z - max) / T)
//   top-k: the first k;  top-p: of those, every code before which less than top_p of their mass lies (the first always);
//   min-p: of those, w >= min_p (of the largest's weight 1)
//   drawn: the first code in INDEX order with (mass of the kept codes up to and with it) > u * (mass of all kept codes)
// T <= 0: the largest score, lowest index.  -inf and NaN are never drawn; a row of nothing else gives -1; where +inf occurs, the
// +inf codes share the draw evenly.
//
// Masses are whole numbers: w rounded to units of 2^-(62 - ceil(log2 V)), exp in f64.  Their sums are exact whatever the order of the
// additions, so histograms by atomics, scans and tree sums all agree to the last bit, and a cut or a draw next to a border falls the
// same way on every run.  With f32 masses a row of 8192 codes would be drawn next to a border about once in 1000 rows.  A weight under
// the unit counts as one unit (2^-49 at V = 8192) unless exp gives 0.
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

template <int DT>
__device__ __forceinline__ float score(const void *z, int64_t i)
{
    float x;
    if (DT == 0) x = reinterpret_cast<const float *>(z)[i];
    else if (DT == 1) x = __uint_as_float((uint32_t) reinterpret_cast<const uint16_t *>(z)[i] << 16);
    else x = (float)reinterpret_cast<const _Float16 *>(z)[i];
    return x == x ? x + 0.0f : -INFINITY;            // NaN is never drawn; -0 and +0 are one score
}
// order-preserving key; -inf is the lowest of the keys that occur
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr uint32_t KEY_NONE = 0x007fffffu;           // key_of(-inf)

struct Row {
    float max;
    double t;
    int shift;
};
__device__ __forceinline__ double weight_of(float x, const Row &r)
{
    return r.max == INFINITY ? (x == INFINITY ? 1.0 : 0.0) : exp(((double)x - (double)r.max) / r.t);
}
__device__ __forceinline__ uint64_t units_of(double w, int shift)
{
    const uint64_t q = (uint64_t)(ldexp(w, shift) + 0.5);
    return q ? q : (w > 0.0 ? 1u : 0u);
}

// block of 256: inclusive scan of v over the threads; *total = sum.  red: 4 entries
template <typename U>
__device__ __forceinline__ U block_scan(U v, U *red, U *total)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const U t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 63) red[w] = v;
    __syncthreads();
    U before = 0, all = 0;
    for (int i = 0; i < 4; ++i) {
        if (i < w) before += red[i];
        all += red[i];
    }
    *total = all;
    return v + before;
}

// What of a row is kept: scores above `key`, and the first `ties` codes (in index order) that have it.
struct Cut {
    uint32_t key;
    int ties;
};

template <int DT>
__global__ __launch_bounds__(256) void sample_kernel(const SampleArgs a)
{
    __shared__ float redf[4];
    __shared__ int redi[4];
    __shared__ unsigned long long red[4], hist[256], goal_above;
    __shared__ uint32_t picked;
    __shared__ int s_ties, found;
    const int64_t n = blockIdx.x;
    const int V = a.V, tid = threadIdx.x;
    if (a.padded && a.padded[n]) {
        if (tid == 0) {
            a.idx[n] = -1;
            if (a.logp) a.logp[n] = 0.f;
        }
        return;
    }
    const int64_t at = n * a.ld;
    const double T = a.temperature ? (double)a.temperature[n] : a.t0;
    const double P = a.top_p ? (double)a.top_p[n] : a.p0;
    double mp = a.min_p ? (double)a.min_p[n] : a.m0;
    mp = mp > 1.0 ? 1.0 : mp;
    const int k = a.top_k ? a.top_k[n] : a.k0;
    // the largest score and its lowest index
    float mx = -INFINITY;
    for (int i = tid; i < V; i += 256) mx = fmaxf(mx, score<DT>(a.z, at + i));
    mx = wave_max(mx);
    if ((tid & 63) == 0) redf[tid >> 6] = mx;
    __syncthreads();
    Row r;
    r.max = fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3]));
    r.t = T;
    r.shift = a.shift;
    if (r.max == -INFINITY) {
        if (tid == 0) {
            a.idx[n] = -1;
            if (a.logp) a.logp[n] = 0.f;
        }
        return;
    }
    if (!(T > 0.0)) {
        int first = INT32_MAX;
        for (int i = tid; i < V; i += 256)
            if (score<DT>(a.z, at + i) == r.max) { first = i; break; }
        for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
        if ((tid & 63) == 0) redi[tid >> 6] = first;
        __syncthreads();
        if (tid == 0) {
            a.idx[n] = min(min(redi[0], redi[1]), min(redi[2], redi[3]));
            if (a.logp) a.logp[n] = 0.f;
        }
        return;
    }
    Cut cut = {KEY_NONE, 0};
    // top-k: the k-th key from above, eight bits at a time
    if (k > 0 && k < V) {
        uint32_t prefix = 0;
        uint64_t need = (uint64_t)k;
        bool all = false;
        for (int sh = 24; sh >= 0 && !all; sh -= 8) {
            hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += 256) {
                const uint32_t key = key_of(score<DT>(a.z, at + i));
                if (key > KEY_NONE && (sh == 24 || (key >> (sh + 8)) == prefix)) atomicAdd(&hist[(key >> sh) & 255u], 1ull);
            }
            __syncthreads();
            uint64_t total;
            const uint64_t mine = hist[255 - tid];
            const uint64_t upto = block_scan<uint64_t>(mine, reinterpret_cast<uint64_t *>(red), &total);
            if (sh == 24 && total <= need) {
                all = true;                                         // fewer codes than k have a score at all
            } else {
                if (upto >= need && upto - mine < need) {
                    picked = (uint32_t)(255 - tid);
                    goal_above = upto - mine;
                }
                __syncthreads();
                prefix = (prefix << 8) | picked;
                need -= goal_above;
            }
            __syncthreads();
        }
        if (!all) cut = Cut{prefix, (int)need};
    }
    // mass of what is kept so far; ties of the border all have one weight
    const auto mass = [&](float x) -> uint64_t {
        const uint32_t key = key_of(x);
        return key > cut.key ? units_of(weight_of(x, r), r.shift) : 0;
    };
    if (P < 1.0) {
        uint64_t part = 0, Z;
        int tied = 0, alltied;
        float tiex = 0.f;
        for (int i = tid; i < V; i += 256) {
            const float x = score<DT>(a.z, at + i);
            part += mass(x);
        }
        block_scan<uint64_t>(part, reinterpret_cast<uint64_t *>(red), &Z);
        (void)tied; (void)alltied;
        uint64_t tiew = 0;
        if (cut.ties) {
            const uint32_t b = (cut.key & 0x80000000u) ? (cut.key & 0x7fffffffu) : ~cut.key;
            tiex = __uint_as_float(b);
            tiew = units_of(weight_of(tiex, r), r.shift);
            Z += tiew * (uint64_t)cut.ties;
        }
        double g = ceil(P * (double)Z);
        uint64_t goal = g > 1.0 ? (uint64_t)g : 1;                  // codes are kept while less than `goal` lies before them
        // the key at which the mass from above reaches the goal
        uint32_t prefix = 0;
        uint64_t above = 0;
        for (int sh = 24; sh >= 0; sh -= 8) {
            hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += 256) {
                const float x = score<DT>(a.z, at + i);
                const uint32_t key = key_of(x);
                if (key > cut.key && (sh == 24 || (key >> (sh + 8)) == prefix)) atomicAdd(&hist[(key >> sh) & 255u], (unsigned long long)mass(x));
            }
            __syncthreads();
            if (tid == 0 && cut.ties && (sh == 24 || (cut.key >> (sh + 8)) == prefix)) hist[(cut.key >> sh) & 255u] += tiew * (uint64_t)cut.ties;
            __syncthreads();
            uint64_t total;
            const uint64_t mine = hist[255 - tid];
            const uint64_t upto = block_scan<uint64_t>(mine, reinterpret_cast<uint64_t *>(red), &total) + above;
            if (upto >= goal && upto - mine < goal) {
                picked = (uint32_t)(255 - tid);
                goal_above = upto - mine;
            }
            __syncthreads();
            prefix = (prefix << 8) | picked;
            above = goal_above;
            __syncthreads();
        }
        // codes that have the border's score: kept while above + j w < goal
        const uint32_t b = (prefix & 0x80000000u) ? (prefix & 0x7fffffffu) : ~prefix;
        const uint64_t w = units_of(weight_of(__uint_as_float(b), r), r.shift);
        int ties = w ? (int)min((goal - above + w - 1) / w, (uint64_t)V) : 0;
        if (prefix == cut.key && cut.ties < ties) ties = cut.ties;
        cut = Cut{prefix, ties};
    }
    // ties in index order, min-p, then the draw: tiles of 256 codes
    uint64_t Z = 0;
    for (int pass = 0; pass < 2; ++pass) {
        uint64_t before = 0;
        int tiebefore = 0;
        uint64_t target = 0;
        if (pass == 1) {
            float u = a.u[n];
            u = u > 0.f ? u : 0.f;                                  // and a NaN
            const double t = floor((double)u * (double)Z);
            target = t < (double)Z ? (uint64_t)t : Z - 1;
            if (target >= Z) target = Z - 1;
            if (tid == 0) found = 0;
            __syncthreads();
        }
        for (int i0 = 0; i0 < V; i0 += 256) {
            const int i = i0 + tid;
            const float x = i < V ? score<DT>(a.z, at + i) : -INFINITY;
            const uint32_t key = key_of(x);
            int tied = i < V && key == cut.key && cut.ties ? 1 : 0, alltied;
            const int rank = block_scan<int>(tied, redi, &alltied) + tiebefore;
            tiebefore += alltied;
            const bool kept = i < V && key > KEY_NONE && (key > cut.key || (tied && rank <= cut.ties));
            const double w = kept ? weight_of(x, r) : 0.0;
            const uint64_t q = kept && !(w < mp) ? units_of(w, r.shift) : 0;
            uint64_t total;
            const uint64_t upto = block_scan<uint64_t>(q, reinterpret_cast<uint64_t *>(red), &total) + before;
            if (pass == 1 && upto > target && upto - q <= target) {
                a.idx[n] = i;
                if (a.logp) a.logp[n] = (float)(log(w) - log(ldexp((double)Z, -r.shift)));
                found = 1;
            }
            before += total;
            if (pass == 1) {
                __syncthreads();
                if (found) return;
            }
        }
        Z = before;
    }
    (void)s_ties;
}

}  // namespace mq

using namespace mq;

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
    SampleArgs a{logits, d->row_stride, d->codes, 62 - bits, uniform, temperature, top_p, min_p, top_k, d->temperature, d->top_p, d->min_p, d->top_k, padded, idx, logp};
    const dim3 grid((unsigned)d->rows);
    if (d->dtype == 0) hipLaunchKernelGGL(sample_kernel<0>, grid, dim3(256), 0, S(stream), a);
    else if (d->dtype == 1) hipLaunchKernelGGL(sample_kernel<1>, grid, dim3(256), 0, S(stream), a);
    else hipLaunchKernelGGL(sample_kernel<2>, grid, dim3(256), 0, S(stream), a);
    MQ_LAUNCH_CHECK("mq_sample_codes");
    return 0;
}
