// Balance loss of a codebook with per-code counts, and its gradient with respect to the scores.
//
//   p_n = softmax(z_n),  P_e = 1/Nv sum_{valid n} p_ne,  f_e = counts_e / (Nv K)
//   L = E sum_e f_e P_e,     dL/dz_ne = g E / Nv p_ne (f_e - sum_j f_j p_nj)
// E codes, K assignments a row, Nv rows that are not padded.  L is 1 where codes are used evenly and E where one code takes all.  The
// counts are whole numbers and carry no gradient.
//
// A row's statistics are an offset and a factor, p = factor * 2^(z log2 e - offset), and never one logarithm for both: a row of nothing but the
// type's lowest value has log(sum) far under half an ulp of its maximum.  The offset is the maximum times log2 e, rounded; all of a row
// uses the same, so its rounding, which is half an ulp of the OFFSET in an exponent, goes into the factor.  That holds while half an ulp is far
// under 1: at 2^20 it is 1/16, at 1e10 it would be 512 and every power 0 or infinite.  From 2^20 on the maximum itself is kept and z - maximum
// taken first: Offset.  A row of -inf alone has p = 0.  Padded rows are not read; their gradient is 0.
//
// Sums: a row's in f32, lane by lane and then as a tree; P's over rows in f32 within a team (a lane adds one row after the other, 16384 rows of 8192
// codes 32 of them, of 1024 codes eight), across teams of a wave and waves in f32 in a fixed order, across blocks and codes in f64.  At 129 x 1000
// the loss is off by 1.4e-7 of it where f64 sums of f32 shares are by 0.9e-7.
//
// Scores are read once forward and once backward, which is the floor: 16384 x 8192 bf16, a fifth padded, 30 us at the 7.1 TB/s of loads alone and
// 83 at the 5.84 TB/s of a copy.  Measured: rows 65 us, partial sums 12, loss 6; gradient 85 (non-temporal accesses: a copy's rate).
// Forward: vector units busy 89 % of the time (12.5 instructions a score), an exchange over waves a row: 512 blocks of eight waves, two rows in
// flight; 256 blocks 89 us for the three kernels where these take 80, 768 82, 1024 87 (more partial sums), four waves of four quads 78, sixteen of
// one 98.  16384 x 1024 f32: 21 + 5 + 3, gradient 20.  Calls of some hundred rows are launches, the autograd engine and the wrapper: 18 us of
// kernels in 105 us, of which a step that does nothing takes 37.
#include "common.h"

namespace mq {

template <typename T> struct Ld;
template <> struct Ld<float> {
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <> struct Ld<uint16_t> {                                       // bf16
    static __device__ __forceinline__ float get(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ __forceinline__ void put(uint16_t *p, float v)
    {
        const uint32_t b = __float_as_uint(v);                          // to nearest even; a NaN stays one
        *p = (b & 0x7fffffffu) > 0x7f800000u ? (uint16_t)((b >> 16) | 0x40) : (uint16_t)((b + 0x7fffu + ((b >> 16) & 1u)) >> 16);
    }
};
template <> struct Ld<_Float16> {
    static __device__ __forceinline__ float get(const _Float16 *p) { return (float)*p; }
    static __device__ __forceinline__ void put(_Float16 *p, float v) { *p = (_Float16)v; }
};

constexpr float LOG2E = 1.44269504088896340736f;
struct Offset {
    float o;                             // max log2 e, or the maximum itself where it is huge
    bool huge;
    __device__ __forceinline__ explicit Offset(float m) : o(m == -INFINITY ? 0.f : m), huge(fabsf(o) > 1048576.f)
    {
#pragma clang fp contract(off)
        o = huge ? o : o * LOG2E;
    }
    __device__ __forceinline__ Offset(float2 stats) : o(stats.x), huge(stats.y < 0.f) {}
    __device__ __forceinline__ float exp(float z) const { return __builtin_amdgcn_exp2f(huge ? (z - o) * LOG2E : fmaf(z, LOG2E, -o)); }
};
// What a sum over part of a row, whose maximum is m, counts for in the row's, whose maximum is M: the difference of the two offsets as the powers
// took them, rounded once, also where only one of them is huge (maxima on both sides of 2^20 may be a fraction apart).  Not contracted: an FMA
// of m, LOG2E and the other offset takes the exact product where the powers took the rounded one, half an ulp of the offset off.
__device__ __forceinline__ float rebase(float m, float M)
{
#pragma clang fp contract(off)
    const Offset a(m), b(M);
    const float same = a.huge ? (a.o - b.o) * LOG2E : a.o - b.o;
    const float mixed = a.huge ? fmaf(a.o, LOG2E, -b.o) : fmaf(-b.o, LOG2E, a.o);
    return __builtin_amdgcn_exp2f(a.huge == b.huge ? same : mixed);
}
// (offset, factor); the factor is negative where the offset is the maximum itself
__device__ __forceinline__ float2 stats_of(float m, float s)
{
    const Offset a(m);
    const float f = m == -INFINITY ? s : 1.0f / s;              // s is 0 in a row of -inf alone, or a NaN
    return make_float2(a.o, a.huge ? -f : f);
}
// x <- 2^(x log2 e - offset); the two ways as a branch, which all lanes of a wave nearly always take together
template <int NQ, int EPQ>
__device__ __forceinline__ void exp_all(float (&x)[NQ][EPQ], const Offset &f)
{
    if (__builtin_amdgcn_ballot_w64(f.huge) == 0) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < EPQ; ++i) x[j][i] = __builtin_amdgcn_exp2f(fmaf(x[j][i], LOG2E, -f.o));
    } else {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < EPQ; ++i) x[j][i] = f.exp(x[j][i]);
    }
}

// ----------------------------------------------------------------------------- a row in registers, read once
// A team of TL lanes (a part of a wave), or of W whole waves (then TL = 64), holds one row as NQ quads of 16 bytes a lane: lane t the
// columns (j TL W + t) EPQ .. + EPQ - 1, j < NQ.  The columns of a lane are the same for every row, so the sums over rows are registers too
// and the row's own maximum and sum are the only things that cross lanes (shuffles; with W > 1 one LDS exchange and one barrier a row,
// the buffer alternating).  Two rows are in flight behind the one that is worked on, as they lie in memory (bf16 takes half the registers).
template <typename T> struct Wide {
    static constexpr int EPQ = 16 / sizeof(T);
};
__device__ __forceinline__ float half_bits(uint32_t lo16, float) { return 0.f; }
__device__ __forceinline__ float half_bits(uint32_t lo16, uint16_t) { return __uint_as_float(lo16 << 16); }
__device__ __forceinline__ float half_bits(uint32_t lo16, _Float16) { return (float)__builtin_bit_cast(_Float16, (uint16_t)lo16); }
template <typename T>
__device__ __forceinline__ void widen(const uint4 &q, float (&x)[Wide<T>::EPQ])
{
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[(2 * i) % Wide<T>::EPQ] = half_bits(w[i] & 0xffffu, T());
            x[(2 * i + 1) % Wide<T>::EPQ] = half_bits(w[i] >> 16, T());
        }
    }
}
template <typename T> struct Lowest;                           // -inf in every element
template <> struct Lowest<float> { static constexpr uint32_t WORD = 0xff800000u; };
template <> struct Lowest<uint16_t> { static constexpr uint32_t WORD = 0xff80ff80u; };
template <> struct Lowest<_Float16> { static constexpr uint32_t WORD = 0xfc00fc00u; };

// a quad from column c; columns at and after E read as -inf.  VEC: rows start on 16 bytes and E is a whole number of quads
// NT: a non-temporal load.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T, bool VEC, bool NT>
__device__ __forceinline__ uint4 load_quad(const T *row, int c, int E)
{
    constexpr uint32_t low = Lowest<T>::WORD;
    if (VEC) {
        u32x4 q = {low, low, low, low};
        if (c < E) q = NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + c)) : *reinterpret_cast<const u32x4 *>(row + c);
        return make_uint4(q.x, q.y, q.z, q.w);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) {
            w[i] = c + i < E ? reinterpret_cast<const uint32_t *>(row)[c + i] : low;
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(row);
            const uint32_t lo = c + 2 * i < E ? h[c + 2 * i] : low & 0xffffu, hi = c + 2 * i + 1 < E ? h[c + 2 * i + 1] : low & 0xffffu;
            w[i] = lo | hi << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_quad(T *row, int c, int E, const float (&x)[Wide<T>::EPQ])
{
    constexpr int EPQ = Wide<T>::EPQ;
    if (VEC) {
        if (c < E) {
            alignas(16) T q[EPQ];
#pragma unroll
            for (int i = 0; i < EPQ; ++i) Ld<T>::put(q + i, x[i]);
            __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(q), reinterpret_cast<u32x4 *>(row + c));
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPQ; ++i)
            if (c + i < E) Ld<T>::put(row + c + i, x[i]);
    }
}
template <int TL> __device__ __forceinline__ float team_max(float v)
{
    if (TL == 64) return wave_max(v);
#pragma unroll
    for (int o = TL / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
template <int TL> __device__ __forceinline__ float team_sum(float v)
{
    if (TL == 64) return wave_sum(v);
#pragma unroll
    for (int o = TL / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float row16_max(float v)
{
    v = fmaxf(v, dpp_mov<0xB1>(v, v));
    v = fmaxf(v, dpp_mov<0x4E>(v, v));
    v = fmaxf(v, dpp_mov<0x141>(v, v));
    return fmaxf(v, dpp_mov<0x140>(v, v));
}
__device__ __forceinline__ float row16_sum(float v)
{
    v += dpp_mov<0xB1>(0.f, v);
    v += dpp_mov<0x4E>(0.f, v);
    v += dpp_mov<0x141>(0.f, v);
    return v + dpp_mov<0x140>(0.f, v);
}

// The rows of a team, two of them in flight.  x0: the present row's quads, none: it is padded (its quads hold nothing then)
template <typename T, int TL, int NQ, int W, bool VEC, bool NT>
struct Rows {
    const T *z;
    int64_t ld, N, n, step;
    const uint8_t *padded;
    int E, t;
    uint4 x0[NQ], x1[NQ], x2[NQ];
    bool none, none1, none2;
    uint32_t pad3, pad4;                                        // the flags of the rows three and four on, as loaded: compared when their turn comes

    __device__ __forceinline__ uint32_t flag(int64_t r) const { return r >= N ? 1u : padded ? (uint32_t)padded[r] : 0u; }
    __device__ __forceinline__ void fetch(int64_t r, bool absent, uint4 (&x)[NQ]) const
    {
        if (absent) return;
        const T *row = z + r * ld;
#pragma unroll
        for (int j = 0; j < NQ; ++j) x[j] = load_quad<T, VEC, NT>(row, (j * TL * W + t) * Wide<T>::EPQ, E);
    }
    __device__ __forceinline__ void begin()
    {
        none = flag(n) != 0;
        none1 = flag(n + step) != 0;
        none2 = flag(n + 2 * step) != 0;
        pad3 = flag(n + 3 * step);
        fetch(n, none, x0);
        fetch(n + step, none1, x1);
    }
    // Issues the row after next, and before it the flag of the row four on: loads return in order, a flag behind the row's quads would be
    // waited for together with them.
    __device__ __forceinline__ void ahead()
    {
        pad4 = flag(n + 4 * step);
        fetch(n + 2 * step, none2, x2);
    }
    __device__ __forceinline__ void advance()
    {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            x0[j] = x1[j];
            x1[j] = x2[j];
        }
        none = none1;
        none1 = none2;
        none2 = pad3 != 0;
        pad3 = pad4;
        n += step;
    }
};

// The assignments as the kernels take them: int32, or int64 with wide = 1
struct Codes {
    const void *p;
    int wide, K;
    __device__ __forceinline__ int64_t at(int64_t i) const { return wide ? reinterpret_cast<const int64_t *>(p)[i] : (int64_t) reinterpret_cast<const int32_t *>(p)[i]; }
};

// Besides its rows a block of W == 1 counts a slice of the assignments (and of the valid rows) in LDS: pcount (blocks, E + 1).
template <typename T, int TL, int NQ, int W, bool VEC>
__global__ __launch_bounds__(W > 1 ? 64 * W : 256) void balance_fwd_kernel(const T *__restrict__ z, int64_t ld, const uint8_t *__restrict__ padded,
                                                                          int64_t N, int E, float2 *__restrict__ stats, float *__restrict__ part,
                                                                          const Codes codes, int32_t *__restrict__ pcount)
{
    constexpr int TEAMS = W > 1 ? 1 : 256 / TL, EPQ = Wide<T>::EPQ;
    __shared__ float2 ex[2][W];
    extern __shared__ float cols[];                             // W == 1: the block's counts, then its column sums
    if (W == 1) {
        int *hist = reinterpret_cast<int *>(cols);
        for (int c = threadIdx.x; c <= E; c += 256) hist[c] = 0;
        __syncthreads();
        const int64_t per = (N + gridDim.x - 1) / gridDim.x, r0 = blockIdx.x * per, r1 = r0 + per < N ? r0 + per : N;
        for (int64_t i = r0 * codes.K + threadIdx.x; i < r1 * codes.K; i += 256) {
            const int64_t r = codes.K == 1 ? i : i / codes.K, c = codes.at(i);
            if (padded && padded[r]) continue;
            if (c >= 0 && c < E) atomicAdd(hist + c, 1);
            if (i == r * codes.K) atomicAdd(hist + E, 1);
        }
        __syncthreads();
        int32_t *to = pcount + (int64_t)blockIdx.x * (E + 1);
        for (int c = threadIdx.x; c <= E; c += 256) to[c] = hist[c];
        __syncthreads();
    }
    Rows<T, TL, NQ, W, VEC, false> a;
    a.z = z; a.ld = ld; a.N = N; a.padded = padded; a.E = E;
    a.t = W > 1 ? threadIdx.x : threadIdx.x % TL;
    a.n = (int64_t)blockIdx.x * TEAMS + (W > 1 ? 0 : threadIdx.x / TL);
    a.step = (int64_t)gridDim.x * TEAMS;
    float acc[NQ][EPQ] = {};
    a.begin();
    int parity = 0;
    // the trip count is one for the whole block (a team beyond the last row finds its rows absent), so lanes of a wave stay together
    for (int64_t left = N - (int64_t)blockIdx.x * TEAMS; left > 0; left -= a.step) {
        a.ahead();
        if (TL < 64 || !a.none) {                               // teams of one wave run side by side; a wave or block of its own skips
            float e[NQ][EPQ], m = -INFINITY, s = 0.f;
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                widen<T>(a.x0[j], e[j]);
#pragma unroll
                for (int i = 0; i < EPQ; ++i) {
                    if (TL < 64) e[j][i] = a.none ? -INFINITY : e[j][i];
                    m = fmaxf(m, e[j][i]);
                }
            }
            m = team_max<TL>(m);
            exp_all(e, Offset(m));
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) s += e[j][i];
            s = team_sum<TL>(s);
            float M = m, S = s;
            if (W > 1) {
                if ((threadIdx.x & 63) == 0) ex[parity][threadIdx.x >> 6] = make_float2(m, s);
                __syncthreads();
                const int w = threadIdx.x & 15;                 // a lane a wave's pair; W <= 16
                const float2 o = w < W ? ex[parity][w] : make_float2(-INFINITY, 0.f);
                M = row16_max(o.x);
                S = row16_sum(o.y == 0.f ? 0.f : o.y * rebase(o.x, M));
                parity ^= 1;
            }
            const float f = s == 0.f ? 0.f : W > 1 ? rebase(m, M) / S : 1.0f / s;
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) acc[j][i] = fmaf(e[j][i], f, acc[j][i]);
            if (a.t == 0 && !a.none) stats[a.n] = stats_of(M, S);
        }
        a.advance();
    }
    float *out = part + (int64_t)blockIdx.x * E;
    if (W > 1) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < EPQ; ++i) {
                const int c = (j * TL * W + a.t) * EPQ + i;
                if (c < E) out[c] = acc[j][i];
            }
        return;
    }
    if (TL < 64) {                                              // the teams of a wave, in an order of their own that never changes
#pragma unroll
        for (int o = 32; o >= TL; o >>= 1)
#pragma unroll
            for (int i = 0; i < EPQ; ++i) acc[0][i] += __shfl_xor(acc[0][i], o, 64);
    }
    for (int w = 0; w < 4; ++w) {                               // then the waves, one after the other
        if ((int)(threadIdx.x >> 6) == w && (threadIdx.x & 63) < TL) {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) {
                    const int c = (j * TL + a.t) * EPQ + i;
                    if (c < E) cols[c] = w ? cols[c] + acc[j][i] : acc[j][i];
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < E; c += 256) out[c] = cols[c];
}

template <typename T, int TL, int NQ, int W, bool VEC>
__global__ __launch_bounds__(W > 1 ? 64 * W : 256) void balance_grad_kernel(const T *__restrict__ z, int64_t ld, const uint8_t *__restrict__ padded,
                                                                           int64_t N, int E, const float2 *__restrict__ stats,
                                                                           const float *__restrict__ f, const float *__restrict__ sums,
                                                                           const float *__restrict__ gout, T *__restrict__ dz)
{
    constexpr int TEAMS = W > 1 ? 1 : 256 / TL, EPQ = Wide<T>::EPQ;
    __shared__ float ex[2][W];
    Rows<T, TL, NQ, W, VEC, true> a;
    a.z = z; a.ld = ld; a.N = N; a.padded = padded; a.E = E;
    a.t = W > 1 ? threadIdx.x : threadIdx.x % TL;
    a.n = (int64_t)blockIdx.x * TEAMS + (W > 1 ? 0 : threadIdx.x / TL);
    a.step = (int64_t)gridDim.x * TEAMS;
    float fr[NQ][EPQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int i = 0; i < EPQ; ++i) {
            const int c = (j * TL * W + a.t) * EPQ + i;
            fr[j][i] = c < E ? f[c] : 0.f;
        }
    const float scale = gout[0] * ((float)E / sums[2 * (int64_t)E]);
    a.begin();
    const auto stat = [&](int64_t r, bool absent) { return absent ? make_float2(0.f, 0.f) : stats[r]; };
    float2 st = stat(a.n, a.none), st1 = stat(a.n + a.step, a.none1);
    int parity = 0;
    for (int64_t left = N - (int64_t)blockIdx.x * TEAMS; left > 0; left -= a.step) {
        a.ahead();
        const float2 st2 = stat(a.n + 2 * a.step, a.none2);
        float e[NQ][EPQ];
        if (TL < 64 || !a.none) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                widen<T>(a.x0[j], e[j]);
            }
            exp_all(e, Offset(st));
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) s = fmaf(fr[j][i], e[j][i], s);
            s = team_sum<TL>(s) * fabsf(st.y);
            if (W > 1) {
                if ((threadIdx.x & 63) == 0) ex[parity][threadIdx.x >> 6] = s;
                __syncthreads();
                s = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) s += ex[parity][w];
                parity ^= 1;
            }
            const float by = scale * fabsf(st.y);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) e[j][i] = by * e[j][i] * (fr[j][i] - s);
        }
        if (a.none) {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < EPQ; ++i) e[j][i] = 0.f;
        }
        if (a.n < N) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) store_quad<T, VEC>(dz + a.n * E, (j * TL * W + a.t) * EPQ, E, e[j]);
        }
        a.advance();
        st = st1;
        st1 = st2;
    }
}

// ----------------------------------------------------------------------------- wider books: the row's statistics first, then column sums
// block of 256: (m, s) pairs joined; red is 8 floats
__device__ __forceinline__ float2 block_join(float m, float s, float *red)
{
    const float wm = wave_max(m);
    const float ws = wave_sum(s == 0.f ? 0.f : s * rebase(m, wm));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = wm;
        red[4 + (threadIdx.x >> 6)] = ws;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float S = 0.f;
    for (int i = 0; i < 4; ++i) S += red[4 + i] == 0.f ? 0.f : red[4 + i] * rebase(red[i], M);
    return make_float2(M, S);
}

template <typename T>
__global__ __launch_bounds__(256) void balance_rows_kernel(const T *__restrict__ z, int64_t ld, const uint8_t *__restrict__ padded, int E,
                                                           float2 *__restrict__ stats)
{
    __shared__ float red[8];
    const int64_t n = blockIdx.x;
    if (padded && padded[n]) return;
    const T *row = z + n * ld;
    float m = -INFINITY, s = 0.f;
    for (int e = threadIdx.x; e < E; e += 256) {
        const float x = Ld<T>::get(row + e);
        const float nm = fmaxf(m, x);
        s = (s == 0.f ? 0.f : s * rebase(m, nm)) + (x == -INFINITY ? 0.f : Offset(nm).exp(x));
        m = nm;
    }
    const float2 j = block_join(m, s, red);
    if (threadIdx.x == 0) stats[n] = stats_of(j.x, j.y);
}

// column sums of p over a chunk of rows: a thread owns one column, no reduction over threads
template <typename T>
__global__ __launch_bounds__(256) void balance_cols_kernel(const T *__restrict__ z, int64_t ld, const uint8_t *__restrict__ padded, int64_t N, int E,
                                                           int64_t chunk, const float2 *__restrict__ stats, float *__restrict__ part)
{
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e >= E) return;
    const int64_t n0 = (int64_t)blockIdx.y * chunk, n1 = n0 + chunk < N ? n0 + chunk : N;
    float a = 0.f;
    for (int64_t n = n0; n < n1; ++n) {
        if (padded && padded[n]) continue;
        const float2 st = stats[n];
        a = fmaf(Offset(st).exp(Ld<T>::get(z + n * ld + e)), fabsf(st.y), a);
    }
    part[(int64_t)blockIdx.y * E + e] = a;
}

// sums = {sum_n p_ne (E), counts (E), valid rows}: what data-parallel ranks add up before the loss is formed.  A block owns 32 columns and
// adds their partial sums (32 threads a column, in f64, joined in order).  The counts come as partial sums too (pcount), or - the forms
// without a histogram - each block reads all assignments for the ones that fall on its columns, four to a load (4 K / 32 bytes out of the
// L2 per score read), and one more block counts the valid rows.
constexpr int BL_COLS = 32;
typedef int int4u __attribute__((ext_vector_type(4), aligned(4)));
typedef long long2u __attribute__((ext_vector_type(2), aligned(8)));
__global__ __launch_bounds__(1024) void balance_sums_kernel(const float *__restrict__ part, const int32_t *__restrict__ pcount, int nparts, const Codes codes,
                                                            const uint8_t *__restrict__ padded, int N, int E, int32_t *__restrict__ counts,
                                                            float *__restrict__ sums)
{
    __shared__ double red[32][BL_COLS + 1];
    __shared__ int hist[BL_COLS];
    const int e0 = blockIdx.x * BL_COLS, c = threadIdx.x % BL_COLS, g = threadIdx.x / BL_COLS;
    if (threadIdx.x < BL_COLS) hist[threadIdx.x] = 0;
    __syncthreads();
    double a = 0.0;
    if (e0 + c < E) {
#pragma unroll 4
        for (int i = g; i < nparts; i += 32) a += (double)part[(int64_t)i * E + e0 + c];
    }
    red[g][c] = a;
    if (pcount) {
        int n = 0;
        if (e0 + c <= E) {
#pragma unroll 4
            for (int i = g; i < nparts; i += 32) n += pcount[(int64_t)i * (E + 1) + e0 + c];
        }
        if (n) atomicAdd(&hist[c], n);
    } else if (e0 >= E) {                                       // the block behind the columns
        int n = 0;
        for (int r = threadIdx.x; r < N; r += 1024) n += !(padded && padded[r]);
        atomicAdd(&hist[0], n);
    } else {
        const int total = N * codes.K, last = min(e0 + BL_COLS, E);
        const auto count = [&](int i, int64_t e) {
            if (e < e0 || e >= last) return;
            if (padded && padded[codes.K == 1 ? i : i / codes.K]) return;
            atomicAdd(&hist[(int)e - e0], 1);
        };
#pragma unroll 4
        for (int i = threadIdx.x * 4; i < total - 3; i += 4096) {
            if (codes.wide) {
                const long *p = reinterpret_cast<const long *>(codes.p) + i;
                const long2u q = *reinterpret_cast<const long2u *>(p), r = *reinterpret_cast<const long2u *>(p + 2);
                count(i, q.x); count(i + 1, q.y); count(i + 2, r.x); count(i + 3, r.y);
            } else {
                const int4u q = *reinterpret_cast<const int4u *>(reinterpret_cast<const int *>(codes.p) + i);
                count(i, q.x); count(i + 1, q.y); count(i + 2, q.z); count(i + 3, q.w);
            }
        }
        if (threadIdx.x < (total & 3)) count((total & ~3) + threadIdx.x, codes.at((total & ~3) + threadIdx.x));
    }
    __syncthreads();
    if (g == 0 && e0 + c < E) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += red[i][c];
        sums[e0 + c] = (float)t;
        sums[E + e0 + c] = (float)hist[c];
        counts[e0 + c] = hist[c];
    }
    if (g == 0 && (pcount ? e0 + c == E : e0 >= E && c == 0)) sums[2 * (int64_t)E] = (float)hist[c];
}

__global__ __launch_bounds__(1024) void balance_final_kernel(const float *__restrict__ sums, int E, int K, float *__restrict__ loss, float *__restrict__ f)
{
    __shared__ double red[16];
    const double nv = sums[2 * (int64_t)E];
    double a = 0.0;
    for (int e = threadIdx.x; e < E; e += 1024) {
        const double fe = nv > 0.0 ? (double)sums[E + e] / (nv * K) : 0.0;
        f[e] = (float)fe;
        a += fe * (double)sums[e];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += red[i];
        loss[0] = nv > 0.0 ? (float)(t * E / nv) : 0.f;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void balance_bwd_kernel(const T *__restrict__ z, int64_t ld, const uint8_t *__restrict__ padded, int E,
                                                          const float2 *__restrict__ stats, const float *__restrict__ f, const float *__restrict__ sums,
                                                          const float *__restrict__ gout, T *__restrict__ dz)
{
    __shared__ float red[4];
    const int64_t n = blockIdx.x;
    T *out = dz + n * E;
    if (padded && padded[n]) {
        for (int e = threadIdx.x; e < E; e += 256) Ld<T>::put(out + e, 0.f);
        return;
    }
    const T *row = z + n * ld;
    const float2 st = stats[n];
    float s = 0.f;
    for (int e = threadIdx.x; e < E; e += 256) s = fmaf(f[e], Offset(st).exp(Ld<T>::get(row + e)) * fabsf(st.y), s);
    s = block_sum<256>(s, red);
    const float scale = gout[0] * ((float)E / sums[2 * (int64_t)E]);
    for (int e = threadIdx.x; e < E; e += 256) {
        const float p = Offset(st).exp(Ld<T>::get(row + e)) * fabsf(st.y);
        Ld<T>::put(out + e, scale * p * (f[e] - s));
    }
}

inline int64_t bl_chunks(int64_t n) { return n < 512 ? n : 512; }

// How a row is held: the smallest team that holds it in at most 4 quads a lane.  wide: the two-pass kernels above
struct BlForm {
    int tl, nq, w;
    bool wide;
};
inline BlForm bl_form(int E, int dtype)
{
    const int epq = dtype == 0 ? 4 : 8, q = (E + epq - 1) / epq;   // quads of a row
    if (q <= 4) return {4, 1, 1, false};
    if (q <= 8) return {8, 1, 1, false};
    if (q <= 16) return {16, 1, 1, false};
    if (q <= 32) return {32, 1, 1, false};
    if (q <= 64) return {64, 1, 1, false};
    if (q <= 128) return {64, 2, 1, false};
    if (q <= 256) return {64, 4, 1, false};
    if (q <= 512) return {64, 2, 4, false};
    if (q <= 1024) return {64, 2, 8, false};
    if (q <= 2048) return {64, 4, 8, false};
    if (q <= 4096 && dtype == 0) return {64, 4, 16, false};          // of two-byte scores it would not fit the registers
    return {0, 0, 0, true};
}
inline int bl_blocks(const BlForm &f, int64_t rows)
{
    const int64_t teams = f.w > 1 ? 1 : 256 / f.tl;
    const int64_t b = cdiv(rows, teams);
    return (int)(b < 512 ? b : 512);
}

}  // namespace mq

using namespace mq;

// partial column sums
extern "C" size_t mq_code_balance_workspace(int64_t rows, int codes, int dtype)
{
    if (rows <= 0 || codes <= 0 || dtype < 0 || dtype > 2) return 0;
    const BlForm f = bl_form(codes, dtype);
    return f.wide ? (size_t)bl_chunks(rows) * codes * 4 : (size_t)bl_blocks(f, rows) * ((size_t)codes * 4 + (f.w > 1 ? 0 : ((size_t)codes + 1) * 4));
}

#define BL_TYPES(call)                                                    \
    switch (dtype) {                                                      \
    case 0: call(float); break;                                           \
    case 1: call(uint16_t); break;                                        \
    default: call(_Float16); break;                                       \
    }
// F(TL, NQ, W): one of the forms of bl_form
#define BL_FORMS(F)                                                       \
    if (f.tl == 4) F(4, 1, 1);                                            \
    else if (f.tl == 8) F(8, 1, 1);                                       \
    else if (f.tl == 16) F(16, 1, 1);                                     \
    else if (f.tl == 32) F(32, 1, 1);                                     \
    else if (f.w == 16) { if constexpr (sizeof(T) == 4) F(64, 4, 16); }   \
    else if (f.w == 8 && f.nq == 4) F(64, 4, 8);                          \
    else if (f.w == 8) F(64, 2, 8);                                       \
    else if (f.w == 4) F(64, 2, 4);                                       \
    else if (f.nq == 1) F(64, 1, 1);                                      \
    else if (f.nq == 2) F(64, 2, 1);                                      \
    else F(64, 4, 1);

template <typename T>
static void bl_forward(const T *z, int64_t ld, const uint8_t *padded, int64_t rows, int codes, float2 *st, float *part, const BlForm &f, int blocks, const Codes &c,
                       int32_t *pcount, hipStream_t s)
{
    const int epq = Wide<T>::EPQ;
    const bool vec = codes % epq == 0 && ld % epq == 0 && (uintptr_t)z % 16 == 0;
#define F(TL, NQ, W)                                                                                                                                  \
    do {                                                                                                                                              \
        const size_t lds = W > 1 ? 0 : ((size_t)codes + 1) * sizeof(float);                                                                                 \
        if (vec) hipLaunchKernelGGL((balance_fwd_kernel<T, TL, NQ, W, true>), dim3(blocks), dim3(W > 1 ? 64 * W : 256), lds, s, z, ld, padded, rows, codes, st, part, c, pcount); \
        else hipLaunchKernelGGL((balance_fwd_kernel<T, TL, NQ, W, false>), dim3(blocks), dim3(W > 1 ? 64 * W : 256), lds, s, z, ld, padded, rows, codes, st, part, c, pcount);    \
    } while (0)
    BL_FORMS(F)
#undef F
}
template <typename T>
static void bl_backward(const T *z, int64_t ld, const uint8_t *padded, int64_t rows, int codes, const float2 *st, const float *fr, const float *sums, const float *gout, T *dz,
                        const BlForm &f, hipStream_t s)
{
    const int epq = Wide<T>::EPQ;
    const bool vec = codes % epq == 0 && ld % epq == 0 && ((uintptr_t)z | (uintptr_t)dz) % 16 == 0;
    const int64_t teams = f.w > 1 ? 1 : 256 / f.tl, want = cdiv(rows, teams), most = f.w > 1 ? 256 * (32 / f.w) : 2048;
    const dim3 grid((unsigned)(want < most ? want : most));
#define F(TL, NQ, W)                                                                                                                                  \
    do {                                                                                                                                              \
        if (vec) hipLaunchKernelGGL((balance_grad_kernel<T, TL, NQ, W, true>), grid, dim3(W > 1 ? 64 * W : 256), 0, s, z, ld, padded, rows, codes, st, fr, sums, gout, dz); \
        else hipLaunchKernelGGL((balance_grad_kernel<T, TL, NQ, W, false>), grid, dim3(W > 1 ? 64 * W : 256), 0, s, z, ld, padded, rows, codes, st, fr, sums, gout, dz);    \
    } while (0)
    BL_FORMS(F)
#undef F
}

extern "C" int mq_code_balance_fwd(const void *logits, int dtype, int64_t row_stride, const void *idx, int idx64, int per_row, const uint8_t *padded,
                                    int64_t rows, int codes, void *stats, int32_t *counts, float *sums, float *loss, float *fractions,
                                    void *workspace, size_t workspace_bytes, mqStream stream)
{
    MQ_REQUIRE(logits && idx && stats && counts && sums && workspace && !loss == !fractions, "mq_code_balance_fwd: NULL argument");
    MQ_REQUIRE(dtype >= 0 && dtype <= 2, "mq_code_balance_fwd: dtype %d (0 f32, 1 bf16, 2 f16)", dtype);
    MQ_REQUIRE(rows > 0 && rows < INT32_MAX && codes > 0 && codes <= (1 << 24) && per_row > 0 && row_stride >= codes,
               "mq_code_balance_fwd: bad sizes (rows %lld, codes %d, per_row %d, row stride %lld)", (long long)rows, codes, per_row, (long long)row_stride);
    MQ_REQUIRE(rows * (int64_t)per_row <= (1 << 30), "mq_code_balance_fwd: more than 2^30 assignments: the counts would near 32 bits");
    MQ_REQUIRE(workspace_bytes >= mq_code_balance_workspace(rows, codes, dtype), "mq_code_balance_fwd: workspace of %zu bytes, %zu needed", workspace_bytes,
               mq_code_balance_workspace(rows, codes, dtype));
    float *part = reinterpret_cast<float *>(workspace);
    float2 *st = reinterpret_cast<float2 *>(stats);
    const BlForm f = bl_form(codes, dtype);
    const Codes c{idx, idx64, per_row};
    int32_t *pcount = nullptr;
    int nparts;
    if (f.wide) {
        const int64_t chunk = cdiv(rows, bl_chunks(rows));
        nparts = (int)cdiv(rows, chunk);
#define CALL(T)                                                                                                                                       \
    hipLaunchKernelGGL(balance_rows_kernel<T>, dim3((unsigned)rows), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, codes, st); \
    hipLaunchKernelGGL(balance_cols_kernel<T>, dim3((unsigned)cdiv(codes, 256), nparts), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, \
                       rows, codes, chunk, st, part)
        BL_TYPES(CALL)
#undef CALL
    } else {
        nparts = bl_blocks(f, rows);
        if (f.w == 1) pcount = reinterpret_cast<int32_t *>(part + (int64_t)nparts * codes);
#define CALL(T) bl_forward(reinterpret_cast<const T *>(logits), row_stride, padded, rows, codes, st, part, f, nparts, c, pcount, S(stream))
        BL_TYPES(CALL)
#undef CALL
    }
    const unsigned grid = pcount ? (unsigned)cdiv(codes + 1, BL_COLS) : (unsigned)cdiv(codes, BL_COLS) + 1;
    hipLaunchKernelGGL(balance_sums_kernel, dim3(grid), dim3(1024), 0, S(stream), part, pcount, nparts, c, padded, (int)rows, codes, counts, sums);
    if (loss) hipLaunchKernelGGL(balance_final_kernel, dim3(1), dim3(1024), 0, S(stream), sums, codes, per_row, loss, fractions);
    MQ_LAUNCH_CHECK("mq_code_balance_fwd");
    return 0;
}

extern "C" int mq_code_balance_final(const float *sums, int codes, int per_row, float *loss, float *fractions, mqStream stream)
{
    MQ_REQUIRE(sums && loss && fractions && codes > 0 && per_row > 0, "mq_code_balance_final: bad arguments");
    hipLaunchKernelGGL(balance_final_kernel, dim3(1), dim3(1024), 0, S(stream), sums, codes, per_row, loss, fractions);
    MQ_LAUNCH_CHECK("mq_code_balance_final");
    return 0;
}

extern "C" int mq_code_balance_bwd(const void *logits, int dtype, int64_t row_stride, const uint8_t *padded, int64_t rows, int codes, const void *stats,
                                   const float *sums, const float *fractions, const float *gout, void *dlogits, mqStream stream)
{
    MQ_REQUIRE(logits && stats && sums && fractions && gout && dlogits, "mq_code_balance_bwd: NULL argument");
    MQ_REQUIRE(dtype >= 0 && dtype <= 2, "mq_code_balance_bwd: dtype %d (0 f32, 1 bf16, 2 f16)", dtype);
    MQ_REQUIRE(rows > 0 && rows < INT32_MAX && codes > 0 && row_stride >= codes, "mq_code_balance_bwd: bad sizes");
    const float2 *st = reinterpret_cast<const float2 *>(stats);
    const BlForm form = bl_form(codes, dtype);
    if (form.wide) {
#define CALL(T)                                                                                                                                       \
    hipLaunchKernelGGL(balance_bwd_kernel<T>, dim3((unsigned)rows), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, codes, st, fractions, \
                       sums, gout, reinterpret_cast<T *>(dlogits))
        BL_TYPES(CALL)
#undef CALL
    } else {
#define CALL(T) bl_backward(reinterpret_cast<const T *>(logits), row_stride, padded, rows, codes, st, fractions, sums, gout, reinterpret_cast<T *>(dlogits), form, S(stream))
        BL_TYPES(CALL)
#undef CALL
    }
    MQ_LAUNCH_CHECK("mq_code_balance_bwd");
    return 0;
}
