// Balance loss of a codebook with per-code counts, and its gradient with respect to the scores.
//
//   p_n = softmax(z_n),  P_e = 1/Nv sum_{valid n} p_ne,  f_e = counts_e / (Nv K)
//   L = E sum_e f_e P_e,     dL/dz_ne = g E / Nv p_ne (f_e - sum_j f_j p_nj)
// E codes, K assignments a row, Nv rows that are not padded.  L is 1 where codes are used evenly and E where one code takes all.  The
// counts are whole numbers and carry no gradient.
//
// A row's statistics are its maximum m and 1 / sum exp(z - m), never their logarithm's sum: a row of nothing but the type's lowest value
// has log(sum) far under half an ulp of m.  A row of -inf alone has p = 0.  Padded rows are not read; their gradient is 0.
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

__device__ __forceinline__ float2 stats_of(float m, float s)            // (subtrahend, factor) of a row
{
    return m == -INFINITY ? make_float2(0.f, s) : make_float2(m, 1.0f / s);      // s is 0 here, or a NaN
}
// block of 256: (m, s) pairs joined; red is 8 floats
__device__ __forceinline__ float2 block_join(float m, float s, float *red)
{
    const float wm = wave_max(m);
    const float ws = wave_sum(s == 0.f ? 0.f : s * __expf(m - wm));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = wm;
        red[4 + (threadIdx.x >> 6)] = ws;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float S = 0.f;
    for (int i = 0; i < 4; ++i) S += red[4 + i] == 0.f ? 0.f : red[4 + i] * __expf(red[i] - M);
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
        s = (s == 0.f ? 0.f : s * __expf(m - nm)) + (x == -INFINITY ? 0.f : __expf(x - nm));
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
        a = fmaf(__expf(Ld<T>::get(z + n * ld + e) - st.x), st.y, a);
    }
    part[(int64_t)blockIdx.y * E + e] = a;
}

__global__ __launch_bounds__(256) void balance_zero_kernel(int *__restrict__ counts, int n)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) counts[i] = 0;
}
// counts[0 .. E) and counts[E] = valid rows.  Whole numbers: the order of the additions does not show.
template <typename I>
__global__ __launch_bounds__(256) void balance_counts_kernel(const I *__restrict__ idx, const uint8_t *__restrict__ padded, int64_t N, int K, int E,
                                                             int in_lds, int *__restrict__ counts)
{
    extern __shared__ int hist[];
    if (in_lds) {
        for (int e = threadIdx.x; e <= E; e += 256) hist[e] = 0;
        __syncthreads();
    }
    int *to = in_lds ? hist : counts;
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < N; n += (int64_t)gridDim.x * 256) {
        if (padded && padded[n]) continue;
        atomicAdd(to + E, 1);
        for (int k = 0; k < K; ++k) {
            const int64_t e = (int64_t)idx[n * K + k];
            if (e >= 0 && e < E) atomicAdd(to + e, 1);
        }
    }
    if (in_lds) {
        __syncthreads();
        for (int e = threadIdx.x; e <= E; e += 256)
            if (hist[e]) atomicAdd(counts + e, hist[e]);
    }
}

// sums = {sum_n p_ne (E), counts (E), valid rows}: what data-parallel ranks add up before the loss is formed
__global__ __launch_bounds__(256) void balance_sums_kernel(const float *__restrict__ part, int nparts, const int *__restrict__ counts, int E,
                                                           float *__restrict__ sums)
{
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e > E) return;
    if (e == E) {
        sums[2 * (int64_t)E] = (float)counts[E];
        return;
    }
    double a = 0.0;
    for (int i = 0; i < nparts; ++i) a += (double)part[(int64_t)i * E + e];
    sums[e] = (float)a;
    sums[E + e] = (float)counts[e];
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
    for (int e = threadIdx.x; e < E; e += 256) s = fmaf(f[e], __expf(Ld<T>::get(row + e) - st.x) * st.y, s);
    s = block_sum<256>(s, red);
    const float scale = gout[0] * ((float)E / sums[2 * (int64_t)E]);
    for (int e = threadIdx.x; e < E; e += 256) {
        const float p = __expf(Ld<T>::get(row + e) - st.x) * st.y;
        Ld<T>::put(out + e, scale * p * (f[e] - s));
    }
}

inline int64_t bl_chunks(int64_t n) { return n < 512 ? n : 512; }

}  // namespace mq

using namespace mq;

// statistics of the rows, then partial column sums
extern "C" size_t mq_code_balance_workspace(int64_t rows, int codes)
{
    if (rows <= 0 || codes <= 0) return 0;
    return (size_t)bl_chunks(rows) * codes * sizeof(float);
}

#define BL_TYPES(call)                                                    \
    switch (dtype) {                                                      \
    case 0: call(float); break;                                           \
    case 1: call(uint16_t); break;                                        \
    default: call(_Float16); break;                                       \
    }

extern "C" int mq_code_balance_sums(const void *logits, int dtype, int64_t row_stride, const void *idx, int idx64, int per_row, const uint8_t *padded,
                                    int64_t rows, int codes, void *stats, int32_t *counts, float *sums, void *workspace, size_t workspace_bytes,
                                    mqStream stream)
{
    MQ_REQUIRE(logits && idx && stats && counts && sums && workspace, "mq_code_balance_sums: NULL argument");
    MQ_REQUIRE(dtype >= 0 && dtype <= 2, "mq_code_balance_sums: dtype %d (0 f32, 1 bf16, 2 f16)", dtype);
    MQ_REQUIRE(rows > 0 && rows < INT32_MAX && codes > 0 && codes <= (1 << 24) && per_row > 0 && row_stride >= codes,
               "mq_code_balance_sums: bad sizes (rows %lld, codes %d, per_row %d, row stride %lld)", (long long)rows, codes, per_row, (long long)row_stride);
    MQ_REQUIRE(rows * (int64_t)per_row < INT32_MAX, "mq_code_balance_sums: the counts would pass 32 bits");
    MQ_REQUIRE(workspace_bytes >= mq_code_balance_workspace(rows, codes), "mq_code_balance_sums: workspace of %zu bytes, %zu needed", workspace_bytes,
               mq_code_balance_workspace(rows, codes));
    float *part = reinterpret_cast<float *>(workspace);
    float2 *st = reinterpret_cast<float2 *>(stats);
    const int64_t chunk = cdiv(rows, bl_chunks(rows));
    const int nparts = (int)cdiv(rows, chunk);
#define CALL(T)                                                                                                                                       \
    hipLaunchKernelGGL(balance_rows_kernel<T>, dim3((unsigned)rows), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, codes, st); \
    hipLaunchKernelGGL(balance_cols_kernel<T>, dim3((unsigned)cdiv(codes, 256), nparts), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, \
                       rows, codes, chunk, st, part)
    BL_TYPES(CALL)
#undef CALL
    hipLaunchKernelGGL(balance_zero_kernel, dim3((unsigned)cdiv(codes + 1, 256)), dim3(256), 0, S(stream), counts, codes + 1);
    const int in_lds = codes < 16384;                               // 64 KiB of the 160 a compute unit has
    const unsigned nb = (unsigned)(cdiv(rows, 256) < 256 ? cdiv(rows, 256) : 256);
    const size_t lds = in_lds ? (size_t)(codes + 1) * sizeof(int) : 0;
    if (idx64)
        hipLaunchKernelGGL(balance_counts_kernel<int64_t>, dim3(nb), dim3(256), lds, S(stream), reinterpret_cast<const int64_t *>(idx), padded, rows, per_row, codes, in_lds, counts);
    else
        hipLaunchKernelGGL(balance_counts_kernel<int32_t>, dim3(nb), dim3(256), lds, S(stream), reinterpret_cast<const int32_t *>(idx), padded, rows, per_row, codes, in_lds, counts);
    hipLaunchKernelGGL(balance_sums_kernel, dim3((unsigned)cdiv(codes + 1, 256)), dim3(256), 0, S(stream), part, nparts, counts, codes, sums);
    MQ_LAUNCH_CHECK("mq_code_balance_sums");
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
#define CALL(T)                                                                                                                                       \
    hipLaunchKernelGGL(balance_bwd_kernel<T>, dim3((unsigned)rows), dim3(256), 0, S(stream), reinterpret_cast<const T *>(logits), row_stride, padded, codes, st, fractions, \
                       sums, gout, reinterpret_cast<T *>(dlogits))
    BL_TYPES(CALL)
#undef CALL
    MQ_LAUNCH_CHECK("mq_code_balance_bwd");
    return 0;
}
