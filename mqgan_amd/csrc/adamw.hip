// One AdamW step over many tensors (decoupled weight decay, gradient-norm clipping), moments in f32 or in 8 bits.
//
//   g' = coef g,  coef = grad_scale min(1, max_norm / (|grad_scale| |g|_2 + 1e-6))     |g|_2 over every tensor of the call
//   m += (g' - m)(1 - b1);  v = v b2 + (1 - b2) g' g'
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)          t: steps THIS tensor has taken
//
// 8-bit moments.  256 consecutive elements of a tensor (a group, what one wave holds as four per lane) share one byte `base`; a code is
// the top bits of the f32 magnitude, counted from the base's binade:
//     m: sign, 7 bits c;  v: 8 bits c;      |x| = bitcast((c + 8 base) << 20) for c > 0, and 0 for c = 0
// i.e. 3 mantissa bits and 4 (m) or 5 (v) exponent bits under the group's largest magnitude, whose binade + 1 is the topmost, so that
// rounding up has a code.  Decoding is a shift and an add, encoding an add and a shift; no table, no division, and the decoded value
// is exact in bf16.  The two last codes are infinity and NaN, which stay with their element.  A positive v never becomes 0 (code 1 at
// least): m / (0 + eps) would be a step of its own kind.  Rounding is STOCHASTIC: 16 random bits are added under the kept ones before
// the rest is cut off.  To nearest, a second moment with b2 = 0.999 would not move at all - its change per step, 0.1 % of
// (g'^2 - v), is far under half a step of a 3-bit mantissa (3-6 %); rounded at random it moves by the right amount on average.  The
// bits are a hash of (seed, call, position in the moments' layout): the same on every replay of a run.
//
// All of it is bound by memory.  f32 moments: 28 bytes an element with f32 gradients, plus 4 for the norm, whose pass
// leaves part of the gradients in the 256 MB cache.  34 M elements in 260 tensors: update 142 us (6.7 TB/s), norm 27, factors 5, where
// the same passes as tensor operations take 1510.  8 bits: 16.02 bytes, 87 us (6.3 TB/s) + norm 33; 150 M elements with bf16 gradients 353-371 us
// (14.02 bytes, 5.8 TB/s) + norm 70-94.  Chunks of 4096 elements as straight-line code with all loads issued first took the f32 update from 170 to 142;
// codes by shifts in place of compares and the hardware's root and reciprocal took an 8-bit step of 34 M with its moments decoded from 202 to 168.
#include "common.h"

namespace mq {

constexpr int AW_CHUNK = 4096;        // elements a block updates: four groups a wave
constexpr int AW_NORM = 4;            // chunks a block of the norm reads
constexpr int64_t AW_MOST = 1 << 24;  // blocks of 256 threads a launch: under 2^32 threads
constexpr int AW_GRADS = 460;         // gradient addresses a launch carries by value (kernel arguments hold 4 KiB)

struct AwRow {                        // one tensor; the layout of the table is private to this file
    float *p;
    void *m, *v;
    uint8_t *mb, *vb;
    int64_t n, position;
    int first_block;
    float wd, lr_scale;
    int pad;
};
struct AwControl {                    // start of the control buffer; AwState per tensor follows at byte 64
    double sumsq;
    int64_t calls;
    float coef;
    uint32_t k0, k1;
    uint32_t pad0;
    double norm_scale;                // |grad_scale| of the call that sumsq is of
    uint32_t pad[6];
};
struct AwState {
    int step;
    float step_size, inv_bc2, keep;   // lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd (1 where nothing decays)
};
struct AwGrads {
    uint64_t g[AW_GRADS];             // address | element type << 62; 0: no gradient
};
struct AwHyper {
    double lr, beta1, beta2, grad_scale, max_norm;
    float omb1, b2, omb2, eps;
    uint64_t seed;
};
static_assert(sizeof(AwRow) == 72 && sizeof(AwControl) == 64 && sizeof(AwState) == 16, "table layout");

typedef float aw_f4 __attribute__((ext_vector_type(4)));
typedef unsigned short aw_u4 __attribute__((ext_vector_type(4)));
// Non-temporal accesses for what a step touches once: plain loads of a large buffer ran at 6.3 TB/s on this card, these at 7.1.
__device__ __forceinline__ float4 nt_load4(const float *p)
{
    const aw_f4 q = __builtin_nontemporal_load(reinterpret_cast<const aw_f4 *>(p));
    return make_float4(q.x, q.y, q.z, q.w);
}
__device__ __forceinline__ void nt_store4(float *p, const float4 &v) { __builtin_nontemporal_store((aw_f4){v.x, v.y, v.z, v.w}, reinterpret_cast<aw_f4 *>(p)); }

__device__ __forceinline__ float aw_half(uint16_t b, int type)
{
    return type == 1 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}
// Four elements from e, one at a time; elements at and after n read as 0.
__device__ __forceinline__ float4 aw_slow4(const float *p, int64_t e, int64_t n)
{
    return make_float4(e < n ? p[e] : 0.f, e + 1 < n ? p[e + 1] : 0.f, e + 2 < n ? p[e + 2] : 0.f, e + 3 < n ? p[e + 3] : 0.f);
}
__device__ __forceinline__ float4 aw_slow4(const uint16_t *p, int64_t e, int64_t n, int type)
{
    return make_float4(e < n ? aw_half(p[e], type) : 0.f, e + 1 < n ? aw_half(p[e + 1], type) : 0.f, e + 2 < n ? aw_half(p[e + 2], type) : 0.f,
                       e + 3 < n ? aw_half(p[e + 3], type) : 0.f);
}
// A thread's sixteen gradients of a chunk (four from each of e, e + 1024, ..): type 0 f32, 1 bf16, 2 f16.  `whole`: the chunk lies inside the
// tensor and its address is aligned to four elements.  Type and whole are uniform over the block, so each way is straight-line code with
// all its loads in flight; deciding per load cost the norm half of its rate.
template <bool NT>
__device__ __forceinline__ void aw_grads(uint64_t tagged, int64_t e, int64_t n, bool whole, float4 (&g)[4])
{
    const int type = (int)(tagged >> 62);
    const uint64_t a = tagged & 0x3fffffffffffffffull;
    if (type == 0) {
        const float *p = reinterpret_cast<const float *>(a);
        if (whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k) g[k] = NT ? nt_load4(p + e + k * 1024) : *reinterpret_cast<const float4 *>(p + e + k * 1024);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) g[k] = aw_slow4(p, e + k * 1024, n);
        }
    } else {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(a);
        if (whole) {
            aw_u4 q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = NT ? __builtin_nontemporal_load(reinterpret_cast<const aw_u4 *>(p + e + k * 1024)) : *reinterpret_cast<const aw_u4 *>(p + e + k * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k) g[k] = make_float4(aw_half(q[k].x, type), aw_half(q[k].y, type), aw_half(q[k].z, type), aw_half(q[k].w, type));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) g[k] = aw_slow4(p, e + k * 1024, n, type);
        }
    }
}
// whether a chunk that starts at e is inside n and the gradient can be read four at a time
__device__ __forceinline__ bool aw_whole(uint64_t tagged, int64_t chunk, int64_t n)
{
    return chunk + AW_CHUNK <= n && (tagged & (tagged >> 62 ? 7 : 15)) == 0;
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Squares in f64: a gradient of 1e20 has a norm, and the sum's order (lane, wave, block) costs nothing in f32 terms.  A block takes
// AW_NORM of the update's chunks, whose rows it looks up together: with one chunk a block the look-ups' latency was half of the time.
__global__ __launch_bounds__(256) void adamw_sumsq_kernel(const AwGrads grads, const AwRow *__restrict__ rows, const int *__restrict__ row_of,
                                                          int row0, int block0, int nb, int part0, double *__restrict__ part)
{
    __shared__ double red[4];
    const int b0 = blockIdx.x * AW_NORM;
    int r[AW_NORM];
    uint64_t tagged[AW_NORM];
    int64_t n[AW_NORM], at[AW_NORM];
#pragma unroll
    for (int c = 0; c < AW_NORM; ++c) r[c] = row_of[block0 + (b0 + c < nb ? b0 + c : nb - 1)];
#pragma unroll
    for (int c = 0; c < AW_NORM; ++c) {
        tagged[c] = grads.g[r[c] - row0];
        n[c] = b0 + c < nb && tagged[c] ? rows[r[c]].n : 0;        // 0: nothing is read
        at[c] = (int64_t)(block0 + b0 + c - rows[r[c]].first_block) * AW_CHUNK;
    }
    double s = 0.0, u = 0.0;
#pragma unroll
    for (int c = 0; c < AW_NORM; ++c) {
        const int type = (int)(tagged[c] >> 62);
        const uint64_t a = tagged[c] & 0x3fffffffffffffffull;
        const auto add = [&](float x, float y) {
            s = fma((double)x, (double)x, s);
            u = fma((double)y, (double)y, u);
        };
        if (type && (a & 15) == 0 && at[c] + AW_CHUNK <= n[c]) {    // two-byte elements, eight to a load
            uint4 q[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) q[k] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(a) + at[c] + k * 2048 + threadIdx.x * 8);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) add(aw_half((uint16_t)w[i], type), aw_half((uint16_t)(w[i] >> 16), type));
            }
        } else {
            float4 g[4];
            aw_grads<false>(tagged[c], at[c] + threadIdx.x * 4, n[c], aw_whole(tagged[c], at[c], n[c]), g);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                add(g[k].x, g[k].y);
                add(g[k].z, g[k].w);
            }
        }
    }
    s = wave_sum_f64(s + u);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[part0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// One block: the norm from the partial sums (first launch of a call), then every tensor's step count and the factors that go with it.
// On the device because a captured step is replayed: count, bias corrections and random bits have to move on without the host.
__global__ __launch_bounds__(1024) void adamw_prepare_kernel(const AwGrads grads, const AwRow *__restrict__ rows, int row0, int nrows, int first,
                                                             const double *__restrict__ part, int nparts, const AwHyper h,
                                                             const float *__restrict__ present, AwControl *__restrict__ ctl, AwState *__restrict__ st)
{
    __shared__ double red[16];
    if (first) {
        double s = 0.0;
        for (int i = threadIdx.x; i < nparts; i += 1024) s += part[i];
        s = wave_sum_f64(s);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int i = 0; i < 16; ++i) t += red[i];
            double coef = h.grad_scale;
            if (h.max_norm > 0.0) {
                const double c = h.max_norm / (sqrt(t) * fabs(h.grad_scale) + 1e-6);
                coef = c < 1.0 ? c * h.grad_scale : (c >= 1.0 ? h.grad_scale : c);    // a NaN norm makes the step NaN, as the formula says
                ctl->sumsq = t;
                ctl->norm_scale = fabs(h.grad_scale);
            }
            ctl->coef = (float)coef;
            const int64_t calls = ctl->calls + 1;
            ctl->calls = calls;
            const SeedKeys k = seed_keys(h.seed + (uint64_t)calls * 0xD1B54A32D192ED03ull);
            ctl->k0 = k.k0;
            ctl->k1 = k.k1;
        }
    }
    for (int i = threadIdx.x; i < nrows; i += 1024) {
        if (!grads.g[i] || (present && !(present[row0 + i] > 0.f))) continue;
        const int t = st[row0 + i].step + 1;
        const double lr = h.lr * (double)rows[row0 + i].lr_scale;
        AwState s;
        s.step = t;
        s.step_size = (float)(lr / (1.0 - pow(h.beta1, (double)t)));
        s.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(h.beta2, (double)t)));
        s.keep = (float)(1.0 - lr * (double)rows[row0 + i].wd);
        st[row0 + i] = s;
    }
}

// ----------------------------------------------------------------------------- 8-bit moments
typedef unsigned short aw_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b)
{
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(aw_u16x2, a), __builtin_bit_cast(aw_u16x2, b)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// both 16-bit halves: their maxima over the wave, in every lane
__device__ __forceinline__ uint32_t wave_pk_max(uint32_t v)
{
    v = pk_max(v, dpp_u32<0xB1>(v));
    v = pk_max(v, dpp_u32<0x4E>(v));
    v = pk_max(v, dpp_u32<0x141>(v));
    v = pk_max(v, dpp_u32<0x140>(v));
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return pk_max(pk_max(a, b), pk_max(c, d));
}
__device__ __forceinline__ uint32_t mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// base from the group's largest exponent: the binade above it is the topmost of 2^EB
template <int EB>
__device__ __forceinline__ uint32_t base_of(uint32_t e)
{
    const int b = (int)e + 1 - ((1 << EB) - 1);
    return b > 0 ? (uint32_t)b : 0u;
}
// code of one element; add: what goes under the kept bits (16 random bits << 4, or the round-to-nearest-even term)
template <int EB>
__device__ __forceinline__ uint32_t code8(float x, uint32_t base, uint32_t add)
{
    const uint32_t b = mag(x);
    const int c = (int)(b - (base << 23) + add) >> 20;             // code 1 starts at (8 base + 1) << 20
    const uint32_t u = (uint32_t)max(c, EB == 5 ? (int)min(b, 1u) : 0);
    if (EB == 4) return u | (u ? (__float_as_uint(x) >> 24) & 0x80u : 0u);
    return u;
}
template <int EB>
__device__ __forceinline__ uint32_t special8(float x)               // of infinity and NaN
{
    constexpr uint32_t most = 1u << (EB + 3);
    const uint32_t c = mag(x) == 0x7f800000u ? most - 2 : most - 1;
    return EB == 4 ? c | ((__float_as_uint(x) >> 24) & 0x80u) : c;
}
// Four elements to a word of codes; `top`: the largest exponent of the group, 255 where something in it is infinite or NaN.  Then the base is
// that of the finite ones and the others get their special codes: a branch the whole wave takes or leaves.
template <int EB, typename ADD>
__device__ __forceinline__ uint32_t word8(const float4 &x, uint32_t base, bool specials, ADD add)
{
    uint32_t c[4] = {code8<EB>(x.x, base, add(x.x, 0)), code8<EB>(x.y, base, add(x.y, 1)), code8<EB>(x.z, base, add(x.z, 2)), code8<EB>(x.w, base, add(x.w, 3))};
    if (specials) {
        if (mag(x.x) >= 0x7f800000u) c[0] = special8<EB>(x.x);
        if (mag(x.y) >= 0x7f800000u) c[1] = special8<EB>(x.y);
        if (mag(x.z) >= 0x7f800000u) c[2] = special8<EB>(x.z);
        if (mag(x.w) >= 0x7f800000u) c[3] = special8<EB>(x.w);
    }
    return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
}
__device__ __forceinline__ uint32_t exponent_max(const float4 &x) { return max(max(mag(x.x), mag(x.y)), max(mag(x.z), mag(x.w))) >> 23; }
__device__ __forceinline__ uint32_t finite_mag(float x)
{
    const uint32_t b = mag(x);
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ uint32_t exponent_max_finite(const float4 &x)
{
    return max(max(finite_mag(x.x), finite_mag(x.y)), max(finite_mag(x.z), finite_mag(x.w))) >> 23;
}
// the group's two exponents (m in the low half); specials: whether anything in it is infinite or NaN
__device__ __forceinline__ uint32_t group_top(const float4 &m, const float4 &v, bool &specials)
{
    uint32_t top = wave_pk_max(exponent_max(m) | exponent_max(v) << 16);
    specials = (top & 0xffffu) == 255u || top >> 16 == 255u;
    if (specials) top = wave_pk_max(exponent_max_finite(m) | exponent_max_finite(v) << 16);
    return top;
}
template <int EB>
__device__ __forceinline__ float decode8(uint32_t u, uint32_t base)
{
    constexpr uint32_t most = 1u << (EB + 3);
    const uint32_t c = u & (most - 1);
    uint32_t b = c ? (c + 8 * base) << 20 : 0u;
    if (EB == 4) b |= (u & 0x80u) << 24;
    return __uint_as_float(b);
}
template <int EB>
__device__ __forceinline__ float decode8_special(uint32_t u, uint32_t base)
{
    constexpr uint32_t most = 1u << (EB + 3);
    const uint32_t c = u & (most - 1);
    if (c < most - 2) return decode8<EB>(u, base);
    return __uint_as_float((c == most - 2 ? 0x7f800000u : 0x7fc00000u) | (EB == 4 ? (u & 0x80u) << 24 : 0u));
}
// whether one of the word's four codes is a special one (its bits 1 .. all set): a byte of t is 0 where it is
template <int EB>
__device__ __forceinline__ bool any_special(uint32_t w)
{
    const uint32_t t = ~w & (EB == 4 ? 0x7e7e7e7eu : 0xfefefefeu);
    return ((t - 0x01010101u) & ~t & 0x80808080u) != 0u;
}
template <int EB>
__device__ __forceinline__ float4 unword8(uint32_t w, uint32_t base, bool specials)
{
    if (specials)
        return make_float4(decode8_special<EB>(w & 255, base), decode8_special<EB>((w >> 8) & 255, base), decode8_special<EB>((w >> 16) & 255, base), decode8_special<EB>(w >> 24, base));
    return make_float4(decode8<EB>(w & 255, base), decode8<EB>((w >> 8) & 255, base), decode8<EB>((w >> 16) & 255, base), decode8<EB>(w >> 24, base));
}
__device__ __forceinline__ uint32_t nearest_add(float x) { return 0x7ffffu + ((mag(x) >> 20) & 1u); }

// Blocks run from the last chunk to the first: the norm has just read the gradients in order, so the last of them are still in the
// 256 MB cache.  Root and reciprocal are the hardware's (one ulp each); v is held up to the smallest normal number under the root,
// which the hardware needs, so with eps = 0 an element that never had a gradient stays put instead of becoming 0 / 0.
template <bool Q8>
__global__ __launch_bounds__(256) void adamw_kernel(const AwGrads grads, const AwRow *__restrict__ rows, const int *__restrict__ row_of, int row0,
                                                    int block0, const AwHyper h, const float *__restrict__ present, const AwControl *__restrict__ ctl,
                                                    const AwState *__restrict__ st)
{
#pragma clang fp contract(off)
    const int block = block0 + (int)(gridDim.x - 1 - blockIdx.x);
    const int r = row_of[block];
    const uint64_t tagged = grads.g[r - row0];
    if (!tagged || (present && !(present[r] > 0.f))) return;        // no gradient this step: the tensor stays as it is
    const AwRow row = rows[r];
    const AwState s = st[r];
    const float coef = ctl->coef;
    const uint32_t k0 = ctl->k0, k1 = ctl->k1;
    const int64_t n = row.n;
    const int64_t room = (n + 255) & ~(int64_t)255;                 // the moments' layout is padded to whole groups
    const int64_t chunk = (int64_t)(block - row.first_block) * AW_CHUNK, e0 = chunk + threadIdx.x * 4;
    const bool whole = chunk + AW_CHUNK <= n && ((uintptr_t)row.p & 15) == 0;
    const float *m32 = reinterpret_cast<const float *>(row.m), *v32 = reinterpret_cast<const float *>(row.v);
    const uint32_t *m8 = reinterpret_cast<const uint32_t *>(row.m), *v8 = reinterpret_cast<const uint32_t *>(row.v);
    float4 p[4], g[4], m[4], v[4];
    uint32_t mc[4], vc[4], mb[4], vb[4];
    aw_grads<true>(tagged, e0, n, aw_whole(tagged, chunk, n), g);
    if (whole) {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = nt_load4(row.p + e0 + k * 1024);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = aw_slow4(row.p, e0 + k * 1024, n);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t e = e0 + k * 1024;
        if (e >= room) continue;                                    // whole waves: a wave's 256 elements are one group
        if (Q8) {
            mc[k] = __builtin_nontemporal_load(m8 + (e >> 2));
            vc[k] = __builtin_nontemporal_load(v8 + (e >> 2));
            mb[k] = row.mb[e >> 8];
            vb[k] = row.vb[e >> 8];
        } else {
            m[k] = nt_load4(m32 + e);
            v[k] = nt_load4(v32 + e);
        }
    }
    const auto one = [&](float &pi, float gi, float &mi, float &vi) {
        gi *= coef;
        mi = mi + (gi - mi) * h.omb1;
        vi = vi * h.b2 + h.omb2 * gi * gi;
        const float denom = __builtin_amdgcn_sqrtf(vi < 1.17549435e-38f ? 1.17549435e-38f : vi) * s.inv_bc2 + h.eps;      // a NaN stays
        pi = pi * s.keep - s.step_size * (mi * __builtin_amdgcn_rcpf(denom));
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t e = e0 + k * 1024;
        if (e >= room) continue;
        if (Q8) {
            const bool held = __builtin_amdgcn_ballot_w64(any_special<4>(mc[k]) || any_special<5>(vc[k])) != 0;
            m[k] = unword8<4>(mc[k], mb[k], held);
            v[k] = unword8<5>(vc[k], vb[k], held);
        }
        one(p[k].x, g[k].x, m[k].x, v[k].x);
        one(p[k].y, g[k].y, m[k].y, v[k].y);
        one(p[k].z, g[k].z, m[k].z, v[k].z);
        one(p[k].w, g[k].w, m[k].w, v[k].w);
        if (whole) {
            nt_store4(row.p + e, p[k]);
        } else {
            if (e < n) row.p[e] = p[k].x;
            if (e + 1 < n) row.p[e + 1] = p[k].y;
            if (e + 2 < n) row.p[e + 2] = p[k].z;
            if (e + 3 < n) row.p[e + 3] = p[k].w;
        }
        if (Q8) {
            bool specials;
            const uint32_t top = group_top(m[k], v[k], specials);
            const uint32_t mbase = base_of<4>(top & 0xffffu), vbase = base_of<5>(top >> 16);
            const uint64_t at = (uint64_t)(row.position + e);
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = mix32((((uint32_t)at + j) ^ k0) + (uint32_t)(at >> 32) * 0x9E3779B1u) + k1;
            __builtin_nontemporal_store(word8<4>(m[k], mbase, specials, [&](float, int j) { return (w[j] >> 16) << 4; }), reinterpret_cast<uint32_t *>(row.m) + (e >> 2));
            __builtin_nontemporal_store(word8<5>(v[k], vbase, specials, [&](float, int j) { return (w[j] & 0xffffu) << 4; }), reinterpret_cast<uint32_t *>(row.v) + (e >> 2));
            if ((threadIdx.x & 63) == 0) {
                row.mb[e >> 8] = (uint8_t)mbase;
                row.vb[e >> 8] = (uint8_t)vbase;
            }
        } else {
            nt_store4(reinterpret_cast<float *>(row.m) + e, m[k]);
            nt_store4(reinterpret_cast<float *>(row.v) + e, v[k]);
        }
    }
}

// f32 moments -> codes, to nearest (loading a state); a wave a group
__global__ __launch_bounds__(256) void moments8_encode_kernel(const float *__restrict__ m, const float *__restrict__ v, int64_t groups,
                                                              uint32_t *__restrict__ mc, uint8_t *__restrict__ mb,
                                                              uint32_t *__restrict__ vc, uint8_t *__restrict__ vb)
{
    const int64_t grp = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (grp >= groups) return;
    const int64_t at = grp * 64 + (threadIdx.x & 63);
    const float4 a = reinterpret_cast<const float4 *>(m)[at], b = reinterpret_cast<const float4 *>(v)[at];
    bool specials;
    const uint32_t top = group_top(a, b, specials);
    const uint32_t bm = base_of<4>(top & 0xffffu), bv = base_of<5>(top >> 16);
    mc[at] = word8<4>(a, bm, specials, [](float x, int) { return nearest_add(x); });
    vc[at] = word8<5>(b, bv, specials, [](float x, int) { return nearest_add(x); });
    if ((threadIdx.x & 63) == 0) {
        mb[grp] = (uint8_t)bm;
        vb[grp] = (uint8_t)bv;
    }
}

// codes -> f32 or bf16 (exact in both); eight elements of both moments a thread
template <bool BF16>
__global__ __launch_bounds__(256) void moments8_decode_kernel(const uint2 *__restrict__ mc, const uint8_t *__restrict__ mb,
                                                              const uint2 *__restrict__ vc, const uint8_t *__restrict__ vb, int64_t n8,
                                                              void *__restrict__ m, void *__restrict__ v)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const uint2 a = mc[i], b = vc[i];
    const uint32_t bm = mb[i >> 5], bv = vb[i >> 5];
    const bool held = __builtin_amdgcn_ballot_w64(any_special<4>(a.x) || any_special<4>(a.y) || any_special<5>(b.x) || any_special<5>(b.y)) != 0;
    const float4 x0 = unword8<4>(a.x, bm, held), x1 = unword8<4>(a.y, bm, held), y0 = unword8<5>(b.x, bv, held), y1 = unword8<5>(b.y, bv, held);
    if (BF16) {
        const auto two = [](float lo, float hi) { return (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xffff0000u); };
        reinterpret_cast<uint4 *>(m)[i] = make_uint4(two(x0.x, x0.y), two(x0.z, x0.w), two(x1.x, x1.y), two(x1.z, x1.w));
        reinterpret_cast<uint4 *>(v)[i] = make_uint4(two(y0.x, y0.y), two(y0.z, y0.w), two(y1.x, y1.y), two(y1.z, y1.w));
    } else {
        reinterpret_cast<float4 *>(m)[2 * i] = x0;
        reinterpret_cast<float4 *>(m)[2 * i + 1] = x1;
        reinterpret_cast<float4 *>(v)[2 * i] = y0;
        reinterpret_cast<float4 *>(v)[2 * i + 1] = y1;
    }
}

inline int64_t aw_blocks(int64_t n) { return cdiv(n, AW_CHUNK); }
inline size_t aw_rows_bytes(int n) { return ((size_t)n * sizeof(AwRow) + 63) / 64 * 64; }

}  // namespace mq

using namespace mq;

extern "C" size_t mq_adamw_table_bytes(const int64_t *numel_host, int n)
{
    if (!numel_host || n <= 0) return 0;
    int64_t blocks = 0;
    for (int i = 0; i < n; ++i) {
        if (numel_host[i] < 0 || numel_host[i] > (1ll << 50)) return 0;
        blocks += aw_blocks(numel_host[i]);
    }
    if (blocks >= AW_MOST) return 0;
    return aw_rows_bytes(n) + (size_t)blocks * sizeof(int);
}

extern "C" size_t mq_adamw_control_bytes(int n) { return n > 0 ? sizeof(AwControl) + (size_t)n * sizeof(AwState) : 0; }

extern "C" size_t mq_adamw_workspace(const int64_t *numel_host, int n)
{
    const size_t t = mq_adamw_table_bytes(numel_host, n);
    return t ? (t - aw_rows_bytes(n)) / sizeof(int) * sizeof(double) + 16 : 0;
}

extern "C" int mq_adamw_table_fill(const mqAdamwTensor *tensors_host, int n, int state_bits, void *table_host, size_t table_bytes)
{
    MQ_REQUIRE(tensors_host && table_host && n > 0, "mq_adamw_table_fill: bad arguments");
    MQ_REQUIRE(state_bits == 32 || state_bits == 8, "mq_adamw_table_fill: moments are held in 32 or 8 bits, not %d", state_bits);
    int64_t blocks = 0;
    for (int i = 0; i < n; ++i) {
        const mqAdamwTensor &t = tensors_host[i];
        MQ_REQUIRE(t.n >= 0 && t.n <= (1ll << 50) && t.position >= 0 && t.position % 256 == 0, "mq_adamw_table_fill: tensor %d: a negative size or a position off the groups of 256", i);
        MQ_REQUIRE(t.n == 0 || (t.param && t.exp_avg && t.exp_avg_sq), "mq_adamw_table_fill: tensor %d has a NULL address", i);
        MQ_REQUIRE((uintptr_t)t.param % 4 == 0 && (uintptr_t)t.exp_avg % 16 == 0 && (uintptr_t)t.exp_avg_sq % 16 == 0,
                   "mq_adamw_table_fill: tensor %d: parameters start at a multiple of 4 bytes, moments of 16", i);
        MQ_REQUIRE(t.n == 0 || state_bits == 32 || (t.base_avg && t.base_avg_sq), "mq_adamw_table_fill: tensor %d: 8-bit moments need their bases", i);
        blocks += aw_blocks(t.n);
        MQ_REQUIRE(blocks < AW_MOST, "mq_adamw_table_fill: too many elements");
    }
    MQ_REQUIRE(table_bytes == aw_rows_bytes(n) + (size_t)blocks * sizeof(int), "mq_adamw_table_fill: the table has %zu bytes, not %zu",
               aw_rows_bytes(n) + (size_t)blocks * sizeof(int), table_bytes);
    AwRow *rows = reinterpret_cast<AwRow *>(table_host);
    int *row_of = reinterpret_cast<int *>(reinterpret_cast<char *>(table_host) + aw_rows_bytes(n));
    int b = 0;
    for (int i = 0; i < n; ++i) {
        const mqAdamwTensor &t = tensors_host[i];
        rows[i] = AwRow{t.param, t.exp_avg, t.exp_avg_sq, t.base_avg, t.base_avg_sq, t.n, t.position, b, t.weight_decay, t.lr_scale, 0};
        for (const int end = b + (int)aw_blocks(t.n); b < end; ++b) row_of[b] = i;
    }
    return 0;
}

static int adamw_step(const mqAdamwDesc *d, const int64_t *numel_host, const void *table, const void *const *grads_host, const uint8_t *grad_types_host,
                      const float *present, void *control, void *workspace, size_t workspace_bytes, mqStream stream)
{
    MQ_REQUIRE(d && numel_host && table && grads_host && control, "mq_adamw_step: bad arguments");
    const int n = d->n_tensors;
    MQ_REQUIRE(n > 0, "mq_adamw_step: no tensors");
    MQ_REQUIRE(d->state_bits == 32 || d->state_bits == 8, "mq_adamw_step: moments are held in 32 or 8 bits, not %d", d->state_bits);
    MQ_REQUIRE(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1 && d->eps >= 0 && d->lr >= 0 && d->max_norm >= 0,
               "mq_adamw_step: lr, eps, max_norm >= 0 and betas in [0, 1) are needed");
    const size_t tb = mq_adamw_table_bytes(numel_host, n);
    MQ_REQUIRE(tb, "mq_adamw_step: bad sizes");
    const int blocks = (int)((tb - aw_rows_bytes(n)) / sizeof(int));
    if (d->max_norm > 0)
        MQ_REQUIRE(workspace && (uintptr_t)workspace % 8 == 0 && workspace_bytes >= (size_t)blocks * sizeof(double),
                   "mq_adamw_step: the norm needs a workspace of %zu bytes, aligned to 8", (size_t)blocks * sizeof(double));
    for (int i = 0; i < n; ++i) {
        const int type = grad_types_host ? grad_types_host[i] : 0;
        MQ_REQUIRE(type <= 2, "mq_adamw_step: gradient %d: element type %d (0 f32, 1 bf16, 2 f16)", i, type);
        MQ_REQUIRE((uintptr_t)grads_host[i] % (type ? 2 : 4) == 0 && ((uint64_t)grads_host[i] >> 62) == 0, "mq_adamw_step: gradient %d is not aligned to its type", i);
    }
    const AwRow *rows = reinterpret_cast<const AwRow *>(table);
    const int *row_of = reinterpret_cast<const int *>(reinterpret_cast<const char *>(table) + aw_rows_bytes(n));
    AwControl *ctl = reinterpret_cast<AwControl *>(control);
    AwState *st = reinterpret_cast<AwState *>(ctl + 1);
    AwHyper h;
    h.lr = d->lr; h.beta1 = d->beta1; h.beta2 = d->beta2; h.grad_scale = d->grad_scale; h.max_norm = d->max_norm;
    h.omb1 = (float)(1.0 - d->beta1); h.b2 = (float)d->beta2; h.omb2 = (float)(1.0 - d->beta2); h.eps = (float)d->eps;
    h.seed = d->seed;
    double *part = reinterpret_cast<double *>(workspace);
    // three passes over the launches of up to AW_GRADS tensors: squares, factors, update
    int parts = 0;
    for (int pass = d->max_norm > 0 ? 0 : 1; pass < 3; ++pass) {
        int block0 = 0;
        for (int row0 = 0; row0 < n; row0 += AW_GRADS) {
            const int nr = n - row0 < AW_GRADS ? n - row0 : AW_GRADS;
            AwGrads g;
            int nb = 0;
            for (int i = 0; i < nr; ++i) {
                const uint64_t a = numel_host[row0 + i] ? (uint64_t)grads_host[row0 + i] : 0;
                g.g[i] = a ? a | (uint64_t)(grad_types_host ? grad_types_host[row0 + i] : 0) << 62 : 0;
                nb += (int)aw_blocks(numel_host[row0 + i]);
            }
            if (pass == 1)
                hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(1024), 0, S(stream), g, rows, row0, nr, row0 == 0, part, parts, h, present, ctl, st);
            else if (nb && pass == 0) {
                const int np = (int)cdiv(nb, AW_NORM);
                hipLaunchKernelGGL(adamw_sumsq_kernel, dim3(np), dim3(256), 0, S(stream), g, rows, row_of, row0, block0, nb, parts, part);
                parts += np;
            } else if (nb && d->state_bits == 8)
                hipLaunchKernelGGL(adamw_kernel<true>, dim3(nb), dim3(256), 0, S(stream), g, rows, row_of, row0, block0, h, present, ctl, st);
            else if (nb)
                hipLaunchKernelGGL(adamw_kernel<false>, dim3(nb), dim3(256), 0, S(stream), g, rows, row_of, row0, block0, h, present, ctl, st);
            block0 += nb;
        }
    }
    MQ_LAUNCH_CHECK("mq_adamw_step");
    return 0;
}

extern "C" int mq_adamw_step(const mqAdamwDesc *d, const int64_t *numel_host, const void *table, const void *const *grads_host,
                             const uint8_t *grad_types_host, void *control, void *workspace, size_t workspace_bytes, mqStream stream)
{
    return adamw_step(d, numel_host, table, grads_host, grad_types_host, nullptr, control, workspace, workspace_bytes, stream);
}

extern "C" int mq_adamw_step_present(const mqAdamwDesc *d, const int64_t *numel_host, const void *table, const void *const *grads_host,
                                     const uint8_t *grad_types_host, const float *present, void *control, void *workspace, size_t workspace_bytes,
                                     mqStream stream)
{
    MQ_REQUIRE(present && (uintptr_t)present % 4 == 0, "mq_adamw_step_present: present is NULL or not aligned");
    return adamw_step(d, numel_host, table, grads_host, grad_types_host, present, control, workspace, workspace_bytes, stream);
}

extern "C" int mq_moments8_encode(const float *exp_avg, const float *exp_avg_sq, int64_t n, uint8_t *codes_avg, uint8_t *base_avg,
                                  uint8_t *codes_avg_sq, uint8_t *base_avg_sq, mqStream stream)
{
    MQ_REQUIRE(exp_avg && exp_avg_sq && codes_avg && base_avg && codes_avg_sq && base_avg_sq && n > 0 && n % 256 == 0, "mq_moments8_encode: bad arguments (n is a multiple of 256)");
    MQ_REQUIRE(((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) % 16 == 0 && ((uintptr_t)codes_avg | (uintptr_t)codes_avg_sq) % 4 == 0, "mq_moments8_encode: moments start at multiples of 16 bytes, codes of 4");
    MQ_REQUIRE(cdiv(n, 1024) < AW_MOST, "mq_moments8_encode: too many elements");
    hipLaunchKernelGGL(moments8_encode_kernel, dim3((unsigned)cdiv(n, 1024)), dim3(256), 0, S(stream), exp_avg, exp_avg_sq, n / 256,
                       reinterpret_cast<uint32_t *>(codes_avg), base_avg, reinterpret_cast<uint32_t *>(codes_avg_sq), base_avg_sq);
    MQ_LAUNCH_CHECK("mq_moments8_encode");
    return 0;
}

extern "C" int mq_moments8_decode(const uint8_t *codes_avg, const uint8_t *base_avg, const uint8_t *codes_avg_sq, const uint8_t *base_avg_sq,
                                  int64_t n, int bf16, void *exp_avg, void *exp_avg_sq, mqStream stream)
{
    MQ_REQUIRE(codes_avg && base_avg && codes_avg_sq && base_avg_sq && exp_avg && exp_avg_sq && n > 0 && n % 256 == 0, "mq_moments8_decode: bad arguments (n is a multiple of 256)");
    MQ_REQUIRE(((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) % 16 == 0 && ((uintptr_t)codes_avg | (uintptr_t)codes_avg_sq) % 8 == 0, "mq_moments8_decode: moments start at multiples of 16 bytes, codes of 8");
    const int64_t n8 = n / 8;
    MQ_REQUIRE(cdiv(n8, 256) < AW_MOST, "mq_moments8_decode: too many elements");
    const uint2 *mc = reinterpret_cast<const uint2 *>(codes_avg), *vc = reinterpret_cast<const uint2 *>(codes_avg_sq);
    if (bf16)
        hipLaunchKernelGGL(moments8_decode_kernel<true>, dim3((unsigned)cdiv(n8, 256)), dim3(256), 0, S(stream), mc, base_avg, vc, base_avg_sq, n8, exp_avg, exp_avg_sq);
    else
        hipLaunchKernelGGL(moments8_decode_kernel<false>, dim3((unsigned)cdiv(n8, 256)), dim3(256), 0, S(stream), mc, base_avg, vc, base_avg_sq, n8, exp_avg, exp_avg_sq);
    MQ_LAUNCH_CHECK("mq_moments8_decode");
    return 0;
}
