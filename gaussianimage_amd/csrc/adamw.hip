// adamw.hip -- the AdamW step over a list of tensors, with states in 32 bits or in 8, and the
// norm of a list of gradients with the clip coefficient that belongs to it.
//
// One element of the step (g the gradient times the clip coefficient, t the step count):
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// 28 bytes move per element in 32 bits, 16 with 8-bit states (10 with bf16 parameters), for ~15
// operations: long lists are bound by memory, short ones by the launch.  So everything about an
// element is done in one pass, and a list of tensors goes into few launches: the pointers of up
// to 64 (48 in 8 bits) tensors travel in the kernel arguments -- nothing is staged in device
// memory, so a call may be captured into a graph -- and a workgroup finds the tensor of its chunk
// with one load per lane and one ballot over the tensors' first chunks.
#include "host.h"

#define ADAMW_THREADS 256
#define ADAMW_CHUNK 2048          // elements of a workgroup: 8 per lane, 8 blocks of 256
#define ADAMW_MAX_NUMEL ((int64_t)1 << 34)
#define ADAMW_MAX_CHUNKS (1 << 23)  // chunks of a launch: 256 lanes each, below 2^32 lanes

struct AdamWScalars {
    float b1, omb1, b2, omb2, eps, decay, step, inv_bc2;
    unsigned key;
};

// (Fields of 4 and 8 bytes only.  A scalar load ignores the two low bits of EACH part of its
// address; with an array of bytes beside the others the compiler split an index 8 k into a base
// + k and an offset 7 k, whose sum alone is aligned: pointers came from the wrong place.)
template <int BITS>
struct AdamWTable {
    static constexpr int N = BITS == 8 ? 48 : 64;
    void *p[N];
    const void *g[N];
    void *m[N];
    void *v[N];
    float *w[N];                            // masters
    float *sm[BITS == 8 ? N : 1], *sv[BITS == 8 ? N : 1];
    long long numel[N];
    int first[N];                           // first chunk of the tensor in this launch
    unsigned block0[BITS == 8 ? N : 1];     // first block of the tensor in the whole call
    int vec[N];                             // every pointer allows four elements per access
    int count;
};

// ---- element types ---------------------------------------------------------------------------
// Half types are widened exactly on the way in and rounded once, to nearest even, on the way out.
template <int TYPE> struct Elem;
template <> struct Elem<GI2D_F32> {
    typedef float type;
    typedef float vec __attribute__((ext_vector_type(4)));
};
template <> struct Elem<GI2D_BF16> {
    typedef __bf16 type;
    typedef __bf16 vec __attribute__((ext_vector_type(4)));
};
template <> struct Elem<GI2D_F16> {
    typedef _Float16 type;
    typedef _Float16 vec __attribute__((ext_vector_type(4)));
};

template <int TYPE>
__device__ __forceinline__ void load4(const void *base, long long i, float *x)
{
    const typename Elem<TYPE>::vec q =
        *(const typename Elem<TYPE>::vec *)((const typename Elem<TYPE>::type *)base + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)q[j];
}

template <int TYPE>
__device__ __forceinline__ void store4(void *base, long long i, const float *x)
{
    typename Elem<TYPE>::vec q;
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = (typename Elem<TYPE>::type)x[j];
    *(typename Elem<TYPE>::vec *)((typename Elem<TYPE>::type *)base + i) = q;
}

template <int TYPE>
__device__ __forceinline__ float load1(const void *base, long long i)
{
    return (float)((const typename Elem<TYPE>::type *)base)[i];
}

template <int TYPE>
__device__ __forceinline__ void store1(void *base, long long i, float x)
{
    ((typename Elem<TYPE>::type *)base)[i] = (typename Elem<TYPE>::type)x;
}

// One element; m and v are the new ones afterwards, the root of v is returned.
__device__ __forceinline__ float adamw_element(const AdamWScalars &h, float g, float &p, float &m,
                                               float &v)
{
    m = m * h.b1 + g * h.omb1;
    v = v * h.b2 + (g * g) * h.omb2;
    const float root = sqrtf(v);
    p = p * h.decay - (m / (root * h.inv_bc2 + h.eps)) * h.step;
    return root;
}

// The tensor a chunk belongs to: the last one whose first chunk is not behind it (a tensor
// without elements is not in the table, so the first chunks rise).
__device__ __forceinline__ int tensor_of(const int *first, int count, int chunk)
{
    const int lane = threadIdx.x & (WAVE - 1);
    const int f = lane < count ? first[lane] : INT_MAX;
    return __popcll(__ballot(f <= chunk)) - 1;
}

template <int PT, int GT, bool MASTER>
__global__ __launch_bounds__(ADAMW_THREADS) void adamw_step_kernel(
    AdamWTable<32> T, AdamWScalars ha, const AdamWScalars *__restrict__ h_dev,
    const float *__restrict__ clip_dev)
{
    const int k = tensor_of(T.first, T.count, (int)blockIdx.x);
    const AdamWScalars h = h_dev ? *h_dev : ha;
    const float clip = clip_dev ? *clip_dev : 1.0f;
    const long long n = T.numel[k];
    const long long base = (long long)((int)blockIdx.x - T.first[k]) * ADAMW_CHUNK;
    void *__restrict__ p = T.p[k];
    const void *__restrict__ g = T.g[k];
    float *__restrict__ m = (float *)T.m[k];
    float *__restrict__ v = (float *)T.v[k];
    float *__restrict__ w = T.w[k];
    if (T.vec[k] && base + ADAMW_CHUNK <= n) {
        float pv[2][4], gv[2][4], mv[2][4], vv[2][4];
        const long long i0 = base + 4 * (int)threadIdx.x;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long long i = i0 + u * (ADAMW_CHUNK / 2);
            load4<GT>(g, i, gv[u]);
            if (MASTER) load4<GI2D_F32>(w, i, pv[u]);
            else load4<PT>(p, i, pv[u]);
            load4<GI2D_F32>(m, i, mv[u]);
            load4<GI2D_F32>(v, i, vv[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long long i = i0 + u * (ADAMW_CHUNK / 2);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                adamw_element(h, gv[u][j] * clip, pv[u][j], mv[u][j], vv[u][j]);
            store4<PT>(p, i, pv[u]);
            if (MASTER) store4<GI2D_F32>(w, i, pv[u]);
            store4<GI2D_F32>(m, i, mv[u]);
            store4<GI2D_F32>(v, i, vv[u]);
        }
        return;
    }
    // the end of a tensor, or one whose pointers allow single elements only
    const long long end = base + ADAMW_CHUNK < n ? base + ADAMW_CHUNK : n;
    for (long long i = base + threadIdx.x; i < end; i += ADAMW_THREADS) {
        float pi = MASTER ? w[i] : load1<PT>(p, i), mi = m[i], vi = v[i];
        adamw_element(h, load1<GT>(g, i) * clip, pi, mi, vi);
        store1<PT>(p, i, pi);
        if (MASTER) w[i] = pi;
        m[i] = mi;
        v[i] = vi;
    }
}

// ---- states in 8 bits ------------------------------------------------------------------------
// A state is held as e4m3 codes with one power-of-two scale for 256 consecutive elements: the
// mean as it is, the square as its root (which halves the range of exponents, and the step needs
// the root anyway).  The scale is the smallest power of two with max|x| <= 448 scale.  A power of
// two rather than max/448: a state that has not changed keeps its code, nothing drifts by being
// rescaled, and encoding needs no division.  Rounding is stochastic: |x| / scale goes to one of
// its two neighbours at random so that the mean is kept.  With b2 = 0.999 the square changes by
// 0.1 % per step and neighbouring codes are 6 to 12 % apart: rounded to nearest it would never
// move again.  The parameters are updated with m and v before they are rounded.
__device__ __forceinline__ unsigned hash32(unsigned x)
{
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ (x >> 16);
}

#define HASH_STRIDE 0x9E3779B9u  // odd: successive indices are far apart before they are hashed

// Largest of the 64 lanes' values, in every lane (a lane's partners by row mirrors, as in
// wave_sum_lane0).
__device__ __forceinline__ unsigned wave_max_u32(unsigned v)
{
    const auto up = [](unsigned a, int b) { return a > (unsigned)b ? a : (unsigned)b; };
    v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
    v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
    v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));
    v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));
    const unsigned r0 = __builtin_amdgcn_readlane((int)v, 0), r1 = __builtin_amdgcn_readlane((int)v, 16);
    const unsigned r2 = __builtin_amdgcn_readlane((int)v, 32), r3 = __builtin_amdgcn_readlane((int)v, 48);
    return up(up(r0, r1), up(r2, r3));
}

// Exponent of the scale for a largest magnitude (its bits): 448 = 1.75 * 2^8.  At least 2^-100 (its
// reciprocal and the codes' values stay normal numbers) and at most 2^119 (448 * 2^119 is finite).
__device__ __forceinline__ int scale_exponent(unsigned top)
{
    const int k = (int)((top + 0x1FFFFFu) >> 23) - 135;
    return k < -100 ? -100 : k > 119 ? 119 : k;
}

// e4m3 code of x / 2^k.  |x| 2^(-k-120) has, as a float, the code's exponent and fraction in its
// upper bits -- e4m3's subnormals line up with fp32's, which this part does not flush -- so adding
// 20 random bits below them and cutting rounds at random.  16 of them are random and the half of
// their last place is set: the mean is kept to 2^-16 of a code's step.
__device__ __forceinline__ unsigned encode_e4m3(float x, int k, unsigned random16)
{
    const unsigned y = __float_as_uint(ldexpf(fabsf(x), -k - 120));
    unsigned c = (y + (random16 * 16u + 8u)) >> 20;
    c = c < 126u ? c : 126u;
    if (!(fabsf(x) <= 3.402823466e38f)) c = 127u;  // infinities and NaN: the NaN code
    return c | ((__float_as_uint(x) >> 24) & 0x80u);
}

__device__ __forceinline__ unsigned finite_bits(float x)
{
    const unsigned b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ void decode4(unsigned codes, float scale, float *x)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    x[0] = lo[0] * scale;
    x[1] = lo[1] * scale;
    x[2] = hi[0] * scale;
    x[3] = hi[1] * scale;
}

// A wave owns whole blocks of 256 elements, four neighbouring ones per lane, so that a block's
// largest magnitudes need no memory and its scale no atomics.
template <int PT, int GT, bool MASTER>
__global__ __launch_bounds__(ADAMW_THREADS) void adamw_step8_kernel(
    AdamWTable<8> T, AdamWScalars ha, const AdamWScalars *__restrict__ h_dev,
    const float *__restrict__ clip_dev)
{
    const int k = tensor_of(T.first, T.count, (int)blockIdx.x);
    const AdamWScalars h = h_dev ? *h_dev : ha;
    const float clip = clip_dev ? *clip_dev : 1.0f;
    const long long n = T.numel[k];
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const bool vec = T.vec[k];
    void *__restrict__ p = T.p[k];
    const void *__restrict__ g = T.g[k];
    unsigned char *__restrict__ m = (unsigned char *)T.m[k];
    unsigned char *__restrict__ v = (unsigned char *)T.v[k];
    float *__restrict__ w = T.w[k];
    float *__restrict__ sm = T.sm[k], *__restrict__ sv = T.sv[k];
    const long long block = (long long)((int)blockIdx.x - T.first[k]) *
                                (ADAMW_CHUNK / GI2D_ADAMW_BLOCK) + wave * 2;
    float pv[2][4], gv[2][4], mv[2][4], vv[2][4], km[2], kv[2];
    unsigned mc[2], vc[2];
    bool whole[2], some[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const long long b0 = (block + u) * GI2D_ADAMW_BLOCK, i = b0 + 4 * lane;
        some[u] = b0 < n;
        whole[u] = vec && b0 + GI2D_ADAMW_BLOCK <= n;
        if (!some[u]) continue;
        km[u] = sm[block + u];
        kv[u] = sv[block + u];
        if (whole[u]) {
            load4<GT>(g, i, gv[u]);
            if (MASTER) load4<GI2D_F32>(w, i, pv[u]);
            else load4<PT>(p, i, pv[u]);
            mc[u] = *(const unsigned *)(m + i);
            vc[u] = *(const unsigned *)(v + i);
        } else {
            mc[u] = vc[u] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                gv[u][j] = pv[u][j] = 0.0f;
                if (i + j < n) {
                    gv[u][j] = load1<GT>(g, i + j);
                    pv[u][j] = MASTER ? w[i + j] : load1<PT>(p, i + j);
                    mc[u] |= (unsigned)m[i + j] << (8 * j);
                    vc[u] |= (unsigned)v[i + j] << (8 * j);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (!some[u]) continue;
        const long long i = (block + u) * GI2D_ADAMW_BLOCK + 4 * lane;
        decode4(mc[u], km[u], mv[u]);
        decode4(vc[u], kv[u], vv[u]);
        float root[4];
        unsigned top_m = 0, top_r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vv[u][j] = vv[u][j] * vv[u][j];
            root[j] = adamw_element(h, gv[u][j] * clip, pv[u][j], mv[u][j], vv[u][j]);
            const unsigned bm = finite_bits(mv[u][j]), br = finite_bits(root[j]);
            top_m = top_m > bm ? top_m : bm;
            top_r = top_r > br ? top_r : br;
        }
        const int em = scale_exponent(wave_max_u32(top_m)), er = scale_exponent(wave_max_u32(top_r));
        const unsigned hb = hash32(h.key + (T.block0[k] + (unsigned)(block + u)) * HASH_STRIDE);
        unsigned cm = 0, cr = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned r = hash32(hb + (unsigned)(4 * lane + j) * HASH_STRIDE);
            const unsigned c = encode_e4m3(mv[u][j], em, r >> 16);
            unsigned d = encode_e4m3(root[j], er, r & 0xffffu);
            // a root that is not zero stays so: with a mean beside it, the next step would divide
            // by eps alone
            if (d == 0u && root[j] > 0.0f) d = 1u;
            cm |= c << (8 * j);
            cr |= d << (8 * j);
        }
        if (whole[u]) {
            store4<PT>(p, i, pv[u]);
            if (MASTER) store4<GI2D_F32>(w, i, pv[u]);
            *(unsigned *)(m + i) = cm;
            *(unsigned *)(v + i) = cr;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < n) {
                    store1<PT>(p, i + j, pv[u][j]);
                    if (MASTER) w[i + j] = pv[u][j];
                    m[i + j] = (unsigned char)(cm >> (8 * j));
                    v[i + j] = (unsigned char)(cr >> (8 * j));
                }
        }
        if (lane == 0) {
            sm[block + u] = __uint_as_float((unsigned)(em + 127) << 23);
            sv[block + u] = __uint_as_float((unsigned)(er + 127) << 23);
        }
    }
}

// ---- step count and learning rate in device memory ---------------------------------------------
static inline __host__ __device__ unsigned step_key(unsigned seed, long long step)
{
    unsigned x = seed;
    for (int i = 0; i < 2; ++i) {
        x ^= x >> 16;
        x *= 0x7feb352du;
        x ^= x >> 15;
        x *= 0x846ca68bu;
        x ^= x >> 16;
        if (i == 0) x ^= (unsigned)step * HASH_STRIDE;
    }
    return x;
}

// For captured steps: what depends on the step count and the learning rate is worked out on the
// device, by one lane, ahead of the step.  Powers by repeated squaring in double (an error of
// t 2^-53), the rest in float: within 2 units in the last place of the host's values.
__global__ void adamw_scalars_kernel(AdamWScalars h, double beta1, double beta2, double lr,
                                     double weight_decay, unsigned seed,
                                     const long long *__restrict__ step_dev, long long step,
                                     const float *__restrict__ lr_dev, AdamWScalars *out)
{
    if (threadIdx.x != 0) return;
    long long t = step_dev ? *step_dev : step;
    if (t < 1) t = 1;
    h.key = step_key(seed, t);
    if (lr_dev) lr = (double)*lr_dev;
    double p1 = 1.0, p2 = 1.0, q1 = beta1, q2 = beta2;
    for (; t > 0; t >>= 1) {
        if (t & 1) {
            p1 = p1 * q1;
            p2 = p2 * q2;
        }
        q1 = q1 * q1;
        q2 = q2 * q2;
    }
    h.decay = (float)(1.0 - lr * weight_decay);
    h.step = (float)lr / (float)(1.0 - p1);
    h.inv_bc2 = 1.0f / sqrtf((float)(1.0 - p2));
    *out = h;
}

// ---- norm of all gradients ---------------------------------------------------------------------
// Each workgroup sums the squares of its chunks in double (no overflow, and the sum of 2^28 squares
// is as exact as one of them) and leaves one partial; one workgroup adds the partials in a fixed
// order: the same bits in every run, no atomics, no memory to clear.
#define NORM_THREADS 256
#define NORM_TENSORS 128
#define NORM_CHUNK_BYTES 16384
#define NORM_GROUPS 2048

struct NormTable {
    const void *g[NORM_TENSORS];
    long long numel[NORM_TENSORS];
    int first[NORM_TENSORS];
    int type[NORM_TENSORS];  // element type, + 4 where 16-byte loads are not allowed
    int count, chunks;
};

__device__ __forceinline__ void add_square(double &s, float x)
{
    const double d = (double)x;
    s = s + d * d;
}

template <int TYPE>
__device__ __forceinline__ void chunk_squares(const void *g, long long n, long long chunk, bool vec,
                                              double *s)
{
    constexpr int SIZE = TYPE == GI2D_F32 ? 4 : 2, V = 16 / SIZE, CHUNK = NORM_CHUNK_BYTES / SIZE;
    typedef typename Elem<TYPE>::type E;
    typedef E vec_t __attribute__((ext_vector_type(V)));
    const long long base = chunk * CHUNK;
    const E *__restrict__ x = (const E *)g;
    if (vec && base + CHUNK <= n) {
        vec_t q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            q[u] = *(const vec_t *)(x + base + (long long)(u * NORM_THREADS + (int)threadIdx.x) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) add_square(s[j & 3], (float)q[u][j]);
        return;
    }
    const long long end = base + CHUNK < n ? base + CHUNK : n;
    for (long long i = base + threadIdx.x; i < end; i += NORM_THREADS) add_square(s[0], (float)x[i]);
}

__device__ __forceinline__ double block_sum(double v, double *lds)
{
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) v = v + __shfl_xor(v, d);
    if ((threadIdx.x & (WAVE - 1)) == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < (int)blockDim.x / WAVE; ++i) t = t + lds[i];
    return t;
}

__global__ __launch_bounds__(NORM_THREADS) void grad_squares_kernel(NormTable T, double *partials)
{
    __shared__ double lds[NORM_THREADS / WAVE];
    const int lane = threadIdx.x & (WAVE - 1);
    const int f0 = lane < T.count ? T.first[lane] : INT_MAX;
    const int f1 = lane + WAVE < T.count ? T.first[lane + WAVE] : INT_MAX;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int c = (int)blockIdx.x; c < T.chunks; c += (int)gridDim.x) {
        const int k = __popcll(__ballot(f0 <= c)) + __popcll(__ballot(f1 <= c)) - 1;
        const int type = T.type[k];
        const bool vec = type < 4;
        const long long chunk = c - T.first[k], n = T.numel[k];
        switch (type & 3) {
            case GI2D_F32: chunk_squares<GI2D_F32>(T.g[k], n, chunk, vec, s); break;
            case GI2D_BF16: chunk_squares<GI2D_BF16>(T.g[k], n, chunk, vec, s); break;
            default: chunk_squares<GI2D_F16>(T.g[k], n, chunk, vec, s); break;
        }
    }
    const double t = block_sum((s[0] + s[1]) + (s[2] + s[3]), lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = t;
}

// out[0] = norm, out[1] = min(1, max_norm / (norm + 1e-6)).  The root in float of a sum brought
// to [1/2, 2) by an even power of two: sums beyond fp32's range have norms within it.
__global__ __launch_bounds__(1024) void grad_norm_kernel(const double *__restrict__ partials, int n,
                                                         float max_norm, float *out)
{
    __shared__ double lds[1024 / WAVE];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += (int)blockDim.x) s = s + partials[i];
    s = block_sum(s, lds);
    if (threadIdx.x != 0) return;
    float norm = (float)s;  // 0, infinity and NaN are their own roots
    if (s > 0.0 && s < __builtin_inf()) {
        int e = __builtin_amdgcn_frexp_exp(s);
        double f = __builtin_amdgcn_frexp_mant(s);
        if (e & 1) {
            f = f * 2.0;
            e -= 1;
        }
        norm = ldexpf(sqrtf((float)f), e / 2);
    }
    out[0] = norm;
    const float c = max_norm / (norm + 1e-6f);
    out[1] = c < 1.0f || c != c ? c : 1.0f;
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------

static bool type_ok(int t) { return t == GI2D_F32 || t == GI2D_BF16 || t == GI2D_F16; }
static int type_size(int t) { return t == GI2D_F32 ? 4 : 2; }
static bool aligned(const void *p, int to) { return ((uintptr_t)p & (uintptr_t)(to - 1)) == 0; }

template <int BITS, int PT, int GT, bool MASTER>
static void adamw_launch(const AdamWTable<BITS> &T, int chunks, const AdamWScalars &h,
                         const AdamWScalars *h_dev, const float *clip, hipStream_t st)
{
    if constexpr (BITS == 8)
        adamw_step8_kernel<PT, GT, MASTER><<<dim3((unsigned)chunks), ADAMW_THREADS, 0, st>>>(T, h, h_dev, clip);
    else
        adamw_step_kernel<PT, GT, MASTER><<<dim3((unsigned)chunks), ADAMW_THREADS, 0, st>>>(T, h, h_dev, clip);
}

template <int BITS>
static void adamw_dispatch(int pt, int gt, bool master, const AdamWTable<BITS> &T, int chunks,
                           const AdamWScalars &h, const AdamWScalars *h_dev, const float *clip,
                           hipStream_t st)
{
#define ADAMW_CASE(P, G, M) \
    if (pt == P && gt == G && master == M) return adamw_launch<BITS, P, G, M>(T, chunks, h, h_dev, clip, st)
#define ADAMW_GRADS(P, M)           \
    ADAMW_CASE(P, GI2D_F32, M);     \
    ADAMW_CASE(P, GI2D_BF16, M);    \
    ADAMW_CASE(P, GI2D_F16, M)
    ADAMW_GRADS(GI2D_F32, false);
    ADAMW_GRADS(GI2D_BF16, false);
    ADAMW_GRADS(GI2D_F16, false);
    ADAMW_GRADS(GI2D_BF16, true);
    ADAMW_GRADS(GI2D_F16, true);
#undef ADAMW_GRADS
#undef ADAMW_CASE
}

// The tensors of one (parameter type, gradient type, masters or not), in tables of N.
template <int BITS>
static int adamw_run(int num_tensors, const gi2d_adamw_tensor *ts, int pt, int gt, bool master,
                     const AdamWScalars &h, const AdamWScalars *h_dev, const float *clip,
                     hipStream_t st)
{
    AdamWTable<BITS> T;
    T.count = 0;
    int chunks = 0;
    unsigned block0 = 0;
    const auto flush = [&]() {
        if (T.count == 0) return GI2D_OK;
        adamw_dispatch<BITS>(pt, gt, master, T, chunks, h, h_dev, clip, st);
        T.count = 0;
        chunks = 0;
        return launch_status();
    };
    for (int i = 0; i < num_tensors; ++i) {
        const gi2d_adamw_tensor &t = ts[i];
        const unsigned blocks = (unsigned)((t.numel + GI2D_ADAMW_BLOCK - 1) / GI2D_ADAMW_BLOCK);
        const unsigned at = block0;
        block0 += blocks;
        if (t.numel == 0 || t.param_type != pt || t.grad_type != gt || (t.master != nullptr) != master)
            continue;
        const int more = (int)((t.numel + ADAMW_CHUNK - 1) / ADAMW_CHUNK);
        if (T.count == AdamWTable<BITS>::N || chunks + more > ADAMW_MAX_CHUNKS) {
            const int rc = flush();
            if (rc != GI2D_OK) return rc;
        }
        const int c = T.count++;
        T.p[c] = t.param;
        T.g[c] = t.grad;
        T.m[c] = t.exp_avg;
        T.v[c] = t.exp_avg_sq;
        T.w[c] = t.master;
        T.numel[c] = t.numel;
        T.first[c] = chunks;
        const int state = BITS == 8 ? 4 : 16;
        T.vec[c] = aligned(t.param, 4 * type_size(pt)) && aligned(t.grad, 4 * type_size(gt)) &&
                   aligned(t.exp_avg, state) && aligned(t.exp_avg_sq, state) &&
                   (!master || aligned(t.master, 16));
        if constexpr (BITS == 8) {
            T.sm[c] = t.exp_avg_scale;
            T.sv[c] = t.exp_avg_sq_scale;
            T.block0[c] = at;
        }
        chunks += more;
    }
    return flush();
}

extern "C" {

int gi2d_adamw_step(int num_tensors, const gi2d_adamw_tensor *tensors,
                    const gi2d_adamw_hyper *hyper, const float *clip_dev, void *stream)
{
    if (num_tensors < 0 || !hyper || (num_tensors > 0 && !tensors)) return GI2D_E_INVALID;
    const bool on_device = hyper->step_dev || hyper->lr_dev;
    if (hyper->state_bits != 32 && hyper->state_bits != 8) return GI2D_E_INVALID;
    if ((!hyper->step_dev && hyper->step < 1) || (on_device && !hyper->scalars_dev)) return GI2D_E_INVALID;
    if (!(hyper->beta1 >= 0.0 && hyper->beta1 < 1.0 && hyper->beta2 >= 0.0 && hyper->beta2 < 1.0))
        return GI2D_E_INVALID;
    const bool bits8 = hyper->state_bits == 8;
    unsigned present = 0;  // one bit per (parameter type, gradient type, masters)
    for (int i = 0; i < num_tensors; ++i) {
        const gi2d_adamw_tensor &t = tensors[i];
        if (!type_ok(t.param_type) || !type_ok(t.grad_type) || t.numel < 0 ||
            t.numel > ADAMW_MAX_NUMEL)
            return GI2D_E_INVALID;
        if (t.numel == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return GI2D_E_INVALID;
        if (bits8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return GI2D_E_INVALID;
        if (t.master && t.param_type == GI2D_F32) return GI2D_E_INVALID;
        present |= 1u << (t.param_type * 6 + t.grad_type * 2 + (t.master ? 1 : 0));
    }
    if (!present) return GI2D_OK;
    hipStream_t st = (hipStream_t)stream;
    AdamWScalars h;
    h.b1 = (float)hyper->beta1;
    h.omb1 = (float)(1.0 - hyper->beta1);
    h.b2 = (float)hyper->beta2;
    h.omb2 = (float)(1.0 - hyper->beta2);
    h.eps = (float)hyper->eps;
    h.decay = h.step = h.inv_bc2 = 0.0f;
    h.key = 0;
    const AdamWScalars *h_dev = nullptr;
    if (on_device) {
        static_assert(sizeof(AdamWScalars) <= GI2D_ADAMW_SCALARS_BYTES, "scalars_dev too small");
        adamw_scalars_kernel<<<1, WAVE, 0, st>>>(h, hyper->beta1, hyper->beta2, hyper->lr,
                                                 hyper->weight_decay, hyper->seed,
                                                 (const long long *)hyper->step_dev, hyper->step,
                                                 hyper->lr_dev, (AdamWScalars *)hyper->scalars_dev);
        const int rc = launch_status();
        if (rc != GI2D_OK) return rc;
        h_dev = (const AdamWScalars *)hyper->scalars_dev;
    } else {
        const double t = (double)hyper->step;
        h.decay = (float)(1.0 - hyper->lr * hyper->weight_decay);
        h.step = (float)(hyper->lr / (1.0 - pow(hyper->beta1, t)));
        h.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(hyper->beta2, t)));
        h.key = step_key(hyper->seed, hyper->step);
    }
    for (int pt = 0; pt < 3; ++pt)
        for (int gt = 0; gt < 3; ++gt)
            for (int master = 0; master < 2; ++master) {
                if (!(present & (1u << (pt * 6 + gt * 2 + master)))) continue;
                const int rc = bits8 ? adamw_run<8>(num_tensors, tensors, pt, gt, master != 0, h,
                                                    h_dev, clip_dev, st)
                                     : adamw_run<32>(num_tensors, tensors, pt, gt, master != 0, h,
                                                     h_dev, clip_dev, st);
                if (rc != GI2D_OK) return rc;
            }
    return GI2D_OK;
}

int64_t gi2d_grad_norm_workspace(int num_tensors)
{
    if (num_tensors < 0) return GI2D_E_INVALID;
    const int64_t launches = ((int64_t)num_tensors + NORM_TENSORS - 1) / NORM_TENSORS;
    return (launches > 1 ? launches : 1) * NORM_GROUPS * (int64_t)sizeof(double);
}

int gi2d_grad_norm(int num_tensors, const void *const *grads, const int64_t *numel,
                   const int *types, double max_norm, void *workspace, float *out, void *stream)
{
    if (num_tensors < 0 || !out || !workspace || !(max_norm >= 0.0)) return GI2D_E_INVALID;
    if (num_tensors > 0 && (!grads || !numel || !types)) return GI2D_E_INVALID;
    for (int i = 0; i < num_tensors; ++i)
        if (!type_ok(types[i]) || numel[i] < 0 || numel[i] > ADAMW_MAX_NUMEL ||
            (numel[i] > 0 && !grads[i]))
            return GI2D_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    double *partials = (double *)workspace;
    NormTable T;
    T.count = T.chunks = 0;
    int done = 0;
    const auto flush = [&]() {
        if (T.count == 0) return GI2D_OK;
        const int groups = T.chunks < NORM_GROUPS ? T.chunks : NORM_GROUPS;
        grad_squares_kernel<<<dim3((unsigned)groups), NORM_THREADS, 0, st>>>(T, partials + done);
        done += groups;
        T.count = T.chunks = 0;
        return launch_status();
    };
    for (int i = 0; i < num_tensors; ++i) {
        if (numel[i] == 0) continue;
        const int64_t chunk = NORM_CHUNK_BYTES / type_size(types[i]);
        const int64_t more = (numel[i] + chunk - 1) / chunk;  // at most 2^22
        // (a table is full at 128 tensors, 2^29 chunks)
        if (T.count == NORM_TENSORS) {
            const int rc = flush();
            if (rc != GI2D_OK) return rc;
        }
        const int c = T.count++;
        T.g[c] = grads[i];
        T.numel[c] = numel[i];
        T.type[c] = types[i] + (aligned(grads[i], 16) ? 0 : 4);
        T.first[c] = T.chunks;
        T.chunks += (int)more;
    }
    int rc = flush();
    if (rc != GI2D_OK) return rc;
    const int threads = done <= 256 ? 256 : 1024;
    grad_norm_kernel<<<1, threads, 0, st>>>(partials, done, (float)max_norm, out);
    return launch_status();
}

}  // extern "C"
