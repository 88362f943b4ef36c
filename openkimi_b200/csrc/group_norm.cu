// Group normalisation with an activation over channels-last activations x [N, S, Ch]:
//
//   z = (x - mean) rstd w + b,  y = z or z sigmoid(z),  mean and variance over the S positions and Ch / G channels of (n, group)
//   dz = dy act'(z);  dw_c = sum dz x^,  db_c = sum dz,  dx = rstd (dz w - m1 - x^ m2),  m1 = mean(dz w), m2 = mean(dz w x^)
//
// HBM-bound: forward one read and one write, backward two reads and one write per value.
//   * S = 1 (every token by itself, groups of up to 1024 channels): L lanes hold a group of one row in registers, so that one pass
//     does it all, the next row on its way meanwhile; the lanes keep their group over the rows they walk and with it w, b and their
//     shares of dw, db.
//   * else: a thread keeps VEC channels and walks rows of a slice of a sample.  Forward: sums of x and x^2 about a row of its own, then
//     about the mean of its first rows, joined over the slice's channels to (mean, sum of squared deviations) of a group, and over
//     the slices at the start of the second pass, which applies.  Backward: per slice and channel the sums of dz and dz x^, which
//     give dw, db and, weighted with w, m1 and m2; then dx.  The second pass reads from L2 what fits there.
// Bound by issue slots (70 % of them used in the first form) and by the latency of small slices: [32768, 768] in groups of 128, BF16
// with SiLU, takes 26 us forward (3.8 TB/s) and 49 backward (3.1 TB/s, 72 bytes of spills); [4, 8191, 768] in 32 groups 49 and 64
// (3.1 and 4.3 TB/s of what its passes read and write).  In the first form the two took 172 and 291 us; what made them faster is two values an instruction, a
// thread's channels all of one group, rows kept as they lie in memory until they are used, and a grid of what is resident.
// Sums are in FP32 over at most 1024 rows, then in 64 bits in a fixed order: no atomics.
#include "kda_common.cuh"

namespace kda {
namespace gn {

using bf16 = __nv_bfloat16;
constexpr int NTHR = 256;
constexpr int SLICE_THR = 384;    // at most, in the kernels over slices
constexpr int ROWS_MAX = 1024;    // channels of a group that 32 lanes hold in registers
constexpr int MAX_SLICES = 256;   // of a sample in the second pass
constexpr int SUM_ROWS = 1024;    // that one FP32 sum adds up
constexpr int GROUPS_MAX = KDA_GROUP_NORM_MAX_GROUPS; // whose numbers fit shared memory where they are not taken row by row

struct Args {
    const void *x, *dy;
    void *y, *dx;
    const float *w, *b;           // may be NULL: 1, 0
    float *mean, *rstd;           // [N, G]
    float *dw, *db;               // [Ch], may be NULL
    float* part;                  // scratch
    long long N, S;
    long long len, span;          // rows of a slice of the first pass, of the second
    int Ch, G, act, slices, cuts; // slices of a sample in either
    float eps;
    double inv_S, inv_Cg;         // 1 / S, 1 / (Ch / G)
};

// VEC elements as they lie in memory: 16 bytes, two elements or one
template <typename T, int VEC> struct Raw { T v[VEC]; };
template <> struct Raw<float, 4> { uint4 v; };
template <> struct Raw<bf16, 8> { uint4 v; };
template <> struct Raw<float, 2> { float2 v; };
template <> struct Raw<bf16, 2> { uint32_t v; };
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, VEC>*>(p); }
__device__ __forceinline__ void unpack(const Raw<float, 1>& r, float (&x)[1]) { x[0] = r.v[0]; }
__device__ __forceinline__ void unpack(const Raw<bf16, 1>& r, float (&x)[1]) { x[0] = __bfloat162float(r.v[0]); }
__device__ __forceinline__ void unpack(const Raw<float, 2>& r, float (&x)[2]) { x[0] = r.v.x; x[1] = r.v.y; }
__device__ __forceinline__ void unpack(const Raw<bf16, 2>& r, float (&x)[2]) { x[0] = __uint_as_float(r.v << 16); x[1] = __uint_as_float(r.v & 0xffff0000u); }
__device__ __forceinline__ void unpack(const Raw<float, 4>& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.v.x); x[1] = __uint_as_float(r.v.y); x[2] = __uint_as_float(r.v.z); x[3] = __uint_as_float(r.v.w);
}
__device__ __forceinline__ void unpack(const Raw<bf16, 8>& r, float (&x)[8]) {
    const uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&v)[VEC]) { unpack(load_raw<T, VEC>(p), v); }
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&v)[VEC]) {
    if constexpr (sizeof(T) * VEC == 16) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                u[i] = __float_as_uint(v[i]);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    } else if constexpr (VEC == 2 && sizeof(T) == 4) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else if constexpr (VEC == 2) {
        *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v[0], v[1]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) stf(p + i, v[i]);
    }
}

// d = a b + c, a b, a + b over VEC elements, two an instruction
template <int VEC, typename A, typename B, typename X>
__device__ __forceinline__ void vfma(float (&d)[VEC], const A& a, const B& b, const X& c) {
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        const float2 r = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), make_float2(c[i], c[i + 1]));
        d[i] = r.x;
        d[i + 1] = r.y;
    }
    if (VEC & 1) d[VEC - 1] = fmaf(a[VEC - 1], b[VEC - 1], c[VEC - 1]);
}
template <int VEC, typename A, typename B>
__device__ __forceinline__ void vmul(float (&d)[VEC], const A& a, const B& b) {
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
        d[i] = r.x;
        d[i + 1] = r.y;
    }
    if (VEC & 1) d[VEC - 1] = a[VEC - 1] * b[VEC - 1];
}
template <int VEC, typename A, typename B>
__device__ __forceinline__ void vadd(float (&d)[VEC], const A& a, const B& b) {
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        const float2 r = __fadd2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
        d[i] = r.x;
        d[i + 1] = r.y;
    }
    if (VEC & 1) d[VEC - 1] = a[VEC - 1] + b[VEC - 1];
}
struct Same { float v; __device__ __forceinline__ float operator[](int) const { return v; } };  // one number for all of them
// sums over a thread's elements, in two halves
template <int VEC>
__device__ __forceinline__ float2 sum2(float2 s, const float (&a)[VEC]) {
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) s = __fadd2_rn(make_float2(a[i], a[i + 1]), s);
    if (VEC & 1) s.x += a[VEC - 1];
    return s;
}
template <int VEC>
__device__ __forceinline__ float2 dot2(float2 s, const float (&a)[VEC], const float (&b)[VEC]) {
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) s = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]), s);
    if (VEC & 1) s.x = fmaf(a[VEC - 1], b[VEC - 1], s.x);
    return s;
}

// FP32 values go through expf and a division, BF16 ones through the hardware's 2^x and 1 / x (2 ulp and 1, and |z| 2^-24 from the
// argument)
template <typename T, int VEC>
__device__ __forceinline__ void sigmoid(float (&s)[VEC], const float (&z)[VEC]) {
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = 1.f / (1.f + expf(-z[i]));
    } else {
        vmul(s, z, Same{-LOG2E});
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = ex2_ftz(s[i]);
        vadd(s, s, Same{1.f});
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] = rcp_ftz(s[i]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void act(float (&y)[VEC], const float (&z)[VEC], bool silu) {
    if (silu) {
        sigmoid<T>(y, z);
        vmul(y, y, z);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[i] = z[i];
    }
}
// dz = dy act'(z), act'(z) = s + s z (1 - s)
template <typename T, int VEC>
__device__ __forceinline__ void act_grad(float (&dz)[VEC], const float (&z)[VEC], const float (&dy)[VEC], bool silu) {
    if (silu) {
        float s[VEC], u[VEC];
        sigmoid<T>(s, z);
        vfma(u, s, Same{-1.f}, Same{1.f});
        vfma(u, u, z, Same{1.f});
        vmul(s, s, dy);
        vmul(dz, s, u);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) dz[i] = dy[i];
    }
}
// over L = 2^i lanes
__device__ __forceinline__ float lanes_sum(float v, int L) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < L) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// three sums at once
__device__ __forceinline__ void lanes_sum(double& a, double& b, double& c, int L) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < L) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
            c += __shfl_xor_sync(0xffffffffu, c, o);
        }
}
// Sums u of w d and q of w d^2, d differences from some number: the sum of w (d - mean)^2, w adding up to 1 / inv.  (In 64 bits the
// difference loses nothing that FP32 d have; rounding leaves it no less than 0, and a NaN stays one.)
__device__ __forceinline__ double deviations(double u, double q, double inv) {
    const double d = q - u * u * inv;
    return d < 0.0 ? 0.0 : d;
}
template <typename T>
__device__ __forceinline__ float inv_sqrt(float v) { return sizeof(T) == 4 ? 1.f / sqrtf(v) : rsqrtf(v); }

// ---- one row at a time ------------------------------------------------------------------------------------------------
// Slots of L lanes; slot s has group s mod G and rows s / G, s / G + step, ...  Every lane of a warp makes the same number of turns.
template <typename T, int VEC, int NV, bool BWD>
__global__ void __launch_bounds__(NTHR, NV * VEC <= 8 ? (BWD ? 3 : 4) : NV * VEC <= 16 ? 2 : 1) group_norm_rows_kernel(const Args a, int L) {
    const int lane = threadIdx.x & (L - 1), Cg = a.Ch / a.G;
    const long long slot = ((long long)blockIdx.x * NTHR + threadIdx.x) / L, slots = (long long)gridDim.x * NTHR / L;
    const long long step = slots / a.G;            // rows between a slot's rows; slots beyond step * G have none
    const bool idle = slot >= step * a.G;
    const int g = (int)(slot % a.G), c0 = g * Cg;
    const float inv = 1.f / Cg;
    const bool silu = a.act;
    pdl_wait();
    const T* X = static_cast<const T*>(a.x);
    float w[NV][VEC], b[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = (j * L + lane) * VEC + i;
            const bool in = c < Cg;
            w[j][i] = in && a.w ? a.w[c0 + c] : 1.f;
            b[j][i] = in && a.b ? a.b[c0 + c] : 0.f;
            dw[j][i] = db[j][i] = 0.f;
        }
    Raw<T, VEC> nx[NV], ndy[NV];                   // the next row
    const long long row0 = slot / a.G, turns = (a.N + step - 1) / step, rows = idle || row0 >= a.N ? 0 : (a.N - row0 + step - 1) / step;
    const size_t first = (size_t)(rows ? row0 : 0) * a.Ch + c0 + lane * VEC, ahead = (size_t)step * a.Ch;
    const int own = Cg - lane * VEC;               // channels of the group from this lane's first on
    auto request = [&](size_t at, bool on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nx[j] = ndy[j] = Raw<T, VEC>{};
            if (on && j * L * VEC < own) {
                nx[j] = load_raw<T, VEC>(X + at + j * L * VEC);
                if (BWD) ndy[j] = load_raw<T, VEC>(static_cast<const T*>(a.dy) + at + j * L * VEC);
            }
        }
    };
    request(first, rows > 0);
    size_t at = first;
    for (long long k = 0; k < turns; ++k, at += ahead) {
        const bool on = k < rows;
        float x[NV][VEC], dy[NV][VEC];
        float2 s = make_float2(0.f, 0.f), q = s;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack(nx[j], x[j]);
            if (BWD) unpack(ndy[j], dy[j]);
            s = sum2(s, x[j]);
        }
        request(at + ahead, k + 1 < rows);
        const float mean = lanes_sum(s.x + s.y, L) * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            vadd(x[j], x[j], Same{-mean});
            if (j * L * VEC < own) q = dot2(q, x[j], x[j]);
        }
        const float var = lanes_sum(q.x + q.y, L) * inv, rstd = on ? inv_sqrt<T>(var + a.eps) : 0.f;  // (no row: no infinity into dw, db)
        if (!BWD) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float y[VEC];
                vmul(x[j], x[j], Same{rstd});
                vfma(x[j], x[j], w[j], b[j]);
                act<T>(y, x[j], silu);
                if (on && j * L * VEC < own) store<T, VEC>(static_cast<T*>(a.y) + at + j * L * VEC, y);
            }
        } else {
            float2 t1 = make_float2(0.f, 0.f), t2 = t1;
#pragma unroll
            for (int j = 0; j < NV; ++j) {  // (beyond the group's end dy = 0)
                float z[VEC];
                vmul(x[j], x[j], Same{rstd});
                vfma(z, x[j], w[j], b[j]);
                act_grad<T>(dy[j], z, dy[j], silu);
                vadd(db[j], db[j], dy[j]);
                vfma(dw[j], dy[j], x[j], dw[j]);
                vmul(dy[j], dy[j], w[j]);
                t1 = sum2(t1, dy[j]);
                t2 = dot2(t2, dy[j], x[j]);
            }
            const float m1 = -lanes_sum(t1.x + t1.y, L) * inv, m2 = -lanes_sum(t2.x + t2.y, L) * inv;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float dx[VEC];
                vadd(dx, dy[j], Same{m1});  // (before rstd: a group of one channel has exactly 0)
                vfma(dx, x[j], Same{m2}, dx);
                vmul(dx, dx, Same{rstd});
                if (on && j * L * VEC < own) store<T, VEC>(static_cast<T*>(a.dx) + at + j * L * VEC, dx);
            }
        }
    }
    if (BWD && a.dw && !idle) {  // part[step][2][Ch]
        float* out = a.part + (size_t)(slot / a.G) * 2 * a.Ch + c0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int c = (j * L + lane) * VEC + i;
                if (c < Cg) {
                    out[c] = dw[j][i];
                    out[a.Ch + c] = db[j][i];
                }
            }
    }
}

// dw, db: sums of part[count][2][Ch] over count, 32 channels a CTA
__global__ void __launch_bounds__(1024) group_norm_params_kernel(const float* part, long long count, int Ch, float* dw, float* db) {
    __shared__ double s[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
    pdl_wait();
    double v = 0.0;
    if (c < Ch)
#pragma unroll 8
        for (long long i = threadIdx.y; i < count; i += 32) v += part[(i * 2 + which) * Ch + c];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0 && c < Ch) {
        for (int i = 1; i < 32; ++i) v += s[i][threadIdx.x];
        (which ? db : dw)[c] = (float)v;
    }
}

// ---- samples of several positions -------------------------------------------------------------------------------------
// A CTA has one slice of one sample; thread = (row of TR, VEC channels), channels in blocks of SLICE_THR * VEC where a row is wider than
// the CTA.
// CTAs per SM.  With the 56 and 80 registers a thread that leaves, the second pass spills 72 bytes forward and 156 backward in its
// 16-byte BF16 form, the first pass next to nothing
__host__ __device__ constexpr int slice_ctas(bool bwd) { return bwd ? 2 : 3; }
struct Slice {
    long long n, i, s0, s1;
    __device__ __forceinline__ Slice(long long S, int slices, long long len) {
        n = blockIdx.x / slices;
        i = blockIdx.x % slices;
        s0 = i * len;
        s1 = min(S, s0 + len);
    }
};
// A thread's rows of a slice, every TR-th, VEC channels each: f(row, x, dy).  The next U rows are on their way while U are used (a load
// of x would not pass a store to y by itself), the first ones from the constructor on.
template <typename T, int VEC, bool TWO, int U>
struct Rows {
    const T *X, *D;
    long long s, s1;
    int TR, Ch;
    Raw<T, VEC> nx[U], nd[U];
    __device__ __forceinline__ Rows(const T* X, const T* D, const Slice& sl, int tr, int TR, int Ch) : X(X), D(D), s(sl.s0 + tr), s1(sl.s1), TR(TR), Ch(Ch) { request(s); }
    __device__ __forceinline__ void request(long long at) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u * TR < s1) {
                nx[u] = load_raw<T, VEC>(X + (size_t)(at + u * TR) * Ch);
                if (TWO) nd[u] = load_raw<T, VEC>(D + (size_t)(at + u * TR) * Ch);
            }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) {
        for (; s < s1; s += U * TR) {
            Raw<T, VEC> rx[U], rd[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = nx[u];
                if (TWO) rd[u] = nd[u];
            }
            request(s + U * TR);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * TR < s1) {
                    float x[VEC], dy[VEC];
                    unpack(rx[u], x);
                    if (TWO) unpack(rd[u], dy);
                    f(s + u * TR, x, dy);
                }
        }
    }
};
// rows in flight, what registers allow: [4, 8191, 768] BF16 in 32 groups, sums of the backward 29 us with one and 37 with two; its second
// pass 31 with two and 33 with one
template <int VEC> constexpr int rows_ahead(bool two) { return VEC <= 2 ? 4 : VEC == 4 || !two ? 2 : 1; }
// scratch: [N * slices][2][Ch] numbers of the channels, then [N][G][slices][2] numbers of the groups
__device__ __forceinline__ float* group_part(const Args& a) { return a.part + (size_t)a.N * a.slices * 2 * a.Ch; }

// Sums s1 of x - b and s2 of (x - b)^2 over k rows, p = -b, become those about the rows' mean: however far the first row lies from
// the others, what follows is added about their middle.
template <int VEC>
__device__ __forceinline__ void about_mean(float (&p)[VEC], float (&s1)[VEC], float (&s2)[VEC], float k) {
    const float inv = 1.f / k;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const float to = fmaf(-inv, s1[i], p[i]), e = p[i] - to;
        s2[i] = fmaf(-e, fmaf(-k, e, 2.f * s1[i]), s2[i]);
        s1[i] = fmaf(-k, e, s1[i]);
        p[i] = to;
    }
}

// MODE 0: per thread and channel the mean less the slice's first row x0 and the sum of squared deviations, joined over the threads, and
// from them a group's; 1: sums of dz x^ and dz, and over a group's channels w times those
template <typename T, int VEC, int MODE>
__global__ void __launch_bounds__(SLICE_THR, slice_ctas(MODE)) group_norm_sums_kernel(const Args a) {
    extern __shared__ float sm[];                  // [2][TR][TC * VEC]
    const int cols = a.Ch / VEC, TC = min(cols, SLICE_THR), TR = SLICE_THR / TC;
    const int tc = threadIdx.x % TC, tr = threadIdx.x / TC, Cg = a.Ch / a.G;
    const Slice sl(a.S, a.slices, a.len);
    const long long n = sl.n;
    const int m = (int)(sl.s1 - sl.s0);            // (at most SUM_ROWS * SLICE_THR)
    const double inv_m = 1.0 / m;
    pdl_wait();
    const T* X = static_cast<const T*>(a.x) + (size_t)n * a.S * a.Ch;
    const T* D = static_cast<const T*>(a.dy) + (size_t)n * a.S * a.Ch;
    float* out = a.part + (size_t)blockIdx.x * 2 * a.Ch;
    const bool silu = a.act;
    for (int v0 = 0; v0 < cols; v0 += TC) {
        const int v = v0 + tc, c = v * VEC;
        const bool on = tr < TR && v < cols;
        float p[VEC], s1[VEC], s2[VEC], mu = 0.f, rs = 0.f;  // (a thread's channels are of one group)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s1[i] = s2[i] = 0.f;
        if (on) {
            Rows<T, VEC, MODE, rows_ahead<VEC>(MODE)> rows(X + c, D + c, sl, tr, TR, a.Ch);
            if (MODE == 0) {
                load<T, VEC>(X + (size_t)(sl.s0 + (tr < m ? tr : 0)) * a.Ch + c, p);
                vmul(p, p, Same{-1.f});
            } else {
                mu = a.mean[n * a.G + c / Cg];
                rs = a.rstd[n * a.G + c / Cg];
            }
            float w[VEC], b[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                w[i] = MODE && a.w ? a.w[c + i] : 1.f;
                b[i] = MODE && a.b ? a.b[c + i] : 0.f;
            }
            int k = 0;
            rows.each([&](long long, float (&x)[VEC], float (&dy)[VEC]) {
                if (MODE == 0) {
                    vadd(x, x, p);
                    vadd(s1, s1, x);
                    vfma(s2, x, x, s2);
                    if (++k >= 8 && (k & (k - 1)) == 0) about_mean(p, s1, s2, (float)k);
                } else {
                    float z[VEC];
                    vadd(x, x, Same{-mu});
                    vmul(x, x, Same{rs});
                    vfma(z, x, w, b);
                    act_grad<T>(dy, z, dy, silu);
                    vfma(s1, dy, x, s1);
                    vadd(s2, s2, dy);
                }
            });
            if (MODE == 0 && k > 0) {
                about_mean(p, s1, s2, (float)k);
                float x0[VEC];
                load<T, VEC>(X + (size_t)sl.s0 * a.Ch + c, x0);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    s1[i] = fmaf(1.f / k, s1[i], -p[i] - x0[i]);
                    s2[i] = s2[i] < 0.f ? 0.f : s2[i];  // (a NaN stays one)
                }
            }
        }
        if (v0) __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (tr < TR) {
                sm[tr * TC * VEC + tc * VEC + i] = s1[i];
                sm[(TR + tr) * TC * VEC + tc * VEC + i] = s2[i];
            }
        __syncthreads();
        // over the TR threads of a channel: a thread does that, or a warp where they are many
        const int L = TR > 32 ? 32 : 1, on_lane = threadIdx.x & (L - 1);
        for (int cc = threadIdx.x / L; cc < TC * VEC; cc += blockDim.x / L) {
            if (v0 * VEC + cc >= a.Ch) continue;
            double u = 0.0, q = 0.0, v = 0.0;
            for (int r = on_lane; r < TR; r += L) {
                const double x = sm[r * TC * VEC + cc], y = sm[(TR + r) * TC * VEC + cc];
                if (MODE == 0) {
                    const double w = x * ((m - r + TR - 1) / TR);  // (r < m, or the thread has had no row)
                    u += r < m ? w : 0.0;
                    q += r < m ? w * x : 0.0;
                } else {
                    u += x;
                }
                v += y;
            }
            lanes_sum(u, q, v, L);
            if (MODE == 0) {
                v += deviations(u, q, inv_m);
                u *= inv_m;
            }
            if (on_lane == 0) {
                out[v0 * VEC + cc] = sm[cc] = (float)u;
                out[(size_t)a.Ch + v0 * VEC + cc] = sm[TR * TC * VEC + cc] = (float)v;
            }
        }
    }
    __syncthreads();
    // a row as wide as one block of channels is still in shared memory; else the CTA reads back what it wrote
    const float *sum1 = cols <= TC ? sm : out, *sum2 = cols <= TC ? sm + TR * TC * VEC : out + a.Ch;
    float* groups = group_part(a) + ((size_t)n * a.G * a.slices + sl.i) * 2;
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < a.G; g += blockDim.x >> 5) {
        double u = 0.0, q = 0.0, v = 0.0;
        const float *s1 = sum1 + g * Cg, *s2 = sum2 + g * Cg;
        if (MODE == 0) {  // about the first channel's mean
            const T* x0 = X + (size_t)sl.s0 * a.Ch + g * Cg;
            const double about = (double)ldf(x0) + s1[0];
            for (int c = lane; c < Cg; c += 32) {
                const double d = (double)ldf(x0 + c) + s1[c] - about;
                u += d;
                q += d * d;
                v += s2[c];
            }
            lanes_sum(u, q, v, 32);
            v += m * deviations(u, q, a.inv_Cg);
            u = about + u * a.inv_Cg;
        } else {
            for (int c = lane; c < Cg; c += 32) {
                const double w = a.w ? a.w[g * Cg + c] : 1.f;
                v += w * s1[c];
                u += w * s2[c];
            }
            lanes_sum(u, q, v, 32);
        }
        if (lane == 0) *reinterpret_cast<float2*>(groups + (size_t)g * a.slices * 2) = make_float2((float)u, (float)v);
    }
}

template <typename T, int VEC, bool BWD>
__global__ void __launch_bounds__(SLICE_THR, slice_ctas(BWD)) group_norm_apply_kernel(const Args a) {
    const int cols = a.Ch / VEC, TC = min(cols, SLICE_THR), TR = SLICE_THR / TC;
    const int tc = threadIdx.x % TC, tr = threadIdx.x / TC, Cg = a.Ch / a.G;
    const Slice sl(a.S, a.cuts, a.span);
    const long long n = sl.n;
    extern __shared__ float stat[];                // [G][2]: mean, rstd; backward: m1, m2
    pdl_wait();
    const T* X = static_cast<const T*>(a.x) + (size_t)n * a.S * a.Ch;
    const T* D = static_cast<const T*>(a.dy) + (size_t)n * a.S * a.Ch;
    T* Y = static_cast<T*>(BWD ? a.dx : a.y) + (size_t)n * a.S * a.Ch;
    Rows<T, VEC, BWD, rows_ahead<VEC>(false)> rows(X + tc * VEC, D + tc * VEC, sl, tr < TR ? tr : 0, TR, a.Ch);
    {   // the sample's slices, a warp per group; means about the first slice's
        const float2* groups = reinterpret_cast<const float2*>(group_part(a)) + (size_t)n * a.slices * a.G;  // [G][slices]
        const int lane = threadIdx.x & 31;
        const double rows = (double)a.len, tail = (double)(a.S - (long long)(a.slices - 1) * a.len), inv = a.inv_S * a.inv_Cg;
        for (int g = threadIdx.x >> 5; g < a.G; g += blockDim.x >> 5) {
            const float2* of = groups + (size_t)g * a.slices;
            const double u0 = BWD ? 0.0 : of[0].x;
            double u = 0.0, q = 0.0, v = 0.0;
#pragma unroll 4
            for (int i = lane; i < a.slices; i += 32) {
                const float2 p = of[i];
                if (BWD) {
                    u += p.x;
                } else {
                    const double d = p.x - u0, w = d * (i == a.slices - 1 ? tail : rows);
                    u += w;
                    q += w * d;
                }
                v += p.y;
            }
            lanes_sum(u, q, v, 32);
            if (!BWD) {
                v += Cg * deviations(u, q, a.inv_S);
                u = u0 + u * a.inv_S;
            }
            if (lane == 0) {
                stat[2 * g] = (float)(BWD ? u * inv : u);
                stat[2 * g + 1] = BWD ? (float)(v * inv) : 1.f / sqrtf((float)(v * inv) + a.eps);
                if (!BWD && sl.s0 == 0) {
                    a.mean[n * a.G + g] = stat[2 * g];
                    a.rstd[n * a.G + g] = stat[2 * g + 1];
                }
            }
        }
        __syncthreads();
    }
    if (tr >= TR) return;
    const bool silu = a.act;
    for (int v = tc; v < cols; v += TC) {
        const int c = v * VEC;
        const int g = c / Cg;  // (a thread's channels are of one group)
        const float mu = BWD ? a.mean[n * a.G + g] : stat[2 * g], rs = BWD ? a.rstd[n * a.G + g] : stat[2 * g + 1];
        // dx = (rstd w) dz + (x - mean) (-rstd^2 m2) - rstd m1
        const float k1 = BWD ? -rs * stat[2 * g] : 0.f, k2 = BWD ? -rs * rs * stat[2 * g + 1] : 0.f;
        float w[VEC], b[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            w[i] = rs * (a.w ? a.w[c + i] : 1.f);
            b[i] = a.b ? a.b[c + i] : 0.f;
        }
        if (v != tc) rows = Rows<T, VEC, BWD, rows_ahead<VEC>(false)>(X + c, D + c, sl, tr, TR, a.Ch);
        rows.each([&](long long s, float (&x)[VEC], float (&dy)[VEC]) {
            float y[VEC];
            float d[VEC], z[VEC];
            vadd(d, x, Same{-mu});
            vfma(z, d, w, b);
            if (BWD) {
                act_grad<T>(y, z, dy, silu);
                vfma(d, d, Same{k2}, Same{k1});
                vfma(y, y, w, d);
            } else {
                act<T>(y, z, silu);
            }
            store<T, VEC>(Y + (size_t)s * a.Ch + c, y);
        });
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------
static bool by_rows(long long S, int Ch, int G) { return S == 1 && Ch / G <= ROWS_MAX; }

// Slices of a sample in the second pass: as many as are resident over all samples, of at least 8 rows, all but the last of the same
// length.  In the first pass the same ones, or shorter where a thread would add up more than SUM_ROWS rows (with one channel an access).
static void cut(Args& a, bool bwd) {
    a.inv_S = 1.0 / a.S;
    a.inv_Cg = (double)a.G / a.Ch;
    long long want = (long long)slice_ctas(bwd) * sm_count() / a.N, most = (a.S + 7) / 8;
    if (want > most) want = most;
    if (want > MAX_SLICES) want = MAX_SLICES;
    if (want < 1) want = 1;
    a.span = (a.S + want - 1) / want;
    a.cuts = (int)((a.S + a.span - 1) / a.span);
    const long long most_rows = (long long)SUM_ROWS * (SLICE_THR / (a.Ch < SLICE_THR ? a.Ch : SLICE_THR));
    a.len = a.span < most_rows ? a.span : most_rows;
    const long long slices = (a.S + a.len - 1) / a.len;
    a.slices = slices < 0x7fffffffLL ? (int)slices : 0x7fffffff;  // (refused)
}

struct RowsGrid { int L; long long ctas, step; };
static RowsGrid rows_grid(long long N, int Ch, int G, int vec, bool bwd) {
    const int Cg = Ch / G;
    RowsGrid r;
    r.L = 1;
    while (r.L < 32 && r.L * vec < Cg) r.L *= 2;
    const long long per = NTHR / r.L, need = (N * G + per - 1) / per;
    long long most = (bwd ? 3 : 4) * (long long)sm_count();
    const long long steps = bwd ? (N + SUM_ROWS - 1) / SUM_ROWS : 1;  // a slot adds at most SUM_ROWS rows to its dw, db
    const long long least = (steps * G + per - 1) / per;              // and every group has a slot
    if (most < least) most = least;
    r.ctas = need < least ? least : need < most ? need : most;
    r.step = r.ctas * per / G;
    return r;
}
// elements per access: 16 bytes where every group starts on 16 bytes, else two or one
static int vec_of(int unit, int es, const void* x, const void* y, const void* z) {
    const int full = 16 / es;
    const uintptr_t at = (uintptr_t)x | (uintptr_t)y | (uintptr_t)z;
    return unit % full == 0 && (at & 15) == 0 ? full : unit % 2 == 0 && (at & (2 * es - 1)) == 0 ? 2 : 1;
}

template <typename T, int VEC, bool BWD>
static cudaError_t rows_launch(const Args& a, cudaStream_t s) {
    const RowsGrid r = rows_grid(a.N, a.Ch, a.G, VEC, BWD);
    const int nv = (a.Ch / a.G + r.L * VEC - 1) / (r.L * VEC);
    cudaError_t e;
    if (nv <= 1) e = launch_dependent(group_norm_rows_kernel<T, VEC, 1, BWD>, dim3((unsigned)r.ctas), NTHR, 0, s, a, r.L);
    else if (nv <= 4) e = launch_dependent(group_norm_rows_kernel<T, VEC, 4, BWD>, dim3((unsigned)r.ctas), NTHR, 0, s, a, r.L);
    else if (VEC > 1 && nv <= 32 / VEC) e = launch_dependent(group_norm_rows_kernel<T, VEC, 32 / VEC, BWD>, dim3((unsigned)r.ctas), NTHR, 0, s, a, r.L);
    else e = launch_dependent(group_norm_rows_kernel<T, VEC, VEC == 1 ? 32 : 1, BWD>, dim3((unsigned)r.ctas), NTHR, 0, s, a, r.L);
    if (e == cudaSuccess && BWD && a.dw)
        e = launch_dependent(group_norm_params_kernel, dim3((a.Ch + 31) / 32, 2), dim3(32, 32), 0, s, (const float*)a.part, r.step, a.Ch, a.dw, a.db);
    return e;
}

template <typename T, int VEC, bool BWD>
static cudaError_t slices_launch(const Args& a, cudaStream_t s) {
    const dim3 grid((unsigned)(a.N * a.slices)), grid2((unsigned)(a.N * a.cuts));
    const int cols = a.Ch / VEC, TC = cols < SLICE_THR ? cols : SLICE_THR, TR = SLICE_THR / TC, threads = (TC * TR + 31) / 32 * 32;
    const size_t smem = (size_t)2 * TR * TC * VEC * sizeof(float), stat = (size_t)2 * a.G * sizeof(float);
    cudaError_t e = stat > 48 * 1024 ? allow_smem(group_norm_apply_kernel<T, VEC, BWD>, GROUPS_MAX * 8) : cudaSuccess;
    if (e == cudaSuccess) e = launch_dependent(group_norm_sums_kernel<T, VEC, BWD ? 1 : 0>, grid, threads, smem, s, a);
    if (e == cudaSuccess) e = launch_dependent(group_norm_apply_kernel<T, VEC, BWD>, grid2, threads, stat, s, a);
    if (e == cudaSuccess && BWD && a.dw)
        e = launch_dependent(group_norm_params_kernel, dim3((a.Ch + 31) / 32, 2), dim3(32, 32), 0, s, (const float*)a.part, a.N * a.slices, a.Ch, a.dw, a.db);
    return e;
}

template <typename T, bool BWD>
static cudaError_t dispatch(const Args& a, cudaStream_t s) {
    constexpr int FULL = 16 / sizeof(T);
    const bool rows = by_rows(a.S, a.Ch, a.G);
    const int vec = vec_of(a.Ch / a.G, sizeof(T), a.x, BWD ? a.dx : a.y, a.dy);
    if (rows) return vec == FULL ? rows_launch<T, FULL, BWD>(a, s) : vec == 2 ? rows_launch<T, 2, BWD>(a, s) : rows_launch<T, 1, BWD>(a, s);
    return vec == FULL ? slices_launch<T, FULL, BWD>(a, s) : vec == 2 ? slices_launch<T, 2, BWD>(a, s) : slices_launch<T, 1, BWD>(a, s);
}

static int check(const Args& a, int dtype) {
    if (dtype != KDA_DTYPE_F32 && dtype != KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
    if (a.N <= 0 || a.S <= 0 || a.Ch <= 0 || a.Ch > 1 << 30 || a.G <= 0 ||  // (two rows of channels are counted in 32 bits)
         a.Ch % a.G || !(a.eps >= 0.f)) return KDA_ERR_SHAPE;
    // the groups' numbers in shared memory, and grids of samples x slices
    if (!by_rows(a.S, a.Ch, a.G)) {
        if (a.G > GROUPS_MAX) return KDA_ERR_SHAPE;
        Args b = a;
        cut(b, false);  // (no fewer slices than in the backward)
        if (b.slices == 0x7fffffff || (b.slices > b.cuts ? b.slices : b.cuts) > 0x7fffffffLL / a.N) return KDA_ERR_SHAPE;
    }
    if (by_rows(a.S, a.Ch, a.G) && a.N > (1LL << 40) / a.G) return KDA_ERR_SHAPE;
    return KDA_OK;
}
static size_t scratch(long long N, long long S, int Ch, int G, int es, bool bwd) {
    if (by_rows(S, Ch, G)) {
        if (!bwd) return 0;
        long long step = 0;  // (the element width is known only with the pointers)
        for (int vec : {1, 2, 16 / es})
            if ((Ch / G) % vec == 0) {
                const long long n = rows_grid(N, Ch, G, vec, true).step;
                if (n > step) step = n;
            }
        return (size_t)step * 2 * Ch * sizeof(float);
    }
    Args a = {};
    a.N = N; a.S = S; a.Ch = Ch; a.G = G;
    cut(a, bwd);
    return (size_t)N * a.slices * 2 * (Ch + G) * sizeof(float);
}

}  // namespace gn
}  // namespace kda

using namespace kda;

extern "C" int kda_group_norm_scratch_bytes(int64_t N, int64_t S, int32_t channels, int32_t groups, int32_t dtype, size_t* fwd_bytes,
                                            size_t* bwd_bytes) {
    gn::Args a = {};
    a.N = N; a.S = S; a.Ch = channels; a.G = groups;
    if (const int rc = gn::check(a, dtype)) return rc;
    const int es = dtype == KDA_DTYPE_F32 ? 4 : 2;
    if (fwd_bytes) *fwd_bytes = gn::scratch(N, S, channels, groups, es, false);
    if (bwd_bytes) *bwd_bytes = gn::scratch(N, S, channels, groups, es, true);
    return KDA_OK;
}

extern "C" int kda_group_norm_fwd(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                                  float* scratch, int64_t N, int64_t S, int32_t channels, int32_t groups, float eps, int32_t silu,
                                  int32_t dtype, void* stream) {
    gn::Args a = {};
    a.x = x; a.y = y; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd; a.part = scratch;
    a.N = N; a.S = S; a.Ch = channels; a.G = groups; a.act = silu; a.eps = eps;
    if (const int rc = gn::check(a, dtype)) return rc;
    if (!x || !y || (!gn::by_rows(S, channels, groups) && (!mean || !rstd || !scratch))) return KDA_ERR_NULL;
    gn::cut(a, false);
    const cudaError_t e = dtype == KDA_DTYPE_F32 ? gn::dispatch<float, false>(a, (cudaStream_t)stream) : gn::dispatch<gn::bf16, false>(a, (cudaStream_t)stream);
    return e == cudaSuccess ? KDA_OK : fail_cuda(e);
}

extern "C" int kda_group_norm_bwd(const void* x, const float* weight, const float* bias, const float* mean, const float* rstd,
                                  const void* dy, void* dx, float* dweight, float* dbias, float* scratch, int64_t N, int64_t S,
                                  int32_t channels, int32_t groups, float eps, int32_t silu, int32_t dtype, void* stream) {
    gn::Args a = {};
    a.x = x; a.dy = dy; a.dx = dx; a.w = weight; a.b = bias; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.dw = dweight; a.db = dbias; a.part = scratch;
    a.N = N; a.S = S; a.Ch = channels; a.G = groups; a.act = silu; a.eps = eps;
    if (const int rc = gn::check(a, dtype)) return rc;
    const bool rows = gn::by_rows(S, channels, groups);
    if (!x || !dy || !dx || (!rows && (!mean || !rstd || !scratch)) || (dweight && (!dbias || !scratch)) || (!dweight && dbias)) return KDA_ERR_NULL;
    gn::cut(a, true);
    const cudaError_t e = dtype == KDA_DTYPE_F32 ? gn::dispatch<float, true>(a, (cudaStream_t)stream) : gn::dispatch<gn::bf16, true>(a, (cudaStream_t)stream);
    return e == cudaSuccess ? KDA_OK : fail_cuda(e);
}
