// Gated delta rule with one decay per value head: shared definitions of its kernels.
//
// With one decay per head the pairwise decays of a chunk are numbers, not vectors: q k^T and k k^T are plain products of the
// rows as they arrive, and decay, beta and the rows' 1 / norm multiply the results in FP32.  So in BF16 mode every product has
// an operand that BF16 holds exactly (q, k, do) or two computed ones (T, V', S, ...).  Computed operands are BF16 in up to three
// parts, x = p0 + p1 + p2 to 2^-24, and a product of parts i and j is taken where i + j < 3: from tensor cores with FP32 accumulators
// results that are 1e-7 to 4e-7 of their norm from 64 bits on mma.sync, and on tcgen05, whose accumulators truncate, 2e-7 to 6e-7 for
// states and up to 1.7e-6 for dg and dbeta.  Where only a BF16 output can see the difference two parts do (2^-17: three outputs in a
// thousand are rounded to the neighbour of the nearest BF16 number).  FP32 tensors go the same way with three parts for q, k, v, do as well.
#pragma once

#include "kda_common.cuh"
#include "kda_tc.cuh"

namespace kda {
namespace gdr {

using namespace tc;
using bf16 = __nv_bfloat16;

constexpr int NBLK = 10;           // 16 x 16 blocks of a lower triangular 64 x 64 matrix
constexpr int BLK = 256;           // elements of one
constexpr int TRI = NBLK * BLK;    // elements of one part of such a matrix
constexpr int AUX = 12 * C;        // floats of a unit's per-row numbers
// e^G, e^(G_last - G), beta, 1/|q|, 1/|k|, G in two floats, [A_LAST][0] = e^G_last; and the factors that the walks use:
// beta e^G / |k|, e^(G_last - G) / |k|, scale e^G / |q|, e^G / |k|
enum { A_GAM, A_FALL, A_BETA, A_RQ, A_RK, A_GHI, A_GLO, A_LAST, A_BGK, A_FK, A_OQ, A_GK };
constexpr int SQ = C * C;          // elements of one part of a 64 x 64 matrix in core-matrix order (cm_idx)
// BF16 with 128 key channels and value columns goes on tcgen05; T and A are then whole matrices in core-matrix order
__host__ __device__ __forceinline__ bool on_tc(const KdaGdrParams& p) { return p.dtype == KDA_DTYPE_BF16 && p.dk == 128 && p.dv == 128; }
constexpr float G_ZERO = -104.f;   // e^g is 0 in FP32 below
constexpr float G_MIN = -1000.f;   // log decays below count as this: e^-1000 is 0 in FP32, and sums of 64 stay finite

__host__ __device__ __forceinline__ constexpr int blk(int I, int J) { return I * (I + 1) / 2 + J; }

// per (chunk, value head) unit, byte offsets
struct Layout {
    size_t aux, T, A, segE, segX, total_nosave, S0, Vn, Tb, total;  // workspace
    size_t dS, Y, part, dqk, segF, bwd_total;                       // backward scratch
    int segs, seg_len;                                              // segments of a sequence (1: none) and their chunks
};
inline int longest(const KdaGdrParams& p) {  // chunks of the longest sequence, 0: not known
    return p.cu_seqlens ? p.max_chunks : (p.T + C - 1) / C;
}
// Segments of the longest sequence in the walks on tcgen05 (gdr_tc.cu).  A walk is a chain of chunks; where walks are few, or one is
// much longer than its share, sequences are cut into segments of equal length that are walked twice: from zero (and from the identity,
// for what a segment does to the state that it is entered with), and again from the states that follow.  Estimated with 3.2 us for a
// chunk without outputs and 3.7 with, 2.6 us for a border and 12 us for the launches: equal sequences go in waves, packed ones fill the
// SMs up to half a segment.  8 walks of 512 chunks, forward: 2312 -> 485 us.  The estimate is rough: a chunk takes 3.8 us without
// outputs and 4.5 to 6.5 with (gdr_tc.cu), the backward is not estimated by itself, and of packed documents it takes the first pass for
// free where most of them end in their first segment (24 571 tokens of 12 documents, 8 heads: two segments, a first pass of 165 us).
// It tends to too few segments.
inline int segment_count(const KdaGdrParams& p) {
    if (!on_tc(p)) return 1;
    const int nc = longest(p), sms = sm_count();
    if (nc < 4) return 1;
    const double walks = (double)p.N * p.HV, all = (double)p.NT * p.HV;
    auto waves = [&](double ctas, double len) { return (double)(long long)((ctas + sms - 1) / sms) * len; };
    auto fill = [&](double chunks, double len) { return chunks <= 0 ? 0.0 : chunks / sms + len / 2 > len ? chunks / sms + len / 2 : len; };
    double best = 3.7 * (p.cu_seqlens ? fill(all, nc) : waves(walks, nc));
    int n = 1;
    for (int s = 2; s <= nc / 2 && s <= 64; ++s) {
        const int len = (nc + s - 1) / s;
        const double t1 = p.cu_seqlens ? fill(2 * (all - 0.75 * walks * len), len) : waves(walks * (2 * s - 3), len),
                     t2 = p.cu_seqlens ? fill(all, len) : waves(walks * s, len), t = 3.2 * t1 + 3.7 * t2 + 2.6 * (s - 2) + 12.0;
        if (t < best) best = t, n = s;
    }
    // (segment buffers of 64 KB a segment and head)
    return walks * n > 8192 ? 1 : n;
}
inline Layout layout(const KdaGdrParams& p) {
    const size_t n = (size_t)p.NT * p.HV, mat = 3 * (on_tc(p) ? SQ : TRI) * 2;
    Layout l;
    l.segs = segment_count(p);
    l.seg_len = l.segs > 1 ? (longest(p) + l.segs - 1) / l.segs : 0x7fffffff;
    const size_t seg_bytes = l.segs > 1 ? (size_t)p.N * p.HV * l.segs * p.dk * p.dv * 4 : 0;
    size_t off = 0;
    l.aux = off; off = align256(off + n * AUX * 4);
    // (I + diag(beta) L)^-1 and scale (q k^T) D as three BF16 parts: blocks of the lower triangle in blk() order, rows swizzled as
    // tri_frag reads them; or (on_tc) [64][64] in core-matrix order of which only those blocks are written, the columns of T times
    // beta, and T itself for the backward
    l.T = off;   off = align256(off + n * mat);
    l.A = off;   off = align256(off + n * mat);
    l.segE = off; off += seg_bytes;  // [sequence, head][segment][dk][dv]: state at the segment's end
    l.segX = off; off += seg_bytes;  // the same of the identity: S_end = X S_begin + E
    l.total_nosave = off;
    // state at the chunk's start [dk][dv] and V' [64][dv], on_tc in the order of rec_idx()
    l.S0 = off;  off = align256(off + n * p.dk * p.dv * 4);
    l.Vn = off;  off = align256(off + n * C * p.dv * 4);
    l.Tb = off;  if (on_tc(p)) off = align256(off + n * mat);
    l.total = off;
    off = 0;
    l.dS = off;   off = align256(off + n * p.dk * p.dv * 4); // gradient of the state at the chunk's end, as S0
    l.Y = off;    off = align256(off + n * C * p.dv * 4);    // T^T dV' [64][dv]
    l.part = off; off = align256(off + n * 2 * 4);           // this unit's share of dA_log and ddt_bias
    l.dqk = off;  if (p.HV != p.H) off = align256(off + n * 2 * C * p.dk * 4);  // shared key heads: this value head's share of dq, dk
    l.segF = off; off += seg_bytes;  // gradient of the state at the segment's start
    l.bwd_total = off;
    return l;
}

// Records of the transposed walks: FP32 [128 value columns][cols], 16 value columns at a time, each [16][cols] in core-matrix order:
// what one K-step of a product over the value columns reads lies together, eight consecutive columns as one piece of 32 bytes.
__host__ __device__ __forceinline__ int rec_idx(int e, int col, int cols) { return (e >> 4) * 16 * cols + cm_idx(e & 15, col, cols); }

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// Fragments of a row-major tile X with rows of LD elements (LD = 8 mod 16 keeps the eight rows of a matrix in different banks).
// a_frag: the 16 x 16 block of X at (r, c) as A.   a_frag_t: the block at (r, c) of X^T as A (X holds it at (c, r)).
// b_frag: X holds B^T, rows n: 16 columns n.. of B, k..k+16.   b_frag_t: X holds B, rows k.   Both give two column tiles (b[0..1], b[2..3]).
template <int LD>
__device__ __forceinline__ void a_frag(uint32_t (&f)[4], uint32_t x, int r, int c, int lane) {
    ldsm(f, x + 2 * ((r + (lane & 15)) * LD + c + (lane >> 4) * 8));
}
template <int LD>
__device__ __forceinline__ void a_frag_t(uint32_t (&f)[4], uint32_t x, int r, int c, int lane) {
    ldsm_t(f, x + 2 * ((c + (lane & 7) + (lane >> 4) * 8) * LD + r + ((lane >> 3) & 1) * 8));
}
template <int LD>
__device__ __forceinline__ void b_frag(uint32_t (&f)[4], uint32_t x, int n, int k, int lane) {
    ldsm(f, x + 2 * ((n + (lane & 7) + (lane >> 4) * 8) * LD + k + ((lane >> 3) & 1) * 8));
}
template <int LD>
__device__ __forceinline__ void b_frag_t(uint32_t (&f)[4], uint32_t x, int n, int k, int lane) {
    ldsm_t(f, x + 2 * ((k + (lane & 7) + ((lane >> 3) & 1) * 8) * LD + n + (lane >> 4) * 8));
}
// 16 x 16 blocks of a lower triangular matrix as the workspace holds them: rows of 32 bytes whose halves change places in rows
// 4..7 and 12..15, so that eight rows of a matrix lie in different banks
__device__ __forceinline__ int tri_idx(int r, int c) { return r * 16 + ((((c >> 3) ^ (r >> 2)) & 1) << 3) + (c & 7); }
__device__ __forceinline__ void tri_frag(uint32_t (&f)[4], uint32_t x, int b, int lane) {
    ldsm(f, x + 2 * (b * BLK + tri_idx(lane & 15, (lane >> 4) * 8)));
}
__device__ __forceinline__ void tri_frag_t(uint32_t (&f)[4], uint32_t x, int b, int lane) {
    ldsm_t(f, x + 2 * (b * BLK + tri_idx((lane & 7) + (lane >> 4) * 8, ((lane >> 3) & 1) * 8)));
}

// Products of the parts of one A block and two column tiles of B.  The tensor core truncates at every accumulation: several products
// are summed from zero, the smallest first, and added in FP32, so that one truncation of a K-step's own size is left of each
// (FP32 tensors: dk 1.8e-6 -> 1.8e-7 of its norm from 64 bits).
template <int PA, int PB, int ORD, int NT>
__device__ __forceinline__ void mma_parts(float (&acc)[NT][4], int pair, const uint32_t (&a)[PA][4], const uint32_t (&b)[PB][4]) {
    if constexpr (PA * PB == 1) {
        mma(acc[2 * pair], a[0], b[0][0], b[0][1]);
        mma(acc[2 * pair + 1], a[0], b[0][2], b[0][3]);
    } else {
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int o = ORD - 1; o >= 0; --o)
#pragma unroll
            for (int j = PB - 1; j >= 0; --j)
                if (o - j >= 0 && o - j < PA) {
                    mma(s[0], a[o - j], b[j][0], b[j][1]);
                    mma(s[1], a[o - j], b[j][2], b[j][3]);
                }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[2 * pair][i] += s[0][i];
            acc[2 * pair + 1][i] += s[1][i];
        }
    }
}

template <int P>
__device__ __forceinline__ void split(float x0, float x1, uint32_t (&w)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (i + 1 < P) {  // (packed: x - p)
            const float2 r = __ffma2_rn(make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), make_float2(-1.f, -1.f), make_float2(x0, x1));
            x0 = r.x;
            x1 = r.y;
        }
    }
}
// two neighbouring elements into the P part tiles at element offset idx
template <int P>
__device__ __forceinline__ void put(bf16* tile, int part, int idx, float x0, float x1) {
    uint32_t w[P];
    split(x0, x1, w);
#pragma unroll
    for (int i = 0; i < P; ++i) *reinterpret_cast<uint32_t*>(tile + i * part + idx) = w[i];
}
template <int P>
__device__ __forceinline__ void put4(bf16* tile, int part, int idx, const float4& x) {
    uint32_t a[P], b[P];
    split(x.x, x.y, a);
    split(x.z, x.w, b);
#pragma unroll
    for (int i = 0; i < P; ++i) *reinterpret_cast<uint2*>(tile + i * part + idx) = make_uint2(a[i], b[i]);
}
// two neighbouring elements of a tile in P parts
template <int P>
__device__ __forceinline__ float2 get2(const bf16* tile, int part, int idx) {
    float2 x = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = P - 1; i >= 0; --i) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + i * part + idx);
        x.x += __uint_as_float(w << 16);
        x.y += __uint_as_float(w & 0xffff0000u);
    }
    return x;
}

template <typename T> struct In;
template <> struct In<bf16> { static constexpr int P = 1, PO = 2; };   // parts of inputs; of computed operands behind a 16-bit output
template <> struct In<float> { static constexpr int P = 3, PO = 3; };

// rows of COLS elements, `stride` apart in memory, into row-major part tiles; rows from `rows` on are zero
template <int COLS, int LD, int NTHR>
__device__ __forceinline__ void load_tile(bf16* dst, const bf16* src, size_t stride, int rows, int tid) {
    constexpr int W = COLS / 8;
#pragma unroll
    for (int i = tid; i < C * W; i += NTHR) {
        const int r = i / W, c = i % W * 8;
        const bool in = r < rows;
        cp_async16_z(dst + r * LD + c, src + (in ? r * stride + c : 0), in);
    }
}
template <int COLS, int LD, int NTHR>
__device__ __forceinline__ void load_tile(bf16* dst, const float* src, size_t stride, int rows, int tid) {
    constexpr int W = COLS / 4;
#pragma unroll 4
    for (int i = tid; i < C * W; i += NTHR) {
        const int r = i / W, c = i % W * 4;
        const float4 x = r < rows ? *reinterpret_cast<const float4*>(src + r * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        put4<3>(dst, C * LD, r * LD + c, x);
    }
}
// 64 rows of COLS elements, `stride` apart in memory, into core-matrix order (SWZ: two halves of 64 columns with 128-byte swizzle,
// swz_bf16).  A lane has row lane mod 8 of every block of eight and, of four chunks of 16 bytes, one; warps share the column blocks.
// Addresses advance by constants: two instructions a copy.
template <int COLS, int NTHR, bool SWZ = false>
__device__ __forceinline__ void load_cm(bf16* dst, const bf16* src, size_t stride, int rows, int tid) {
    static_assert(!SWZ || COLS == 128, "two halves");
    constexpr int NW = NTHR / 32, CG = COLS / 32;
    static_assert(CG % NW == 0, "whole column blocks per warp");
    const int lane = tid & 31, w = tid >> 5, r = lane & 7, c = lane >> 3;
#pragma unroll
    for (int g = 0; g < CG / NW; ++g) {
        const int cc = ((g * NW + w) * 4 + c) * 8;
        const bf16* s = src + (size_t)r * stride + cc;
        const uint32_t d = smem_u32(dst + (SWZ ? swz_bf16(r, cc) : cm_idx(r, cc, COLS)));
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const bool in = 8 * b + r < rows;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + b * (SWZ ? 1024 : COLS * 16)), "l"(in ? s : src), "r"(in ? 16 : 0) : "memory");
            s += 8 * stride;
        }
    }
}
// `count` 16-byte words
template <int NTHR>
__device__ __forceinline__ void load_words(bf16* dst, const bf16* src, int count, int tid) {
    for (int i = tid; i < count; i += NTHR) cp_async16_z(dst + 8 * i, src + 8 * i, true);
}

__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load2(const bf16* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void store2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store2(bf16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }

__device__ __forceinline__ float load_g(const KdaGdrParams& p, const void* x, size_t i) {
    return p.g_dtype == KDA_DTYPE_F32 ? static_cast<const float*>(x)[i] : __bfloat162float(static_cast<const bf16*>(x)[i]);
}
__device__ __forceinline__ void store_g(const KdaGdrParams& p, void* x, size_t i, float v) {
    if (p.g_dtype == KDA_DTYPE_F32) static_cast<float*>(x)[i] = v;
    else static_cast<bf16*>(x)[i] = __float2bfloat16_rn(v);
}
// log decay of a token (a NaN stays one)
__device__ __forceinline__ float log_decay(const KdaGdrParams& p, size_t i, int h) {
    float g = load_g(p, p.g, i);
    if (p.flags & KDA_FLAG_GATE) g = -expf(p.A_log[h]) * softplus_f(g + (p.dt_bias ? p.dt_bias[h] : 0.f));
    return g < G_MIN ? G_MIN : g;
}
// the three index tables take the same fields as KdaParams
__device__ __forceinline__ size_t state_at(const KdaGdrParams& p, int d, int e) {
    return (p.flags & KDA_FLAG_STATE_V_FIRST) ? (size_t)e * p.dk + d : (size_t)d * p.dv + e;
}

// Gradients of the log decays from those of their running sums G; a lane has two neighbouring rows.  d: the rows' gradients without the
// share of the chunk's end, which is h_j at the last row and -h_j at row j itself for every row j.  Summed from row t on, the h_j of the
// rows before t remain: they are added up as such, not as what is left of -h_j + h_j.  end = e^G_last <S0, dS>.
__device__ __forceinline__ float2 decay_gradients(const double (&d)[2], const double (&h)[2], double end, int lane) {
    double after = d[0] + d[1], before = h[0] + h[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double a = __shfl_down_sync(0xffffffffu, after, o), b = __shfl_up_sync(0xffffffffu, before, o);
        if (lane + o < 32) after += a;
        if (lane >= o) before += b;
    }
    after = __shfl_down_sync(0xffffffffu, after, 1);
    before = __shfl_up_sync(0xffffffffu, before, 1);
    if (lane == 31) after = 0.0;
    if (lane == 0) before = 0.0;
    const double r1 = after + d[1], r0 = r1 + d[0];
    return make_float2((float)(r0 + (before + end)), (float)(r1 + (before + h[0] + end)));
}
// the gradients of g, beta and a unit's share of those of A_log, dt_bias from those of log decay and beta; a lane has two neighbouring rows
__device__ __forceinline__ void gate_gradients(const KdaGdrParams& p, const Layout& lay, const ChunkInfo& ci, size_t unit, int h, float dg0, float dg1,
                                               float db0, float db1, float be0, float be1, int lane) {
    float dA = 0.f, dbias = 0.f;
    const bool gate = p.flags & KDA_FLAG_GATE;
    const float eA = gate ? expf(p.A_log[h]) : 0.f, bias = gate && p.dt_bias ? p.dt_bias[h] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        if (r >= ci.len) continue;
        const size_t at = (size_t)(ci.tok0 + r) * p.HV + h;
        float d = i ? dg1 : dg0, b = i ? db1 : db0;
        const float be = i ? be1 : be0;
        const float a = load_g(p, p.g, at) + bias, decay = gate ? -eA * softplus_f(a) : a;
        // nothing passes through a token whose decay is 0: what d has there is the rounding of sums that cancel (a NaN is left)
        if (decay < G_ZERO && d == d) d = 0.f;
        if (gate && d != 0.f) {  // (e^A_log may be infinite where d is 0)
            dA += d * fmaxf(decay, G_MIN);
            d *= -eA * (a > 20.f ? 1.f : sigmoid_f(a));
            dbias += d;
        }
        if (p.flags & KDA_FLAG_BETA_SIGMOID) b *= be * (1.f - be);
        store_g(p, p.grad_g, at, d);
        store_g(p, p.grad_beta, at, b);
    }
    if (gate) {
        dA = warp_sum(dA);
        dbias = warp_sum(dbias);
        if (lane == 0) *reinterpret_cast<float2*>(static_cast<char*>(p.bwd_scratch) + lay.part + unit * 8) = make_float2(dA, dbias);
    }
}
// 32 bytes at a time: eight floats
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store8(float* p, const float* x) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]),
                 "f"(x[6]), "f"(x[7]) : "memory");
}

}  // namespace gdr
}  // namespace kda
