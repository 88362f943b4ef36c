// Gated delta rule, the part of a chunk that needs no state: per key head the products q k^T and k k^T of the 64 rows, and for
// every value head of its group
//     A = scale (q^ k^T) D,  L = beta (k^ k^T) D strictly below the diagonal,  T = (I + L)^-1,     D_ij = e^(G_i - G_j)
// as records of three BF16 parts (the lower triangle's blocks), with the rows' e^G, e^(G_last - G), beta and 1 / norm.
//
// One CTA of four warps per (chunk, key head); warp w holds rows 16 w .. 16 w + 15 of both products in registers for all value
// heads.  G is summed in 64 bits and kept in two floats, so that a difference of two large sums still gives a decay to FP32.  The
// inverse goes by blocks: the four 16 x 16 diagonal blocks by substitution (a lane per column), then neighbours joined twice,
// T_21 = -T_22 (L_21 T_11), in FP32 multiply-adds.
//
// Bound by latency between its barriers and by issue slots: 16 x 2048 tokens of 6 heads (BF16, 128 channels) take 90 us, 64 KB of HBM traffic a unit
// at 2.1 TB/s.  The matrices take the place of the rows in shared memory, so that five CTAs fit an SM instead of three, the
// gates of up to four heads are summed while the rows are on their way, and most decays are products of a row's and a column's
// exponential: 116 us without the three.
#include "gdr.cuh"

namespace kda {
namespace gdr {

constexpr int LDL = 68;  // floats per row of L / T

template <typename T, int K>
__host__ __device__ constexpr int tiles_bytes() {
    constexpr int a = 2 * In<T>::P * C * (K + 8) * 2, b = (C * LDL + 32 * 36) * 4;
    return a > b ? a : b;
}

// squares of eight elements of a tile in P parts, in two sums
template <int P>
__device__ __forceinline__ float2 sum_sq(const bf16* tile, int part) {
    uint4 w[P];
#pragma unroll
    for (int i = 0; i < P; ++i) w[i] = *reinterpret_cast<const uint4*>(tile + i * part);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 x = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = P - 1; i >= 0; --i) {
            const uint32_t u = reinterpret_cast<const uint32_t*>(&w[i])[j];
            x.x += __uint_as_float(u << 16);
            x.y += __uint_as_float(u & 0xffff0000u);
        }
        s = __ffma2_rn(x, x, s);
    }
    return s;
}
// eight neighbouring elements into three part tiles
__device__ __forceinline__ void put8(bf16* tile, int part, int idx, const float (&x)[8]) {
    uint32_t w[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) split(x[2 * i], x[2 * i + 1], w[i]);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(tile + i * part + idx) = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
}

// Inverses of two neighbouring diagonal blocks of S = 16 R into that of the block of 2 S: T_21 = -T_22 (L_21 T_11).  Pair `pr`,
// thread q of it; Z [32][36].  (Nothing is above the diagonal, and of what is not in a diagonal block of 16 nothing is written.)
template <int R>
__device__ __forceinline__ void join(float* L, float* Z, int pr, int q) {
    constexpr int S = 16 * R, Q = S / 4;
    const int r = q / Q * R, c0 = q % Q * 4;
    float *low = L + (2 * S * pr + S) * LDL + 2 * S * pr, *z = Z + 16 * pr * 36;
    float2 acc[R][2];
    auto product = [&](const float* a, const float* b, int ldb, int m0, int m1) {
#pragma unroll
        for (int i = 0; i < R; ++i) acc[i][0] = acc[i][1] = make_float2(0.f, 0.f);
#pragma unroll 2
        for (int m = m0; m < m1; m += 4) {
            float4 x[R], y[4];
#pragma unroll
            for (int i = 0; i < R; ++i) x[i] = *reinterpret_cast<const float4*>(a + (r + i) * LDL + m);
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (m + j) * ldb + c0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const float v = reinterpret_cast<const float*>(&x[i])[j];
                    acc[i][0] = __ffma2_rn(make_float2(v, v), make_float2(y[j].x, y[j].y), acc[i][0]);
                    acc[i][1] = __ffma2_rn(make_float2(v, v), make_float2(y[j].z, y[j].w), acc[i][1]);
                }
        }
    };
    product(low, low - S * LDL, LDL, c0 & 16, S);
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<float4*>(z + (r + i) * 36 + c0) = make_float4(acc[i][0].x, acc[i][0].y, acc[i][1].x, acc[i][1].y);
    __syncthreads();
    product(low + S, z, 36, 0, ((r + R - 1) | 3) + 1);
#pragma unroll
    for (int i = 0; i < R; ++i) *reinterpret_cast<float4*>(low + (r + i) * LDL + c0) = make_float4(-acc[i][0].x, -acc[i][0].y, -acc[i][1].x, -acc[i][1].y);
    __syncthreads();
}

// what the gates of a chunk and value head say of its rows: G in two floats, beta, e^G, e^(G_last - G) and e^(G_ref - G), G_ref at the
// last row of the row's block of 16
enum { R_HI, R_LO, R_BETA, R_GAM, R_FALL, R_COL, NG };
__device__ __forceinline__ void head_gates(const KdaGdrParams& p, const ChunkInfo& ci, int h, float* out, int lane) {
    double s[2];  // a lane has two neighbouring rows
    float be[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const size_t at = (size_t)(ci.tok0 + r) * p.HV + h;
        s[i] = r < ci.len ? (double)log_decay(p, at, h) : 0.0;
        be[i] = r < ci.len ? load_g(p, p.beta, at) : 0.f;
        if (r < ci.len && (p.flags & KDA_FLAG_BETA_SIGMOID)) be[i] = sigmoid_f(be[i]);
    }
    double run = s[0] + s[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
    }
    const double G[2] = {run - s[1], run}, last = __shfl_sync(0xffffffffu, run, 31), ref = __shfl_sync(0xffffffffu, run, lane | 7);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 2 * lane + i;
        const float hi = (float)G[i], lo = (float)(G[i] - hi);
        out[R_HI * C + r] = hi;
        out[R_LO * C + r] = lo;
        out[R_BETA * C + r] = be[i];
        out[R_GAM * C + r] = expf(hi) * (1.f + lo);
        out[R_FALL * C + r] = expf((float)(last - G[i]));
        out[R_COL * C + r] = expf((float)(ref - G[i]));
    }
}

template <typename T, int K, bool CM>  // CM: records in core-matrix order
__global__ void __launch_bounds__(128, In<T>::P == 1 ? 5 : 1) gdr_intra_kernel(const KdaGdrParams p, const Layout lay) {
    constexpr int P = In<T>::P, LD = K + 8, TILE = C * LD, PART = CM ? SQ : TRI;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* sq = reinterpret_cast<bf16*>(smem);
    bf16* sk = sq + P * TILE;
    float* L = reinterpret_cast<float*>(smem);       // (where q and k were)
    float* Z = L + C * LDL;                          // 32 x 36
    float* rows = reinterpret_cast<float*>(smem + tiles_bytes<T, K>());
    float *rq = rows, *rk = rows + C;                // 1 / norm
    float* gates = rows + 2 * C;                     // of four heads: [head][R_*][64]
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int c = blockIdx.x / p.H, kh = blockIdx.x % p.H, grp = p.HV / p.H;
    pdl_wait();
    const ChunkInfo ci = chunk_info(p, c);
    const size_t row0 = (size_t)ci.tok0 * p.H + kh;
    load_tile<K, LD, 128>(sq, static_cast<const T*>(p.q) + row0 * K, (size_t)p.H * K, ci.len, tid);
    load_tile<K, LD, 128>(sk, static_cast<const T*>(p.k) + row0 * K, (size_t)p.H * K, ci.len, tid);
    cp_async_commit();
    if (w < grp) head_gates(p, ci, kh * grp + w, gates + w * NG * C, lane);
    cp_async_wait<0>();
    __syncthreads();
    {   // 1 / norm: two lanes per row
        const int r = tid >> 1, half = tid & 1;
        float nq = 1.f, nk = 1.f;
        if (p.flags & KDA_FLAG_QK_L2NORM) {
            float a = 0.f, b = 0.f;
#pragma unroll 2
            for (int i = 0; i < K / 16; ++i) {  // eight channels; four rows and their halves read from different banks
                const int at = r * LD + 8 * ((i & 3) + 4 * half + 8 * (i >> 2));
                const float2 u = sum_sq<P>(sq + at, TILE), v = sum_sq<P>(sk + at, TILE);
                a += u.x + u.y;
                b += v.x + v.y;
            }
            a += __shfl_xor_sync(0xffffffffu, a, 1);
            b += __shfl_xor_sync(0xffffffffu, b, 1);
            nq = 1.f / fmaxf(sqrtf(a), 1e-6f);
            nk = 1.f / fmaxf(sqrtf(b), 1e-6f);
        }
        if (!(tid & 1)) rq[r] = nq, rk[r] = nk;
    }
    // q k^T and k k^T, columns up to the diagonal block
    float qk[8][4], kk[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) qk[n][i] = kk[n][i] = 0.f;
    const uint32_t aq = smem_u32(sq), ak = smem_u32(sk);
#pragma unroll 2
    for (int ks = 0; ks < K; ks += 16) {
        uint32_t fq[P][4], fk[P][4];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            a_frag<LD>(fq[i], aq + 2 * i * TILE, 16 * w, ks, lane);
            a_frag<LD>(fk[i], ak + 2 * i * TILE, 16 * w, ks, lane);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (n > w) break;
            uint32_t b[P][4];
#pragma unroll
            for (int i = 0; i < P; ++i) b_frag<LD>(b[i], ak + 2 * i * TILE, 16 * n, ks, lane);
            mma_parts<P, P, P>(qk, n, fq, b);
            mma_parts<P, P, P>(kk, n, fk, b);
        }
    }
    __syncthreads();
    const int i0 = 16 * w + g;
    for (int hg = 0; hg < grp; ++hg) {
        const int h = kh * grp + hg;
        const size_t unit = (size_t)c * p.HV + h;
        float* aux = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.aux) + unit * AUX;
        if (hg % 4 == 0 && hg) {
            if (hg + w < grp) head_gates(p, ci, h + w, gates + w * NG * C, lane);
            __syncthreads();
        }
        const float* G = gates + (hg % 4) * NG * C;
        const float *ghi = G + R_HI * C, *glo = G + R_LO * C, *sb = G + R_BETA * C, *col = G + R_COL * C;
        {   // a row's numbers, two threads a row
            const int r = tid & 63;
            const float gam = G[R_GAM * C + r], fall = G[R_FALL * C + r], nk = rk[r], be = sb[r];
            if (tid < 64) {
                aux[A_GAM * C + r] = gam;
                aux[A_FALL * C + r] = fall;
                aux[A_BGK * C + r] = be * gam * nk;
                aux[A_FK * C + r] = fall * nk;
                aux[A_OQ * C + r] = p.scale * gam * rq[r];
                aux[A_GK * C + r] = gam * nk;
                if (r == 63) aux[A_LAST * C] = G[R_GAM * C + 63];
            } else {
                aux[A_BETA * C + r] = be;
                aux[A_RQ * C + r] = rq[r];
                aux[A_RK * C + r] = nk;
                aux[A_GHI * C + r] = ghi[r];
                aux[A_GLO * C + r] = glo[r];
            }
        }
        bf16* A = reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.A) + unit * 3 * PART;
        // left of the diagonal block D_ij = e^(G_i - G_ref) e^(G_ref - G_j) about the last row of j's block: an exponential a row
        // and block, not one an element
        const float si[2] = {p.scale * rq[i0], p.scale * rq[i0 + 8]}, bi[2] = {sb[i0] * rk[i0], sb[i0 + 8] * rk[i0 + 8]};
        const float hi[2] = {ghi[i0], ghi[i0 + 8]}, lo[2] = {glo[i0], glo[i0 + 8]};
#pragma unroll
        for (int J = 0; J < 4; ++J) {
            if (J > w) break;
            float fall[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) fall[r] = J < w ? expf(hi[r] - ghi[16 * J + 15] + (lo[r] - glo[16 * J + 15])) : 1.f;
#pragma unroll
            for (int n = 2 * J; n < 2 * J + 2; ++n) {
                const int j = 8 * n + 2 * t;
                float2 cf = *reinterpret_cast<const float2*>(rk + j);
                if (J < w) {
                    const float2 f = *reinterpret_cast<const float2*>(col + j);
                    cf = make_float2(cf.x * f.x, cf.y * f.y);
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int i = i0 + 8 * r;
                    float d[2] = {fall[r] * cf.x, fall[r] * cf.y}, a[2], l[2];
                    if (J == w)
#pragma unroll
                        for (int x = 0; x < 2; ++x) d[x] = i >= j + x ? d[x] * expf(hi[r] - ghi[j + x] + (lo[r] - glo[j + x])) : 0.f;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        a[x] = i >= j + x ? si[r] * qk[n][2 * r + x] * d[x] : 0.f;
                        l[x] = i > j + x ? bi[r] * kk[n][2 * r + x] * d[x] : 0.f;
                    }
                    put<3>(A, PART, CM ? cm_idx(i, j, C) : blk(w, J) * BLK + tri_idx(i & 15, j & 15), a[0], a[1]);
                    *reinterpret_cast<float2*>(L + i * LDL + j) = make_float2(l[0], l[1]);
                }
            }
        }
        __syncwarp();
        {   // diagonal block w in place: column `col` of its inverse by substitution
            const int col = lane & 15;
            float* B = L + 16 * w * LDL + 16 * w;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = i == col ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < 16; m += 4)
#pragma unroll
                for (int i = m + 1; i < 16; ++i) {
                    const float4 v = *reinterpret_cast<const float4*>(B + i * LDL + m);
                    x[i] = fmaf(-v.x, x[m], x[i]);
                    if (i > m + 1) x[i] = fmaf(-v.y, x[m + 1], x[i]);
                    if (i > m + 2) x[i] = fmaf(-v.z, x[m + 2], x[i]);
                    if (i > m + 3) x[i] = fmaf(-v.w, x[m + 3], x[i]);
                }
            __syncwarp();
            if (lane < 16)
#pragma unroll
                for (int i = 0; i < 16; ++i) B[i * LDL + col] = x[i];
        }
        __syncthreads();
        // join blocks of 16, then of 32: a thread has one row, then two, and four columns
        join<1>(L, Z, tid >> 6, tid & 63);
        join<2>(L, Z, 0, tid);
        bf16* Tm = reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.T) + unit * 3 * PART;
        bf16* Tb = reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.Tb) + unit * 3 * PART;
        for (int i = tid; i < NBLK * 32; i += 128) {
            const int b = i >> 5, r = i & 15, c0 = (i >> 1) & 8;
            const int I = b < 1 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, J = b - blk(I, 0);
            float x[8], y[8];
            *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(L + (16 * I + r) * LDL + 16 * J + c0);
            *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(L + (16 * I + r) * LDL + 16 * J + c0 + 4);
            if (CM) {
                const int at = cm_idx(16 * I + r, 16 * J + c0, C);
                if (!(p.flags & KDA_FLAG_NO_SAVE)) put8(Tb, PART, at, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = x[j] * sb[16 * J + c0 + j];
                put8(Tm, PART, at, y);
            } else {
                put8(Tm, PART, b * BLK + tri_idx(r, c0), x);
            }
        }
        __syncthreads();
    }
}

template <typename T, int K, bool CM>
static cudaError_t launch_intra(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = tiles_bytes<T, K>() + (2 + 4 * NG) * C * 4;
    cudaError_t e = allow_smem(gdr_intra_kernel<T, K, CM>, bytes);
    if (e != cudaSuccess) return e;
    return launch_dependent(gdr_intra_kernel<T, K, CM>, p.NT * p.H, 128, bytes, s, p, l);
}

cudaError_t intra(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    if (p.dtype == KDA_DTYPE_F32) return p.dk == 64 ? launch_intra<float, 64, false>(p, l, s) : launch_intra<float, 128, false>(p, l, s);
    if (on_tc(p)) return launch_intra<bf16, 128, true>(p, l, s);
    return p.dk == 64 ? launch_intra<bf16, 64, false>(p, l, s) : launch_intra<bf16, 128, false>(p, l, s);
}

}  // namespace gdr
}  // namespace kda
