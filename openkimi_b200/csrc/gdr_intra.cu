// Gated delta rule, the part of a chunk that needs no state: per key head the products q k^T and k k^T of the 64 rows, and for
// every value head of its group
//     A = scale (q^ k^T) D,  L = beta (k^ k^T) D strictly below the diagonal,  T = (I + L)^-1,     D_ij = e^(G_i - G_j)
// as records of three BF16 parts (the lower triangle's blocks), with the rows' e^G, e^(G_last - G), beta and 1 / norm.
//
// One CTA of four warps per (chunk, key head); warp w holds rows 16 w .. 16 w + 15 of both products in registers for all value
// heads.  G is summed in 64 bits and kept in two floats, so that a difference of two large sums still gives a decay to FP32.  The
// inverse goes by blocks: the four 16 x 16 diagonal blocks by substitution (a lane per column), then neighbours joined twice,
// T_21 = -T_22 (L_21 T_11), in FP32 multiply-adds.
#include "gdr.cuh"

namespace kda {
namespace gdr {

constexpr int LDL = 68;  // floats per row of L / T

template <typename T, int K, bool CM>  // CM: records in core-matrix order
__global__ void __launch_bounds__(128) gdr_intra_kernel(const KdaGdrParams p, const Layout lay) {
    constexpr int P = In<T>::P, LD = K + 8, TILE = C * LD, PART = CM ? SQ : TRI;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* sq = reinterpret_cast<bf16*>(smem);
    bf16* sk = sq + P * TILE;
    float* L = reinterpret_cast<float*>(sk + P * TILE);
    float* Z = L + C * LDL;                 // 32 x 36
    float* rows = Z + 32 * 36;              // rq, rk, G high, G low, beta: 5 x 64
    float *rq = rows, *rk = rows + C, *ghi = rows + 2 * C, *glo = rows + 3 * C, *sb = rows + 4 * C;
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int c = blockIdx.x / p.H, kh = blockIdx.x % p.H, grp = p.HV / p.H;
    pdl_wait();
    const ChunkInfo ci = chunk_info(p, c);
    const size_t row0 = (size_t)ci.tok0 * p.H + kh;
    load_tile<K, LD, 128>(sq, static_cast<const T*>(p.q) + row0 * K, (size_t)p.H * K, ci.len, tid);
    load_tile<K, LD, 128>(sk, static_cast<const T*>(p.k) + row0 * K, (size_t)p.H * K, ci.len, tid);
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    {   // 1 / norm: two lanes per row
        const int r = tid >> 1, c0 = (tid & 1) * (K / 2);
        float nq = 1.f, nk = 1.f;
        if (p.flags & KDA_FLAG_QK_L2NORM) {
            float a = 0.f, b = 0.f;
#pragma unroll 8
            for (int i = 0; i < K / 2; i += 2) {
                const float2 x = get2<P>(sq, TILE, r * LD + c0 + i), y = get2<P>(sk, TILE, r * LD + c0 + i);
                a = fmaf(x.x, x.x, fmaf(x.y, x.y, a));
                b = fmaf(y.x, y.x, fmaf(y.y, y.y, b));
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
        if (w == 0) {  // a lane has two neighbouring rows
            double s[2];
            float be[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 2 * lane + i;
                const size_t at = (size_t)(ci.tok0 + r) * p.HV + h;
                s[i] = r < ci.len ? (double)log_decay(p, at, h) : 0.0;
                be[i] = r < ci.len ? load_g(p, p.beta, at) : 0.f;
                if (r < ci.len && (p.flags & KDA_FLAG_BETA_SIGMOID)) be[i] = sigmoid_f(be[i]);
            }
            double pair = s[0] + s[1], run = pair;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += up;
            }
            const double G[2] = {run - s[1], run}, last = __shfl_sync(0xffffffffu, run, 31);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 2 * lane + i;
                const float hi = (float)G[i], lo = (float)(G[i] - hi);
                ghi[r] = hi; glo[r] = lo; sb[r] = be[i];
                const float gam = expf(hi) * (1.f + lo), fall = expf((float)(last - G[i]));
                aux[A_GAM * C + r] = gam;
                aux[A_FALL * C + r] = fall;
                aux[A_BGK * C + r] = be[i] * gam * rk[r];
                aux[A_FK * C + r] = fall * rk[r];
                aux[A_OQ * C + r] = p.scale * gam * rq[r];
                aux[A_GK * C + r] = gam * rk[r];
                aux[A_BETA * C + r] = be[i];
                aux[A_RQ * C + r] = rq[r];
                aux[A_RK * C + r] = rk[r];
                aux[A_GHI * C + r] = hi;
                aux[A_GLO * C + r] = lo;
            }
            if (lane == 0) aux[A_LAST * C] = expf((float)last);
        }
        __syncthreads();
        bf16* A = reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.A) + unit * 3 * PART;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            if (n / 2 > w) break;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int i = i0 + 8 * r, j = 8 * n + 2 * t;
                float a[2], l[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int jj = j + x;
                    const float d = i >= jj ? expf(ghi[i] - ghi[jj] + (glo[i] - glo[jj])) : 0.f;
                    a[x] = i >= jj ? p.scale * qk[n][2 * r + x] * rq[i] * rk[jj] * d : 0.f;
                    l[x] = i > jj ? sb[i] * (kk[n][2 * r + x] * rk[i] * rk[jj] * d) : 0.f;
                }
                put<3>(A, PART, CM ? cm_idx(i, j, C) : blk(w, n / 2) * BLK + tri_idx(i & 15, j & 15), a[0], a[1]);
                *reinterpret_cast<float2*>(L + i * LDL + j) = make_float2(l[0], l[1]);
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
            for (int m = 0; m < 15; ++m)
#pragma unroll
                for (int i = m + 1; i < 16; ++i) x[i] = fmaf(-B[i * LDL + m], x[m], x[i]);
            __syncwarp();
            if (lane < 16)
#pragma unroll
                for (int i = 0; i < 16; ++i) B[i * LDL + col] = x[i];
        }
        __syncthreads();
        // join blocks of 16, then of 32
#pragma unroll
        for (int s = 16; s <= 32; s *= 2) {
            const int per = 4 * s;                                // threads per joined pair: 64, 128
            const int pr = tid / per, q = tid % per, r = q / 4, c0 = (q % 4) * (s / 4);
            const int R = 2 * s * pr + s, Cc = 2 * s * pr;
            float acc[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll 4
            for (int m = c0 & 16; m < s; ++m) {                   // (nothing is above the diagonal, and not all of it is written)
                const float a = L[(R + r) * LDL + Cc + m];
#pragma unroll
                for (int i = 0; i < s / 4; ++i) acc[i] = fmaf(a, L[(Cc + m) * LDL + Cc + c0 + i], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < s / 4; ++i) Z[(s == 16 ? 16 * pr + r : r) * 36 + c0 + i] = acc[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll 4
            for (int m = 0; m <= r; ++m) {
                const float a = L[(R + r) * LDL + R + m];
#pragma unroll
                for (int i = 0; i < s / 4; ++i) acc[i] = fmaf(a, Z[(s == 16 ? 16 * pr + m : m) * 36 + c0 + i], acc[i]);
            }
#pragma unroll
            for (int i = 0; i < s / 4; ++i) L[(R + r) * LDL + Cc + c0 + i] = -acc[i];
            __syncthreads();
        }
        bf16* Tm = reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.T) + unit * 3 * PART;
        for (int i = tid; i < NBLK * 128; i += 128) {
            const int b = i >> 7, r = (i >> 3) & 15, cc = (i & 7) * 2;
            const int I = b < 1 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, J = b - blk(I, 0);
            const float2 x = *reinterpret_cast<const float2*>(L + (16 * I + r) * LDL + 16 * J + cc);
            if (CM) {
                const int at = cm_idx(16 * I + r, 16 * J + cc, C);
                put<3>(Tm, PART, at, x.x * sb[16 * J + cc], x.y * sb[16 * J + cc + 1]);
                if (!(p.flags & KDA_FLAG_NO_SAVE)) put<3>(reinterpret_cast<bf16*>(static_cast<char*>(p.workspace) + lay.Tb) + unit * 3 * PART, PART, at, x.x, x.y);
            } else {
                put<3>(Tm, PART, b * BLK + tri_idx(r, cc), x.x, x.y);
            }
        }
        __syncthreads();
    }
}

template <typename T, int K, bool CM>
static cudaError_t launch_intra(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = 2 * In<T>::P * C * (K + 8) * 2 + (C * LDL + 32 * 36 + 5 * C) * 4;
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
