// Gated delta rule, backward: what the gradient kernels share once a chunk's products are in registers.  256 threads; fragments of
// 16 x 8 tiles as mma.sync leaves them (row g and g + 8 of row block rb = warp mod 4, columns 2 t, 2 t + 1), half = warp / 4 of the
// columns.
#pragma once

#include "gdr.cuh"

namespace kda {
namespace gdr {

namespace gr {
constexpr int LDZ = C + 8;
enum { R_N = 0, R_B = 2, R_F = 4, R_E = 6, R_H = 8, R_Y = 10, R_COL = 11, RED = 15 };  // rows of `red`: sums of N (2 halves), dL KKD (2), q.F (2), k.E (2), k.H (2), Y.v, columns of N (4)
}

// the chunk's rows and where its 64 x 64 matrices go
template <typename T, int K>
struct GradRows {
    static constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, ROWS = C * LDK, ZPART = C * gr::LDZ;
    const bf16 *q, *k;     // row-major parts
    uint32_t qa, ka;       // their shared-memory addresses
    bf16 *Z, *X;
    uint32_t za, xa;
    const float *gam, *fall, *be, *rq, *rk, *ghi, *glo;
    float* red;
    float last;
};

// q k^T and k k^T, the tiles of this warp's half
template <typename T, int K>
__device__ __forceinline__ void grad_rows_products(const GradRows<T, K>& m, int rb, int half, int lane, float (&qk)[4][4], float (&kk)[4][4]) {
    constexpr int P = In<T>::P, LDK = K + 8;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) qk[j][i] = kk[j][i] = 0.f;
#pragma unroll 1
    for (int d = 0; d < K; d += 16) {
        uint32_t fq[P][4], fk[P][4];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            a_frag<LDK>(fq[i], m.qa + 2 * i * m.ROWS, 16 * rb, d, lane);
            a_frag<LDK>(fk[i], m.ka + 2 * i * m.ROWS, 16 * rb, d, lane);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (2 * half + j > rb) break;
            uint32_t b[P][4];
#pragma unroll
            for (int i = 0; i < P; ++i) b_frag<LDK>(b[i], m.ka + 2 * i * m.ROWS, 32 * half + 16 * j, d, lane);
            mma_parts<P, P, P>(qk, j, fq, b);
            mma_parts<P, P, P>(kk, j, fk, b);
        }
    }
}

// Z, X and the sums over rows and columns of N and over rows of dL KKD
template <typename T, int K>
__device__ __forceinline__ void grad_pairs(const GradRows<T, K>& m, float scale, int rb, int half, int lane, const float (&dA)[4][4],
                                           const float (&dL)[4][4], const float (&qk)[4][4], const float (&kk)[4][4]) {
    using namespace gr;
    constexpr int PO = In<T>::PO;
    const int g = lane >> 2, t = lane & 3;
    const int r0 = 16 * rb + g;
    float rn[2] = {0.f, 0.f}, rbeta[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (2 * half + j / 2 > rb) break;
        float col[2] = {0.f, 0.f};
        const int j0 = 32 * half + 8 * j + 2 * t;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            float z[2], x[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int cc = j0 + y;
                const float d = r >= cc ? expf(m.ghi[r] - m.ghi[cc] + (m.glo[r] - m.glo[cc])) : 0.f;
                const float a = r >= cc ? dA[j][2 * i + y] * scale * d * m.rq[r] * m.rk[cc] : 0.f;
                const float kkd = m.rk[r] * m.rk[cc] * d, l = r > cc ? -dL[j][2 * i + y] * kkd : 0.f;
                z[y] = a;
                x[y] = l * m.be[r];
                const float lk = l * kk[j][2 * i + y];
                const float nn = r > cc ? fmaf(a, qk[j][2 * i + y], m.be[r] * lk) : 0.f;
                rn[i] += nn;
                rbeta[i] += r > cc ? lk : 0.f;
                col[y] += nn;
            }
            put<PO>(m.Z, m.ZPART, r * LDZ + j0, z[0], z[1]);
            put<PO>(m.X, m.ZPART, r * LDZ + j0, x[0], x[1]);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) col[y] += __shfl_xor_sync(0xffffffffu, col[y], o);
            if (g == 0) m.red[(R_COL + rb) * C + j0 + y] = col[y];
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            rn[i] += __shfl_xor_sync(0xffffffffu, rn[i], o);
            rbeta[i] += __shfl_xor_sync(0xffffffffu, rbeta[i], o);
        }
        if (t == 0) {
            m.red[(R_N + half) * C + r0 + 8 * i] = rn[i];
            m.red[(R_B + half) * C + r0 + 8 * i] = rbeta[i];
        }
    }
}

// The products with the states in the rows' units: F becomes its share of dq, E that of dk (E and H), and the row sums with q and k
template <typename T, int K>
__device__ __forceinline__ void grad_scale(const GradRows<T, K>& m, float scale, int rb, int half, int lane, float (&F)[K / 16][4],
                                           float (&E)[K / 16][4], const float (&H)[K / 16][4]) {
    using namespace gr;
    constexpr int P = In<T>::P, LDK = K + 8, NK = K / 16;
    const int g = lane >> 2, t = lane & 3, r0 = 16 * rb + g;
    // this half's share of the row sums; scale the products with the states to the rows' units
    float rf[2] = {0.f, 0.f}, re[2] = {0.f, 0.f}, rh[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i, d = half * (K / 2) + 8 * j + 2 * t;
            const float2 q = get2<P>(m.q, m.ROWS, r * LDK + d), k = get2<P>(m.k, m.ROWS, r * LDK + d);
            const float ff = scale * m.gam[r] * m.rq[r], fe = m.gam[r] * m.rk[r], fh = m.fall[r] * m.rk[r];
            float &f0 = F[j][2 * i], &f1 = F[j][2 * i + 1];
            f0 *= ff; f1 *= ff;
            const float e0 = E[j][2 * i] * fe, e1 = E[j][2 * i + 1] * fe, h0 = H[j][2 * i] * fh, h1 = H[j][2 * i + 1] * fh;
            rf[i] += q.x * f0 + q.y * f1;
            re[i] += k.x * e0 + k.y * e1;
            rh[i] += k.x * h0 + k.y * h1;
            E[j][2 * i] = h0 - m.be[r] * e0;
            E[j][2 * i + 1] = h1 - m.be[r] * e1;
        }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            rf[i] += __shfl_xor_sync(0xffffffffu, rf[i], o);
            re[i] += __shfl_xor_sync(0xffffffffu, re[i], o);
            rh[i] += __shfl_xor_sync(0xffffffffu, rh[i], o);
        }
        if (t == 0) {
            const int r = r0 + 8 * i;
            m.red[(R_F + half) * C + r] = rf[i];
            m.red[(R_E + half) * C + r] = re[i];
            m.red[(R_H + half) * C + r] = rh[i];
        }
    }
}

// dq and dk of 16 rows and half of the channels (in F and E), the gate's and beta's gradients; total = <S0, dS>
template <typename T, int K, class Sync>
__device__ __forceinline__ void grad_finish(const KdaGdrParams& p, const Layout& lay, const GradRows<T, K>& m, const ChunkInfo& ci, size_t unit, int h,
                                            int kh, int grp, float total, float (&F)[K / 16][4], float (&E)[K / 16][4], int w, int lane, Sync sync) {
    using namespace gr;
    constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, NK = K / 16;
    const int g = lane >> 2, t = lane & 3, rb = w & 3, half = w >> 2, r0 = 16 * rb + g;
    const size_t qrow = (size_t)ci.tok0 * p.H + kh;
    sync();  // Z, X and the sums are there
    // dq (in F) and dk (in E) of 16 rows and this half of the channels
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        uint32_t fz[PO][4], fx[PO][4], zt[PO][4], xt[PO][4];
#pragma unroll
        for (int i = 0; i < PO; ++i) {
            if (b <= rb) {
                a_frag<LDZ>(fz[i], m.za + 2 * i * m.ZPART, 16 * rb, 16 * b, lane);
                a_frag<LDZ>(fx[i], m.xa + 2 * i * m.ZPART, 16 * rb, 16 * b, lane);
            }
            if (b >= rb) {
                a_frag_t<LDZ>(zt[i], m.za + 2 * i * m.ZPART, 16 * rb, 16 * b, lane);
                a_frag_t<LDZ>(xt[i], m.xa + 2 * i * m.ZPART, 16 * rb, 16 * b, lane);
            }
        }
#pragma unroll
        for (int j = 0; j < NK / 2; ++j) {
            uint32_t bk[P][4], bq[P][4];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                b_frag_t<LDK>(bk[i], m.ka + 2 * i * m.ROWS, half * (K / 2) + 16 * j, 16 * b, lane);
                b_frag_t<LDK>(bq[i], m.qa + 2 * i * m.ROWS, half * (K / 2) + 16 * j, 16 * b, lane);
            }
            if (b <= rb) {
                mma_parts<PO, P, PO>(F, j, fz, bk);
                mma_parts<PO, P, PO>(E, j, fx, bk);
            }
            if (b >= rb) {
                mma_parts<PO, P, PO>(E, j, xt, bk);
                mma_parts<PO, P, PO>(E, j, zt, bq);
            }
        }
    }
    if (w == 0) {  // the gate's and beta's gradients, two neighbouring rows per lane
        double dG[2], hsum = 0.0;
        float db[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i, I = r >> 4;
            float colsum = 0.f;
            for (int x = I; x < 4; ++x) colsum += m.red[(R_COL + x) * C + r];
            const float n = m.red[R_N * C + r] + m.red[(R_N + 1) * C + r], bb = m.red[R_B * C + r] + m.red[(R_B + 1) * C + r];
            const float f = m.red[R_F * C + r] + m.red[(R_F + 1) * C + r], e = m.red[R_E * C + r] + m.red[(R_E + 1) * C + r],
                        hh = m.red[R_H * C + r] + m.red[(R_H + 1) * C + r];
            dG[i] = (double)n - colsum + f - (double)m.be[r] * e - hh;
            hsum += hh;
            db[i] = m.red[R_Y * C + r] - e + bb;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) hsum += __shfl_xor_sync(0xffffffffu, hsum, o);
        double run = dG[0] + dG[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double dn = __shfl_down_sync(0xffffffffu, run, o);
            if (lane + o < 32) run += dn;
        }
        run += (double)m.last * total + hsum;
        const double dg[2] = {run, run - dG[0]};
        float dAl = 0.f, dbi = 0.f;
        const float eA = (p.flags & KDA_FLAG_GATE) ? expf(p.A_log[h]) : 0.f, bias = (p.flags & KDA_FLAG_GATE) && p.dt_bias ? p.dt_bias[h] : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            if (r < ci.len) {
                const size_t at = (size_t)(ci.tok0 + r) * p.HV + h;
                float d = (float)dg[i], b = db[i];
                if (p.flags & KDA_FLAG_GATE) {
                    const float a = load_g(p, p.g, at) + bias, sp = softplus_f(a);
                    dAl += d * fmaxf(-eA * sp, G_MIN);
                    d *= -eA * (a > 20.f ? 1.f : sigmoid_f(a));
                    dbi += d;
                }
                if (p.flags & KDA_FLAG_BETA_SIGMOID) b *= m.be[r] * (1.f - m.be[r]);
                store_g(p, p.grad_g, at, d);
                store_g(p, p.grad_beta, at, b);
            }
        }
        if (p.flags & KDA_FLAG_GATE) {
            dAl = warp_sum(dAl);
            dbi = warp_sum(dbi);
            if (lane == 0) *reinterpret_cast<float2*>(static_cast<char*>(p.bwd_scratch) + lay.part + unit * 8) = make_float2(dAl, dbi);
        }
    }
    if (grp > 1) {  // the group's value heads are added up by gdr_heads_kernel
        float* out = reinterpret_cast<float*>(static_cast<char*>(p.bwd_scratch) + lay.dqk) + unit * 2 * C * K;
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (r0 + 8 * i) * K + half * (K / 2) + 8 * j + 2 * t;
                store2(out + at, F[j][2 * i], F[j][2 * i + 1]);
                store2(out + C * K + at, E[j][2 * i], E[j][2 * i + 1]);
            }
        return;
    }
    float dot[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    if (p.flags & KDA_FLAG_QK_L2NORM) {
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (r0 + 8 * i) * LDK + half * (K / 2) + 8 * j + 2 * t;
                const float2 q = get2<P>(m.q, m.ROWS, at), k = get2<P>(m.k, m.ROWS, at);
                dot[0][i] += q.x * F[j][2 * i] + q.y * F[j][2 * i + 1];
                dot[1][i] += k.x * E[j][2 * i] + k.y * E[j][2 * i + 1];
            }
        sync();  // (the sums above have been read)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) dot[x][i] += __shfl_xor_sync(0xffffffffu, dot[x][i], o);
                if (t == 0) m.red[(2 * x + half) * C + r0 + 8 * i] = dot[x][i];
            }
        sync();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            // a row shorter than 1e-6 is divided by that, whatever its length
            dot[0][i] = m.rq[r] < 1e6f ? m.rq[r] * m.rq[r] * (m.red[r] + m.red[C + r]) : 0.f;
            dot[1][i] = m.rk[r] < 1e6f ? m.rk[r] * m.rk[r] * (m.red[2 * C + r] + m.red[3 * C + r]) : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = r0 + 8 * i;
        if (r >= ci.len) continue;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
            const int d = half * (K / 2) + 8 * j + 2 * t;
            const float2 q = get2<P>(m.q, m.ROWS, r * LDK + d), k = get2<P>(m.k, m.ROWS, r * LDK + d);
            const size_t at = (qrow + (size_t)r * p.H) * K + d;
            store2(static_cast<T*>(p.grad_q) + at, F[j][2 * i] - q.x * dot[0][i], F[j][2 * i + 1] - q.y * dot[0][i]);
            store2(static_cast<T*>(p.grad_k) + at, E[j][2 * i] - k.x * dot[1][i], E[j][2 * i + 1] - k.y * dot[1][i]);
        }
    }
}

}  // namespace gdr
}  // namespace kda
