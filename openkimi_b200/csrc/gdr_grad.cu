// Gated delta rule, backward: the gradients of a chunk once the state S0 at its start and the gradient dS at its end are known.
//
//   F = do S0^T, E = Y S0^T, H = V' dS^T;   dA = do V'^T (i >= j),  dL = -Y V'^T (i > j)
//   Z = scale dA D / (|q_i| |k_j|),  X = dL beta_i D / (|k_i| |k_j|)
//   dq = scale e^G / |q| F + Z k          dk = -e^G beta / |k| E + e^(G_last - G) / |k| H + X k + X^T k + Z^T q
// and, with L2 norm, dq -= q (q . dq) / |q|^2, the same for k.  (Everything is in units of the rows as they arrive.)
//   dbeta = Y . v - e^G k^ . E + rows of dL KKD
//   dG = rows - columns of N + q^ . (scale e^G F) - e^G beta k^ . E - e^(G_last-G) k^ . H,   N = dA A + dL beta KKD below the diagonal
//   dG_last += e^G_last <S0, dS> + sum e^(G_last-G) k^ . H,    dg = reverse cumulative sum of dG
// The diagonal of A does not depend on G: left out of N, where its share of rows and columns would cancel (kept, it costs a factor
// 20 of dg's precision at decays of e^-4 a token).
//
// One CTA of eight warps per (chunk, value head): warp w has rows 16 (w mod 4).. and half w / 4 of the columns of every product.
// The value columns come in panels of 32, as three BF16 parts each of S0, dS, Y, V'.
// Bound by mma.sync and the conversions before it: a unit in FP32 (64 key channels, 128 columns) takes 34 us alone on its SM, where
// three parts of either operand are six products each.  BF16 with 128 channels and columns goes on tcgen05 (gdr_grad_tc.cu).
#include "gdr.cuh"

namespace kda {
namespace gdr {

// What follows has fragments of 16 x 8 tiles as mma.sync leaves them: row g and g + 8 of row block rb = warp mod 4, columns 2 t, 2 t + 1,
// half = warp / 4 of the columns.
namespace gr {
constexpr int NTHR = 256, EP = 32, LDE = EP + 8, PAN = C * LDE, LDZ = C + 8;
enum { R_B = 0, R_F = 2, R_E = 4, R_H = 6, R_Y = 8, RED = 9 };  // rows of `red`: sums of dL KKD (2 halves), q.F (2), k.E (2), k.H (2), Y.v
// rows of `sumN`, in 64 bits: sums over rows of N (2 halves) and over its columns (4 blocks of rows).  In dG's running sum a pair of rows
// cancels between its row and its column: with sums in FP32 their rounding was left, 4e-6 of dA_log's terms at decays of e^-0.3 to e^-32.
enum { N_ROW = 0, N_COL = 2, SUMN = 6 };
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
    double* sumN;
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
    double rn[2] = {0.0, 0.0};
    float rbeta[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (2 * half + j / 2 > rb) break;
        double col[2] = {0.0, 0.0};
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
            if (g == 0) m.sumN[(N_COL + rb) * C + j0 + y] = col[y];
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
            m.sumN[(N_ROW + half) * C + r0 + 8 * i] = rn[i];
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

// dq and dk of 16 rows and half of the channels (in F and E), the gate's and beta's gradients; total = <S0, dS>.
template <typename T, int K>
__device__ __forceinline__ void grad_finish(const KdaGdrParams& p, const Layout& lay, const GradRows<T, K>& m, const ChunkInfo& ci, size_t unit, int h,
                                            int kh, int grp, float total, float (&F)[K / 16][4], float (&E)[K / 16][4], int w, int lane) {
    using namespace gr;
    constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, NK = K / 16;
    const int g = lane >> 2, t = lane & 3, rb = w & 3, half = w >> 2, r0 = 16 * rb + g;
    const size_t qrow = (size_t)ci.tok0 * p.H + kh;
    __syncthreads();  // Z, X and the sums are there
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
        double dG[2], h1[2];
        float db[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i, I = r >> 4;
            double n = m.sumN[N_ROW * C + r] + m.sumN[(N_ROW + 1) * C + r];
            for (int x = I; x < 4; ++x) n -= m.sumN[(N_COL + x) * C + r];
            const float bb = m.red[R_B * C + r] + m.red[(R_B + 1) * C + r];
            const float f = m.red[R_F * C + r] + m.red[(R_F + 1) * C + r], e = m.red[R_E * C + r] + m.red[(R_E + 1) * C + r],
                        hh = m.red[R_H * C + r] + m.red[(R_H + 1) * C + r];
            dG[i] = n + f - (double)m.be[r] * e;
            h1[i] = hh;
            db[i] = m.red[R_Y * C + r] - e + bb;
        }
        const float2 dg = decay_gradients(dG, h1, (double)m.last * total, lane);
        gate_gradients(p, lay, ci, unit, h, dg.x, dg.y, db[0], db[1], m.be[2 * lane], m.be[2 * lane + 1], lane);
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
        __syncthreads();  // (the sums above have been read)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) dot[x][i] += __shfl_xor_sync(0xffffffffu, dot[x][i], o);
                if (t == 0) m.red[(2 * x + half) * C + r0 + 8 * i] = dot[x][i];
            }
        __syncthreads();
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

template <typename T, int K>
struct GradMap {
    static constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, ROWS = C * LDK;
    static constexpr int Q = 0, KK = P * ROWS, DO = 2 * P * ROWS, Y = DO + P * gr::PAN, V = Y + 3 * gr::PAN, S0 = V + 3 * gr::PAN,
                         DS = S0 + 3 * K * gr::LDE, END = DS + 3 * K * gr::LDE;
    static constexpr int Z = DO, X = Z + PO * C * gr::LDZ;  // over the panels, once they have been used
    static_assert(X + PO * C * gr::LDZ <= END, "Z and X fit");
    static constexpr int FLOATS = 7 * C + (gr::RED + 1) * C; // rows' numbers; sums over rows
    static constexpr int BYTES = 2 * END + FLOATS * 4 + gr::SUMN * C * 8;
    static_assert((2 * END + FLOATS * 4) % 8 == 0, "sums in 64 bits");
};

template <typename T, int K>
__global__ void __launch_bounds__(256) gdr_grad_kernel(const KdaGdrParams p, const Layout lay) {
    using namespace gr;
    using M = GradMap<T, K>;
    constexpr int P = M::P, LDK = M::LDK, NK = K / 16;  // NK column tiles of a warp's half of K
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* sm = reinterpret_cast<bf16*>(smem);
    const uint32_t sa = smem_u32(sm);
    float* sx = reinterpret_cast<float*>(smem + 2 * M::END);
    float* red = sx + 7 * C;   // [RED] sums, then the warps' shares of <S0, dS>
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rb = w & 3, half = w >> 2;
    const int c = blockIdx.x / p.HV, h = blockIdx.x % p.HV, grp = p.HV / p.H, kh = h / grp;
    const size_t unit = blockIdx.x;
    pdl_wait();
    const ChunkInfo ci = chunk_info(p, c);
    const char* ws = static_cast<const char*>(p.workspace);
    const char* sc = static_cast<const char*>(p.bwd_scratch);
    const size_t qrow = (size_t)ci.tok0 * p.H + kh, vrow = (size_t)ci.tok0 * p.HV + h;
    load_tile<K, LDK, NTHR>(sm + M::Q, static_cast<const T*>(p.q) + qrow * K, (size_t)p.H * K, ci.len, tid);
    load_tile<K, LDK, NTHR>(sm + M::KK, static_cast<const T*>(p.k) + qrow * K, (size_t)p.H * K, ci.len, tid);
    cp_async_commit();
    const float* aux = reinterpret_cast<const float*>(ws + lay.aux) + unit * AUX;
    for (int i = tid; i < 7 * C; i += NTHR) sx[i] = aux[i];
    const GradRows<T, K> m = {sm + M::Q, sm + M::KK, sa + 2 * M::Q, sa + 2 * M::KK, sm + M::Z, sm + M::X, sa + 2 * M::Z, sa + 2 * M::X,
                              sx, sx + C, sx + 2 * C, sx + 3 * C, sx + 4 * C, sx + 5 * C, sx + 6 * C, red, reinterpret_cast<double*>(sx + M::FLOATS), aux[A_LAST * C]};

    float F[NK][4], E[NK][4], H[NK][4], dA[4][4], dL[4][4];
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) F[j][i] = E[j][i] = H[j][i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) dA[j][i] = dL[j][i] = 0.f;
    float ss = 0.f, yv[2] = {0.f, 0.f};
    const float* gY = reinterpret_cast<const float*>(sc + lay.Y) + unit * C * p.dv;
    const float* gV = reinterpret_cast<const float*>(ws + lay.Vn) + unit * C * p.dv;
    const float* gS = reinterpret_cast<const float*>(ws + lay.S0) + unit * K * p.dv;
    const float* gD = reinterpret_cast<const float*>(sc + lay.dS) + unit * K * p.dv;
    const int pr = tid >> 3, pc = (tid & 7) * 4;  // this thread's rows pr, pr + 32, .. and columns of a panel
#pragma unroll 1
    for (int e0 = 0; e0 < p.dv; e0 += EP) {
        if (e0) __syncthreads();
        load_tile<EP, LDE, NTHR>(sm + M::DO, static_cast<const T*>(p.grad_o) + vrow * p.dv + e0, (size_t)p.HV * p.dv, ci.len, tid);
        cp_async_commit();
        float4 ry[2], rv[2], rs[K / 32], rd[K / 32];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ry[i] = *reinterpret_cast<const float4*>(gY + (size_t)(pr + 32 * i) * p.dv + e0 + pc);
            rv[i] = *reinterpret_cast<const float4*>(gV + (size_t)(pr + 32 * i) * p.dv + e0 + pc);
        }
#pragma unroll
        for (int i = 0; i < K / 32; ++i) {
            rs[i] = *reinterpret_cast<const float4*>(gS + (size_t)(pr + 32 * i) * p.dv + e0 + pc);
            rd[i] = *reinterpret_cast<const float4*>(gD + (size_t)(pr + 32 * i) * p.dv + e0 + pc);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (pr + 32 * i < ci.len) {
                const T* v = static_cast<const T*>(p.v) + (vrow + (size_t)(pr + 32 * i) * p.HV) * p.dv + e0 + pc;
                const float2 a = load2(v), b = load2(v + 2);
                yv[i] += ry[i].x * a.x + ry[i].y * a.y + ry[i].z * b.x + ry[i].w * b.y;
            }
            put4<3>(sm + M::Y, PAN, (pr + 32 * i) * LDE + pc, ry[i]);
            put4<3>(sm + M::V, PAN, (pr + 32 * i) * LDE + pc, rv[i]);
        }
#pragma unroll
        for (int i = 0; i < K / 32; ++i) {
            ss += rs[i].x * rd[i].x + rs[i].y * rd[i].y + rs[i].z * rd[i].z + rs[i].w * rd[i].w;
            put4<3>(sm + M::S0, K * LDE, (pr + 32 * i) * LDE + pc, rs[i]);
            put4<3>(sm + M::DS, K * LDE, (pr + 32 * i) * LDE + pc, rd[i]);
        }
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll 1
        for (int e = 0; e < EP; e += 16) {
            uint32_t fo[P][4], fy[3][4], fv[3][4];
#pragma unroll
            for (int i = 0; i < P; ++i) a_frag<LDE>(fo[i], sa + 2 * (M::DO + i * PAN), 16 * rb, e, lane);
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                a_frag<LDE>(fy[i], sa + 2 * (M::Y + i * PAN), 16 * rb, e, lane);
                a_frag<LDE>(fv[i], sa + 2 * (M::V + i * PAN), 16 * rb, e, lane);
            }
#pragma unroll
            for (int j = 0; j < NK / 2; ++j) {
                uint32_t b[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag<LDE>(b[i], sa + 2 * (M::S0 + i * K * LDE), half * (K / 2) + 16 * j, e, lane);
                mma_parts<P, 3, 3>(F, j, fo, b);
                mma_parts<3, 3, 3>(E, j, fy, b);
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag<LDE>(b[i], sa + 2 * (M::DS + i * K * LDE), half * (K / 2) + 16 * j, e, lane);
                mma_parts<3, 3, 3>(H, j, fv, b);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (2 * half + j > rb) break;
                uint32_t b[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag<LDE>(b[i], sa + 2 * (M::V + i * PAN), 32 * half + 16 * j, e, lane);
                mma_parts<P, 3, 3>(dA, j, fo, b);
                mma_parts<3, 3, 3>(dL, j, fy, b);
            }
        }
    }
    float qk[4][4], kk[4][4];
    grad_rows_products(m, rb, half, lane, qk, kk);
    // Y . v: eight lanes have a row
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) yv[i] += __shfl_xor_sync(0xffffffffu, yv[i], o);
        if ((tid & 7) == 0) red[R_Y * C + pr + 32 * i] = yv[i];
    }
    ss = warp_sum(ss);
    if (lane == 0) red[RED * C + w] = ss;
    __syncthreads();  // the panels have been used
    grad_pairs<T, K>(m, p.scale, rb, half, lane, dA, dL, qk, kk);
    grad_scale(m, p.scale, rb, half, lane, F, E, H);
    float total = 0.f;
    for (int i = 0; i < 8; ++i) total += red[RED * C + i];
    grad_finish<T, K>(p, lay, m, ci, unit, h, kh, grp, total, F, E, w, lane);
}

// dq and dk of shared key heads: the shares of a group's value heads in their order, then the gradient of the L2 norm.  A warp per
// (row, key head).
// two or four consecutive values
template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 v = load2(p + i);
        x[i] = v.x; x[i + 1] = v.y;
    }
}
template <>
__device__ __forceinline__ void load_row<4>(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <int N>
__device__ __forceinline__ void load_row(const bf16* p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 v = load2(p + i);
        x[i] = v.x; x[i + 1] = v.y;
    }
}
template <typename T, int K>
__global__ void __launch_bounds__(256) gdr_heads_kernel(const KdaGdrParams p, const Layout lay) {
    constexpr int N = K / 32, R = 4;
    const int lane = threadIdx.x & 31, grp = p.HV / p.H;
    const int b = gridDim.x - 1 - blockIdx.x, c = b / p.H, kh = b % p.H;  // what was written last is still in L2
    pdl_wait();
    const ChunkInfo ci = chunk_info(p, c);
    const float* aux = reinterpret_cast<const float*>(static_cast<const char*>(p.workspace) + lay.aux) + ((size_t)c * p.HV + kh * grp) * AUX;
    const float* in = reinterpret_cast<const float*>(static_cast<const char*>(p.bwd_scratch) + lay.dqk) + ((size_t)c * p.HV + kh * grp) * 2 * C * K;
    // a warp has R rows at a time, q's and k's in turn, all of their loads on the way before the first is used
    for (int x0 = (threadIdx.x >> 5) * R; x0 < 2 * ci.len; x0 += 8 * R) {
        float s[R][N], xv[R][N];
#pragma unroll
        for (int y = 0; y < R; ++y) {
            const int x = min(x0 + y, 2 * ci.len - 1), r = x >> 1, which = x & 1;
            load_row(in + (size_t)which * C * K + r * K + N * lane, s[y]);
            load_row(static_cast<const T*>(which ? p.k : p.q) + (((size_t)ci.tok0 + r) * p.H + kh) * K + N * lane, xv[y]);
        }
        for (int hg = 1; hg < grp; ++hg) {
            float v[R][N];
#pragma unroll
            for (int y = 0; y < R; ++y) {
                const int x = min(x0 + y, 2 * ci.len - 1);
                load_row(in + ((size_t)hg * 2 + (x & 1)) * C * K + (x >> 1) * K + N * lane, v[y]);
            }
#pragma unroll
            for (int y = 0; y < R; ++y)
#pragma unroll
                for (int i = 0; i < N; ++i) s[y][i] += v[y][i];
        }
#pragma unroll
        for (int y = 0; y < R; ++y) {
            const int x = x0 + y, r = x >> 1, which = x & 1;
            if (x >= 2 * ci.len) break;
            float f = 0.f;
            if (p.flags & KDA_FLAG_QK_L2NORM) {
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) dot = fmaf(xv[y][i], s[y][i], dot);
                const float inv = aux[(which ? A_RK : A_RQ) * C + r];
                f = inv < 1e6f ? inv * inv * warp_sum(dot) : 0.f;
            }
            T* out = static_cast<T*>(which ? p.grad_k : p.grad_q) + (((size_t)ci.tok0 + r) * p.H + kh) * K + N * lane;
#pragma unroll
            for (int i = 0; i < N; i += 2) store2(out + i, s[y][i] - xv[y][i] * f, s[y][i + 1] - xv[y][i + 1] * f);
        }
    }
}

// dA_log and ddt_bias: the units' shares of a value head, in a fixed order and in 64 bits
__global__ void __launch_bounds__(256) gdr_param_kernel(const KdaGdrParams p, const Layout lay) {
    __shared__ double s[2][256];
    const int h = blockIdx.x;
    pdl_wait();
    const float2* part = reinterpret_cast<const float2*>(static_cast<const char*>(p.bwd_scratch) + lay.part);
    double a = 0.0, b = 0.0;
    for (int c = threadIdx.x; c < p.NT; c += 256) {
        const float2 x = part[(size_t)c * p.HV + h];
        a += x.x;
        b += x.y;
    }
    s[0][threadIdx.x] = a;
    s[1][threadIdx.x] = b;
    for (int o = 128; o > 0; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o) {
            s[0][threadIdx.x] += s[0][threadIdx.x + o];
            s[1][threadIdx.x] += s[1][threadIdx.x + o];
        }
    }
    if (threadIdx.x == 0) {
        p.grad_A_log[h] = (float)s[0][0];
        if (p.grad_dt_bias) p.grad_dt_bias[h] = (float)s[1][0];
    }
}

cudaError_t grad_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s);  // gdr_grad_tc.cu

template <typename T, int K>
static cudaError_t launch_grad(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = GradMap<T, K>::BYTES;
    static_assert(bytes <= 232448, "shared memory");
    cudaError_t e = cudaSuccess;
    if (on_tc(p)) {
        e = grad_tc(p, l, s);
    } else {
        e = allow_smem(gdr_grad_kernel<T, K>, bytes);
        if (e == cudaSuccess) e = launch_dependent(gdr_grad_kernel<T, K>, p.NT * p.HV, gr::NTHR, bytes, s, p, l);
    }
    if (e == cudaSuccess && p.HV != p.H) e = launch_dependent(gdr_heads_kernel<T, K>, p.NT * p.H, 256, 0, s, p, l);
    if (e == cudaSuccess && (p.flags & KDA_FLAG_GATE)) e = launch_dependent(gdr_param_kernel, p.HV, 256, 0, s, p, l);
    return e;
}

cudaError_t grad(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    if (p.dtype == KDA_DTYPE_F32) return p.dk == 64 ? launch_grad<float, 64>(p, l, s) : launch_grad<float, 128>(p, l, s);
    return p.dk == 64 ? launch_grad<bf16, 64>(p, l, s) : launch_grad<bf16, 128>(p, l, s);
}

}  // namespace gdr
}  // namespace kda
