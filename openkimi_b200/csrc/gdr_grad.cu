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
#include "gdr_grad.cuh"

namespace kda {
namespace gdr {

namespace gr {
constexpr int NTHR = 256, EP = 32, LDE = EP + 8, PAN = C * LDE;
}

template <typename T, int K>
struct GradMap {
    static constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, ROWS = C * LDK;
    static constexpr int Q = 0, KK = P * ROWS, DO = 2 * P * ROWS, Y = DO + P * gr::PAN, V = Y + 3 * gr::PAN, S0 = V + 3 * gr::PAN,
                         DS = S0 + 3 * K * gr::LDE, END = DS + 3 * K * gr::LDE;
    static constexpr int Z = DO, X = Z + PO * C * gr::LDZ;  // over the panels, once they have been used
    static_assert(X + PO * C * gr::LDZ <= END, "Z and X fit");
    static constexpr int FLOATS = 7 * C + 16 * C;            // rows' numbers; sums over rows and columns
    static constexpr int BYTES = 2 * END + FLOATS * 4;
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
                              sx, sx + C, sx + 2 * C, sx + 3 * C, sx + 4 * C, sx + 5 * C, sx + 6 * C, red, aux[A_LAST * C]};

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
    grad_pairs(m, p.scale, rb, half, lane, dA, dL, qk, kk);
    grad_scale(m, p.scale, rb, half, lane, F, E, H);
    float total = 0.f;
    for (int i = 0; i < 8; ++i) total += red[RED * C + i];
    grad_finish(p, lay, m, ci, unit, h, kh, grp, total, F, E, w, lane, [] { __syncthreads(); });
}

// dq and dk of shared key heads: the shares of a group's value heads in their order, then the gradient of the L2 norm.  A warp per
// (row, key head).
template <typename T, int K>
__global__ void __launch_bounds__(256) gdr_heads_kernel(const KdaGdrParams p, const Layout lay) {
    constexpr int N = K / 32;
    const int lane = threadIdx.x & 31, grp = p.HV / p.H;
    const int c = blockIdx.x / p.H, kh = blockIdx.x % p.H;
    pdl_wait();
    const ChunkInfo ci = chunk_info(p, c);
    const float* aux = reinterpret_cast<const float*>(static_cast<const char*>(p.workspace) + lay.aux) + ((size_t)c * p.HV + kh * grp) * AUX;
    const float* in = reinterpret_cast<const float*>(static_cast<const char*>(p.bwd_scratch) + lay.dqk) + ((size_t)c * p.HV + kh * grp) * 2 * C * K;
    for (int x = threadIdx.x >> 5; x < 2 * ci.len; x += 8) {
        const int r = x >> 1, which = x & 1;  // q, k
        float s[N];
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = 0.f;
        for (int hg = 0; hg < grp; ++hg)
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 v = load2(in + ((size_t)hg * 2 + which) * C * K + r * K + N * lane + i);
                s[i] += v.x; s[i + 1] += v.y;
            }
        const size_t at = (((size_t)ci.tok0 + r) * p.H + kh) * K + N * lane;
        const T* row = static_cast<const T*>(which ? p.k : p.q) + at;
        T* out = static_cast<T*>(which ? p.grad_k : p.grad_q) + at;
        float xv[N], dot = 0.f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 v = load2(row + i);
            xv[i] = v.x; xv[i + 1] = v.y;
            dot += v.x * s[i] + v.y * s[i + 1];
        }
        float f = 0.f;
        if (p.flags & KDA_FLAG_QK_L2NORM) {
            const float inv = aux[(which ? A_RK : A_RQ) * C + r];
            f = inv < 1e6f ? inv * inv * warp_sum(dot) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; i += 2) store2(out + i, s[i] - xv[i] * f, s[i + 1] - xv[i + 1] * f);
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
