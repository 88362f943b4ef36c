// Gated delta rule, the walk along the chunks of a sequence: forward with the state, backward with its gradient.
//
//   forward   R = v - e^G (k^ S),  V' = T (beta R),  o = scale e^G (q^ S) + A V',  S <- e^G_last S + k^^T (e^(G_last - G) V')
//   backward  dV' = A^T do + e^(G_last - G) (k^ dS),  Y = T^T dV',  dv = beta Y,
//             dS <- e^G_last dS + q^^T (scale e^G do) - k^^T (e^G beta Y)
//
// The value columns of a state are independent, so a CTA of four warps walks VP of them for one (sequence, value head): the chain
// of a chunk gets shorter with VP and there are dv / VP times as many CTAs.  The panel of the state stays in registers, in the
// accumulators of its update (warp w: key channels w dk/4 ..), and goes to shared memory in three BF16 parts as the operand of the
// next chunk.  The next chunk's q, k, T, A (and do) are requested as soon as their other copy is free.
// Bound by the chain of a chunk: 6.3 us forward and 7.6 backward in FP32 (8 chunks of 64 key channels, 64 CTAs of 16 columns: 51 and
// 61 us).  BF16 with 128 channels and columns goes on tcgen05 (gdr_tc.cu).
#include "gdr.cuh"

namespace kda {
namespace gdr {

template <typename T, int K, int VP>
struct FwdMap {
    static constexpr int P = In<T>::P, PO = In<T>::PO, LDK = K + 8, LDE = VP + 8, STAGES = P == 1 ? 2 : 1;
    static constexpr int ROWS = C * LDK, Q = 0, KK = P * ROWS, TM = 2 * P * ROWS, AM = TM + 3 * TRI, STAGE = AM + PO * TRI;  // elements
    static constexpr int PAN = C * LDE, S = STAGES * STAGE, R = S + 3 * K * LDE, V = R + 3 * PAN, W = V + PO * PAN, END = W + 3 * PAN;
    static constexpr int BYTES = 2 * END;
};

template <typename T, int K, int VP, bool SAVE>
__global__ void __launch_bounds__(128) gdr_fwd_state_kernel(const KdaGdrParams p, const Layout lay) {
    using M = FwdMap<T, K, VP>;
    constexpr int P = M::P, PO = M::PO, LDK = M::LDK, LDE = M::LDE, NV = VP / 8, MT = K / 64;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* sm = reinterpret_cast<bf16*>(smem);
    const uint32_t sa = smem_u32(sm);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int panels = p.dv / VP, e0 = blockIdx.x % panels * VP, nh = blockIdx.x / panels, h = nh % p.HV, n = nh / p.HV, kh = h / (p.HV / p.H);
    pdl_wait();
    int c0, nc;
    long long tok_begin, tok_end;
    seq_chunks(p, n, c0, nc);
    seq_tokens(p, n, tok_begin, tok_end);
    const char* ws = static_cast<const char*>(p.workspace);

    float S[MT][NV][4];
    const int d0 = w * (K / 4) + g;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[m][j][i] = p.h0 ? p.h0[(size_t)nh * K * p.dv + state_at(p, d0 + 16 * m + 8 * (i >> 1), e0 + 8 * j + 2 * t + (i & 1))] : 0.f;

    auto request = [&](int c, int stage) {
        bf16* s = sm + stage * M::STAGE;
        const long long tok = tok_begin + (long long)c * C;
        const int rows = (int)min((long long)C, tok_end - tok);
        const size_t unit = (size_t)(c0 + c) * p.HV + h, row0 = (size_t)tok * p.H + kh;
        load_tile<K, LDK, 128>(s + M::KK, static_cast<const T*>(p.k) + row0 * K, (size_t)p.H * K, rows, tid);
        load_tile<K, LDK, 128>(s + M::Q, static_cast<const T*>(p.q) + row0 * K, (size_t)p.H * K, rows, tid);
        load_words<128>(s + M::TM, reinterpret_cast<const bf16*>(ws + lay.T) + unit * 3 * TRI, 3 * TRI / 8, tid);
        load_words<128>(s + M::AM, reinterpret_cast<const bf16*>(ws + lay.A) + unit * 3 * TRI, PO * TRI / 8, tid);
        cp_async_commit();
    };
    auto put_state = [&] {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                put<3>(sm + M::S, K * LDE, (d0 + 16 * m) * LDE + 8 * j + 2 * t, S[m][j][0], S[m][j][1]);
                put<3>(sm + M::S, K * LDE, (d0 + 16 * m + 8) * LDE + 8 * j + 2 * t, S[m][j][2], S[m][j][3]);
            }
    };
    if (nc > 0 && M::STAGES == 2) request(0, 0);
    put_state();
    const int r0 = 16 * w + g;
    for (int c = 0; c < nc; ++c) {
        const long long tok = tok_begin + (long long)c * C;
        const int rows = (int)min((long long)C, tok_end - tok);
        const size_t unit = (size_t)(c0 + c) * p.HV + h;
        const float* aux = reinterpret_cast<const float*>(ws + lay.aux) + unit * AUX;
        // this thread's rows
        float gam[2], fall[2], be[2], rk[2], rq[2];
        float2 v[2][NV];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            gam[i] = aux[A_GAM * C + r]; fall[i] = aux[A_FALL * C + r]; be[i] = aux[A_BETA * C + r];
            rq[i] = aux[A_RQ * C + r]; rk[i] = aux[A_RK * C + r];
            const T* src = static_cast<const T*>(p.v) + ((size_t)(tok + r) * p.HV + h) * p.dv + e0 + 2 * t;
#pragma unroll
            for (int j = 0; j < NV; ++j) v[i][j] = r < rows ? load2(src + 8 * j) : make_float2(0.f, 0.f);
        }
        const float last = aux[A_LAST * C];
        int stage = 0;
        if constexpr (M::STAGES == 2) {
            stage = c & 1;
            cp_async_wait<0>();
            __syncthreads();  // the chunk's rows and the state's parts are there; the other stage is free
            if (c + 1 < nc) request(c + 1, stage ^ 1);
        } else {
            __syncthreads();
            request(c, 0);
            cp_async_wait<0>();
            __syncthreads();
        }
        const uint32_t st = sa + 2 * stage * M::STAGE;
        if (SAVE) {
            float* S0 = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.S0) + unit * K * p.dv;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        store2(S0 + (size_t)(d0 + 16 * m + 8 * i) * p.dv + e0 + 8 * j + 2 * t, S[m][j][2 * i], S[m][j][2 * i + 1]);
        }
        float ks[NV][4], qs[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) ks[j][i] = qs[j][i] = 0.f;
#pragma unroll 2
        for (int d = 0; d < K; d += 16) {
            uint32_t fk[P][4], fq[P][4];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                a_frag<LDK>(fk[i], st + 2 * (M::KK + i * M::ROWS), 16 * w, d, lane);
                a_frag<LDK>(fq[i], st + 2 * (M::Q + i * M::ROWS), 16 * w, d, lane);
            }
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t b[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag_t<LDE>(b[i], sa + 2 * (M::S + i * K * LDE), 16 * j, d, lane);
                mma_parts<P, 3, 3>(ks, j, fk, b);
                mma_parts<P, 3, PO>(qs, j, fq, b);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float f = gam[i] * rk[i];
                put<3>(sm + M::R, M::PAN, (r0 + 8 * i) * LDE + 8 * j + 2 * t, be[i] * (v[i][j].x - f * ks[j][2 * i]),
                       be[i] * (v[i][j].y - f * ks[j][2 * i + 1]));
            }
        __syncthreads();
        float vn[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) vn[j][i] = 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b > w) break;
            uint32_t ft[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i) tri_frag(ft[i], st + 2 * (M::TM + i * TRI), blk(w, b), lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t x[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag_t<LDE>(x[i], sa + 2 * (M::R + i * M::PAN), 16 * j, 16 * b, lane);
                mma_parts<3, 3, 3>(vn, j, ft, x);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (r0 + 8 * i) * LDE + 8 * j + 2 * t;
                const float x = vn[j][2 * i], y = vn[j][2 * i + 1], f = fall[i] * rk[i];
                put<3>(sm + M::W, M::PAN, at, f * x, f * y);
                put<PO>(sm + M::V, M::PAN, at, x, y);
                if (SAVE)
                    store2(reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.Vn) + (unit * C + r0 + 8 * i) * p.dv + e0 + 8 * j + 2 * t, x, y);
            }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[m][j][i] *= last;
#pragma unroll
        for (int b = 0; b < C; b += 16) {
            uint32_t fk[MT][P][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < P; ++i) a_frag_t<LDK>(fk[m][i], st + 2 * (M::KK + i * M::ROWS), w * (K / 4) + 16 * m, b, lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t x[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag_t<LDE>(x[i], sa + 2 * (M::W + i * M::PAN), 16 * j, b, lane);
#pragma unroll
                for (int m = 0; m < MT; ++m) mma_parts<P, 3, 3>(S[m], j, fk[m], x);
            }
        }
        put_state();
        float o[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = p.scale * gam[i >> 1] * rq[i >> 1] * qs[j][i];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b > w) break;
            uint32_t fa[PO][4];
#pragma unroll
            for (int i = 0; i < PO; ++i) tri_frag(fa[i], st + 2 * (M::AM + i * TRI), blk(w, b), lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t x[PO][4];
#pragma unroll
                for (int i = 0; i < PO; ++i) b_frag_t<LDE>(x[i], sa + 2 * (M::V + i * M::PAN), 16 * j, 16 * b, lane);
                mma_parts<PO, PO, PO>(o, j, fa, x);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (r0 + 8 * i < rows) {
                T* dst = static_cast<T*>(p.o) + ((size_t)(tok + r0 + 8 * i) * p.HV + h) * p.dv + e0 + 2 * t;
#pragma unroll
                for (int j = 0; j < NV; ++j) store2(dst + 8 * j, o[j][2 * i], o[j][2 * i + 1]);
            }
    }
    if (p.ht) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    p.ht[(size_t)nh * K * p.dv + state_at(p, d0 + 16 * m + 8 * (i >> 1), e0 + 8 * j + 2 * t + (i & 1))] = S[m][j][i];
    }
}

template <typename T, int K, int VP>
struct BwdMap {
    static constexpr int P = In<T>::P, LDK = K + 8, LDE = VP + 8, STAGES = P == 1 ? 2 : 1;
    static constexpr int ROWS = C * LDK, PAN = C * LDE;
    static constexpr int Q = 0, KK = P * ROWS, TM = 2 * P * ROWS, AM = TM + 3 * TRI, DO = AM + 3 * TRI, STAGE = DO + P * PAN;
    static constexpr int S = STAGES * STAGE, X = S + 3 * K * LDE, W = X + 3 * PAN, END = W + 3 * PAN;  // X: dV', then e^G beta Y; W: scale e^G do
    static constexpr int BYTES = 2 * END;
};

template <typename T, int K, int VP>
__global__ void __launch_bounds__(128) gdr_bwd_state_kernel(const KdaGdrParams p, const Layout lay) {
    using M = BwdMap<T, K, VP>;
    constexpr int P = M::P, LDK = M::LDK, LDE = M::LDE, NV = VP / 8, MT = K / 64;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* sm = reinterpret_cast<bf16*>(smem);
    const uint32_t sa = smem_u32(sm);
    const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t = lane & 3;
    const int panels = p.dv / VP, e0 = blockIdx.x % panels * VP, nh = blockIdx.x / panels, h = nh % p.HV, n = nh / p.HV, kh = h / (p.HV / p.H);
    pdl_wait();
    int c0, nc;
    long long tok_begin, tok_end;
    seq_chunks(p, n, c0, nc);
    seq_tokens(p, n, tok_begin, tok_end);
    const char* ws = static_cast<const char*>(p.workspace);
    char* sc = static_cast<char*>(p.bwd_scratch);

    float S[MT][NV][4];
    const int d0 = w * (K / 4) + g;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[m][j][i] = p.grad_ht ? p.grad_ht[(size_t)nh * K * p.dv + state_at(p, d0 + 16 * m + 8 * (i >> 1), e0 + 8 * j + 2 * t + (i & 1))] : 0.f;

    auto request = [&](int c, int stage) {
        bf16* s = sm + stage * M::STAGE;
        const long long tok = tok_begin + (long long)c * C;
        const int rows = (int)min((long long)C, tok_end - tok);
        const size_t unit = (size_t)(c0 + c) * p.HV + h, row0 = (size_t)tok * p.H + kh;
        load_tile<K, LDK, 128>(s + M::KK, static_cast<const T*>(p.k) + row0 * K, (size_t)p.H * K, rows, tid);
        load_tile<VP, LDE, 128>(s + M::DO, static_cast<const T*>(p.grad_o) + ((size_t)tok * p.HV + h) * p.dv + e0, (size_t)p.HV * p.dv, rows, tid);
        load_words<128>(s + M::AM, reinterpret_cast<const bf16*>(ws + lay.A) + unit * 3 * TRI, 3 * TRI / 8, tid);
        load_words<128>(s + M::TM, reinterpret_cast<const bf16*>(ws + lay.T) + unit * 3 * TRI, 3 * TRI / 8, tid);
        load_tile<K, LDK, 128>(s + M::Q, static_cast<const T*>(p.q) + row0 * K, (size_t)p.H * K, rows, tid);
        cp_async_commit();
    };
    auto put_state = [&] {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                put<3>(sm + M::S, K * LDE, (d0 + 16 * m) * LDE + 8 * j + 2 * t, S[m][j][0], S[m][j][1]);
                put<3>(sm + M::S, K * LDE, (d0 + 16 * m + 8) * LDE + 8 * j + 2 * t, S[m][j][2], S[m][j][3]);
            }
    };
    if (nc > 0 && M::STAGES == 2) request(nc - 1, (nc - 1) & 1);
    put_state();
    const int r0 = 16 * w + g;
    for (int c = nc - 1; c >= 0; --c) {
        const long long tok = tok_begin + (long long)c * C;
        const int rows = (int)min((long long)C, tok_end - tok);
        const size_t unit = (size_t)(c0 + c) * p.HV + h;
        const float* aux = reinterpret_cast<const float*>(ws + lay.aux) + unit * AUX;
        float gam[2], fall[2], be[2], rk[2], rq[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i;
            gam[i] = aux[A_GAM * C + r]; fall[i] = aux[A_FALL * C + r]; be[i] = aux[A_BETA * C + r];
            rq[i] = aux[A_RQ * C + r]; rk[i] = aux[A_RK * C + r];
        }
        const float last = aux[A_LAST * C];
        int stage = 0;
        if constexpr (M::STAGES == 2) {
            stage = c & 1;
            cp_async_wait<0>();
            __syncthreads();
            if (c > 0) request(c - 1, stage ^ 1);
        } else {
            __syncthreads();
            request(c, 0);
            cp_async_wait<0>();
            __syncthreads();
        }
        const uint32_t st = sa + 2 * stage * M::STAGE;
        const bf16* sdo = sm + stage * M::STAGE + M::DO;
        {
            float* dS = reinterpret_cast<float*>(sc + lay.dS) + unit * K * p.dv;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        store2(dS + (size_t)(d0 + 16 * m + 8 * i) * p.dv + e0 + 8 * j + 2 * t, S[m][j][2 * i], S[m][j][2 * i + 1]);
        }
        float dv[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) dv[j][i] = 0.f;
#pragma unroll 2
        for (int d = 0; d < K; d += 16) {
            uint32_t fk[P][4];
#pragma unroll
            for (int i = 0; i < P; ++i) a_frag<LDK>(fk[i], st + 2 * (M::KK + i * M::ROWS), 16 * w, d, lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t b[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag_t<LDE>(b[i], sa + 2 * (M::S + i * K * LDE), 16 * j, d, lane);
                mma_parts<P, 3, 3>(dv, j, fk, b);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) dv[j][i] *= fall[i >> 1] * rk[i >> 1];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b < w) continue;
            uint32_t fa[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i) tri_frag_t(fa[i], st + 2 * (M::AM + i * TRI), blk(b, 0) + w, lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t x[P][4];
#pragma unroll
                for (int i = 0; i < P; ++i) b_frag_t<LDE>(x[i], st + 2 * (M::DO + i * M::PAN), 16 * j, 16 * b, lane);
                mma_parts<3, P, 3>(dv, j, fa, x);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (r0 + 8 * i) * LDE + 8 * j + 2 * t;
                put<3>(sm + M::X, M::PAN, at, dv[j][2 * i], dv[j][2 * i + 1]);
                const float2 x = get2<P>(sdo, M::PAN, at);
                const float f = p.scale * gam[i] * rq[i];
                put<3>(sm + M::W, M::PAN, at, f * x.x, f * x.y);
            }
        __syncthreads();
        float y[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[j][i] = 0.f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            if (b < w) continue;
            uint32_t ft[3][4];
#pragma unroll
            for (int i = 0; i < 3; ++i) tri_frag_t(ft[i], st + 2 * (M::TM + i * TRI), blk(b, 0) + w, lane);
#pragma unroll
            for (int j = 0; j < NV / 2; ++j) {
                uint32_t x[3][4];
#pragma unroll
                for (int i = 0; i < 3; ++i) b_frag_t<LDE>(x[i], sa + 2 * (M::X + i * M::PAN), 16 * j, 16 * b, lane);
                mma_parts<3, 3, 3>(y, j, ft, x);
            }
        }
        __syncthreads();  // X has been read
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = y[j][2 * i], b = y[j][2 * i + 1], f = -gam[i] * rk[i] * be[i];
                put<3>(sm + M::X, M::PAN, (r0 + 8 * i) * LDE + 8 * j + 2 * t, f * a, f * b);
                store2(reinterpret_cast<float*>(sc + lay.Y) + (unit * C + r0 + 8 * i) * p.dv + e0 + 8 * j + 2 * t, a, b);
                if (r0 + 8 * i < rows)
                    store2(static_cast<T*>(p.grad_v) + ((size_t)(tok + r0 + 8 * i) * p.HV + h) * p.dv + e0 + 8 * j + 2 * t, be[i] * a, be[i] * b);
            }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[m][j][i] *= last;
        auto add = [&](int rows_at, int pan_at) {  // S += rows^T panel
#pragma unroll
            for (int b = 0; b < C; b += 16) {
                uint32_t f[MT][P][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < P; ++i) a_frag_t<LDK>(f[m][i], st + 2 * (rows_at + i * M::ROWS), w * (K / 4) + 16 * m, b, lane);
#pragma unroll
                for (int j = 0; j < NV / 2; ++j) {
                    uint32_t x[3][4];
#pragma unroll
                    for (int i = 0; i < 3; ++i) b_frag_t<LDE>(x[i], sa + 2 * (pan_at + i * M::PAN), 16 * j, b, lane);
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma_parts<P, 3, 3>(S[m], j, f[m], x);
                }
            }
        };
        add(M::Q, M::W);
        __syncthreads();
        add(M::KK, M::X);
        put_state();
    }
    if (p.grad_h0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    p.grad_h0[(size_t)nh * K * p.dv + state_at(p, d0 + 16 * m + 8 * (i >> 1), e0 + 8 * j + 2 * t + (i & 1))] = S[m][j][i];
    }
}

template <typename T, int K, int VP, bool SAVE>
static cudaError_t launch_fwd(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = FwdMap<T, K, VP>::BYTES;
    static_assert(bytes <= 232448, "shared memory");
    cudaError_t e = allow_smem(gdr_fwd_state_kernel<T, K, VP, SAVE>, bytes);
    if (e != cudaSuccess) return e;
    return launch_dependent(gdr_fwd_state_kernel<T, K, VP, SAVE>, p.N * p.HV * (p.dv / VP), 128, bytes, s, p, l);
}
template <typename T, int K, int VP>
static cudaError_t launch_bwd(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = BwdMap<T, K, VP>::BYTES;
    static_assert(bytes <= 232448, "shared memory");
    cudaError_t e = allow_smem(gdr_bwd_state_kernel<T, K, VP>, bytes);
    if (e != cudaSuccess) return e;
    return launch_dependent(gdr_bwd_state_kernel<T, K, VP>, p.N * p.HV * (p.dv / VP), 128, bytes, s, p, l);
}

template <typename T, int K, int VP>
static cudaError_t fwd_saved(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    return p.flags & KDA_FLAG_NO_SAVE ? launch_fwd<T, K, VP, false>(p, l, s) : launch_fwd<T, K, VP, true>(p, l, s);
}

cudaError_t fwd_state(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    if (p.dtype == KDA_DTYPE_F32) return p.dk == 64 ? fwd_saved<float, 64, 16>(p, l, s) : fwd_saved<float, 128, 16>(p, l, s);
    return p.dk == 64 ? fwd_saved<bf16, 64, 32>(p, l, s) : fwd_saved<bf16, 128, 32>(p, l, s);
}
cudaError_t bwd_state(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    if (p.dtype == KDA_DTYPE_F32) return p.dk == 64 ? launch_bwd<float, 64, 16>(p, l, s) : launch_bwd<float, 128, 16>(p, l, s);
    return p.dk == 64 ? launch_bwd<bf16, 64, 32>(p, l, s) : launch_bwd<bf16, 128, 32>(p, l, s);
}

}  // namespace gdr
}  // namespace kda
