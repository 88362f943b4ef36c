// Recurrent gated delta rule for decoding: a few tokens per (sequence, value head), FP32 state in and out, one decay per head.
//
//   e = beta (v - a S^T k)          S' = a S + k e^T          o = scale S'^T q = a S^T (scale q) + scale (q.k) e          a = e^g
//
// What bounds it: the state's HBM traffic (2 x 64 KB per unit at dk = dv = 128, read and written once however many tokens the call
// has) for many units, latency for few.  A warp owns R value columns with all their key channels and keeps them in registers over
// all tokens; both inner products come from the OLD state, so that one reduction across the lanes serves both.
//   * [dv][dk] states: a lane holds four consecutive key channels of every column (a row is one 512-byte line);
//   * [dk][dv] states: a lane holds four consecutive value columns at every (128 / lanes)th key channel.
// The tokens' prologue (L2 norm, gate, sigmoid) is evaluated once per CTA, a warp per token, into shared memory.
// 256 sequences of 12 heads (128 x 128, one token): 68 us, 5.9 TB/s, 92 % of a copy's rate.  One sequence of 6 heads: 8.5 us a call, of
// which the kernel is 4; five sequences of seven tokens: 9.1 us.
#include "gdr.cuh"
#include "kda_decode.cuh"

namespace kda {
namespace gdr {

namespace dec {
constexpr int NW = 4;     // warps per CTA
constexpr int TB = 16;    // tokens whose prologue is in shared memory at a time
// floats of one token's prologue: k, scale q, v, then a, beta, scale q.k, padding
__host__ __device__ constexpr int tok_floats(int K, int V) { return 2 * K + V + 4; }
}  // namespace dec

struct StepArgs {
    KdaGdrParams p;  // q, k, v, g, beta, A_log, dt_bias, o, sizes, types, flags, scale; B sequences of T tokens
    const float* state_in;
    float* state_out;
    int vec;         // rows of q, k, v start on a four-element boundary
};

template <typename T, int K, int V, bool VF, int R>
__global__ void __launch_bounds__(32 * dec::NW) gdr_recurrent_kernel(const StepArgs a) {
    using namespace dec;
    const KdaGdrParams& p = a.p;
    constexpr int LD = VF ? K / 4 : 128 / R;          // lanes along the key channels of one column
    constexpr int LE = 32 / LD;                       // lane groups along the value columns
    constexpr int NE = R / LE, ND = K / LD;           // columns and key channels a lane holds
    constexpr int BIT0 = VF ? 1 : LE;                 // lowest lane bit of the key-channel index
    static_assert(VF ? ND == 4 : NE == 4, "one 16-byte word per access");
    extern __shared__ __align__(16) float sm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int NP = V / (R * NW);                  // CTAs per (sequence, value head)
    const int nh = blockIdx.x / NP, h = nh % p.HV, n = nh / p.HV, kh = h / (p.HV / p.H);
    const int ld = VF ? lane & (LD - 1) : lane / LE, le = VF ? lane / LD : lane & (LE - 1);
    const int e0 = (blockIdx.x % NP * NW + warp) * R;
    auto col = [&](int i) { return VF ? e0 + le + LE * i : e0 + 4 * le + i; };
    auto chn = [&](int j) { return VF ? 4 * ld + j : ld + LD * j; };
    const size_t sbase = (size_t)nh * K * V;
    pdl_wait();

    float S[NE][ND];  // requested first; it arrives behind the prologue
    if (a.state_in) {
        if constexpr (VF) {
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const float4 x = __ldcs(reinterpret_cast<const float4*>(a.state_in + sbase + (size_t)col(i) * K + 4 * ld));
                S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < ND; ++j) {
                const float4 x = __ldcs(reinterpret_cast<const float4*>(a.state_in + sbase + (size_t)chn(j) * V + e0 + 4 * le));
                S[0][j] = x.x; S[1][j] = x.y; S[2][j] = x.z; S[3][j] = x.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < ND; ++j) S[i][j] = 0.f;
    }
    constexpr int PK = K / 32, PV = V / 32;           // prologue: consecutive channels per lane
    for (int t0 = 0; t0 < p.T; t0 += TB) {
        const int nt = min(TB, p.T - t0);
        if (t0) __syncthreads();                      // the previous tokens' prologue has been consumed
        for (int t = warp; t < nt; t += NW) {
            const size_t tok = (size_t)n * p.T + t0 + t, krow = (tok * p.H + kh) * K, vrow = tok * p.HV + h;
            float qv[PK], kv[PK], vv[PV];
            load_row(static_cast<const T*>(p.q) + krow + PK * lane, qv, a.vec);
            load_row(static_cast<const T*>(p.k) + krow + PK * lane, kv, a.vec);
            load_row(static_cast<const T*>(p.v) + vrow * V + PV * lane, vv, a.vec);
            float b = load_g(p, p.beta, vrow);
            const float al = expf(log_decay(p, vrow, h));
            float sq = 0.f, sk = 0.f, qk = 0.f;
#pragma unroll
            for (int i = 0; i < PK; ++i) {
                sq = fmaf(qv[i], qv[i], sq);
                sk = fmaf(kv[i], kv[i], sk);
                qk = fmaf(qv[i], kv[i], qk);
            }
            float iq = p.scale, ik = 1.f;
            if (p.flags & KDA_FLAG_QK_L2NORM) {
                iq *= 1.f / fmaxf(sqrtf(warp_sum(sq)), 1e-6f);
                ik = 1.f / fmaxf(sqrtf(warp_sum(sk)), 1e-6f);
            }
            qk = warp_sum(qk) * iq * ik;
            float* s = sm + t * tok_floats(K, V);
#pragma unroll
            for (int i = 0; i < PK; ++i) {
                s[PK * lane + i] = kv[i] * ik;
                s[K + PK * lane + i] = qv[i] * iq;
            }
#pragma unroll
            for (int i = 0; i < PV; ++i) s[2 * K + PV * lane + i] = vv[i];
            if (p.flags & KDA_FLAG_BETA_SIGMOID) b = sigmoid_f(b);
            if (lane == 0) *reinterpret_cast<float4*>(s + 2 * K + V) = make_float4(al, b, qk, 0.f);
        }
        __syncthreads();
#pragma unroll 1
        for (int t = 0; t < nt; ++t) {
            const float* s = sm + t * tok_floats(K, V);
            const float4 num = *reinterpret_cast<const float4*>(s + 2 * K + V);  // a, beta, scale q.k
            float dot[2 * NE], kk[ND];
#pragma unroll
            for (int i = 0; i < 2 * NE; ++i) dot[i] = 0.f;
            if constexpr (VF) {
                float qa[4];
                load_n(s + 4 * ld, kk);
                load_n(s + K + 4 * ld, qa);
#pragma unroll
                for (int i = 0; i < NE; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        dot[i] = fmaf(kk[j], S[i][j], dot[i]);
                        dot[NE + i] = fmaf(qa[j], S[i][j], dot[NE + i]);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < ND; ++j) {
                    const float qa = s[K + chn(j)];
                    kk[j] = s[chn(j)];
#pragma unroll
                    for (int i = 0; i < NE; ++i) {
                        dot[i] = fmaf(kk[j], S[i][j], dot[i]);
                        dot[NE + i] = fmaf(qa, S[i][j], dot[NE + i]);
                    }
                }
            }
            int which = 0;
            TransposeSum<2 * NE, LD, BIT0>::run(dot, lane, which);
            // `which` = NE * (0: prediction, 1: output) + column; the lane bit BIT0 tells the two kinds apart
            static_assert(2 * NE <= LD, "every lane ends with exactly one value");
            const bool is_out = lane & BIT0;
            const int mine = col(which & (NE - 1));
            const float err = num.y * (s[2 * K + mine] - num.x * dot[0]);
            const float pair = __shfl_xor_sync(0xffffffffu, err, BIT0);
            // the first 2 NE reduction lanes hold all values, the others copies
            if (is_out && ld < 2 * NE)
                stf(static_cast<T*>(p.o) + (((size_t)n * p.T + t0 + t) * p.HV + h) * V + mine, fmaf(num.z, pair, num.x * dot[0]));
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                // lane that holds the prediction of this lane's column i: reduction bits = column index, lowest bit last
                int src = 0;
#pragma unroll
                for (int m = NE / 2, b = 2; m >= 1; m >>= 1, b <<= 1) src |= (i & m) ? b * BIT0 : 0;
                src |= VF ? lane & ~(LD - 1) : lane & (LE - 1);
                const float ei = __shfl_sync(0xffffffffu, err, src);
#pragma unroll
                for (int j = 0; j < ND; ++j) S[i][j] = fmaf(num.x, S[i][j], kk[j] * ei);
            }
        }
    }
    if (!a.state_out) return;
    if constexpr (VF) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
            __stcs(reinterpret_cast<float4*>(a.state_out + sbase + (size_t)col(i) * K + 4 * ld), make_float4(S[i][0], S[i][1], S[i][2], S[i][3]));
    } else {
#pragma unroll
        for (int j = 0; j < ND; ++j)
            __stcs(reinterpret_cast<float4*>(a.state_out + sbase + (size_t)chn(j) * V + e0 + 4 * le), make_float4(S[0][j], S[1][j], S[2][j], S[3][j]));
    }
}

template <typename T, int K, int V, bool VF, int R>
static cudaError_t launch(const StepArgs& a, cudaStream_t s) {
    const int tb = a.p.T < dec::TB ? a.p.T : dec::TB;
    return launch_dependent(gdr_recurrent_kernel<T, K, V, VF, R>, a.p.B * a.p.HV * (V / (R * dec::NW)), 32 * dec::NW,
                            (size_t)tb * dec::tok_floats(K, V) * sizeof(float), s, a);
}

// Columns per warp: eight give short chains per token and twice the CTAs, sixteen half the prologues and, for [dk][dv] states, 64
// instead of 32 consecutive bytes per access: eight until every SM has 64 KB of [dv][dk] states, or 16 KB of [dk][dv] states.
template <typename T, int K, int V>
static cudaError_t launch_columns(const StepArgs& a, cudaStream_t s) {
    const bool vf = a.p.flags & KDA_FLAG_STATE_V_FIRST;
    if ((long long)a.p.B * a.p.HV * K * V < (vf ? 16384LL : 4096LL) * sm_count())
        return vf ? launch<T, K, V, true, 8>(a, s) : launch<T, K, V, false, 8>(a, s);
    return vf ? launch<T, K, V, true, 16>(a, s) : launch<T, K, V, false, 16>(a, s);
}
template <typename T>
static cudaError_t launch_sizes(const StepArgs& a, cudaStream_t s) {
    if (a.p.dk == 64) return a.p.dv == 64 ? launch_columns<T, 64, 64>(a, s) : launch_columns<T, 64, 128>(a, s);
    return a.p.dv == 64 ? launch_columns<T, 128, 64>(a, s) : launch_columns<T, 128, 128>(a, s);
}

}  // namespace gdr
}  // namespace kda

extern "C" int kda_gdr_recurrent_fwd(const void* q, const void* k, const void* v, const void* g, const void* beta, const float* A_log,
                                     const float* dt_bias, const float* state_in, float* state_out, void* o, int32_t N, int32_t T,
                                     int32_t H, int32_t HV, int32_t dk, int32_t dv, int32_t dtype, int32_t g_dtype, int32_t flags,
                                     float scale, void* stream) {
    using namespace kda;
    if (!q || !k || !v || !g || !beta || !o || ((flags & KDA_FLAG_GATE) && !A_log)) return KDA_ERR_NULL;
    if (N <= 0 || T <= 0 || H <= 0 || HV <= 0 || HV % H || (dk != 64 && dk != 128) || (dv != 64 && dv != 128)) return KDA_ERR_SHAPE;
    if ((long long)N * HV > 0x7fffffffLL / 8) return KDA_ERR_SHAPE;  // (at most four CTAs per unit)
    for (int t : {dtype, g_dtype})
        if (t != KDA_DTYPE_F32 && t != KDA_DTYPE_BF16) return KDA_ERR_DTYPE;
    if (((uintptr_t)state_in | (uintptr_t)state_out) & 15) return KDA_ERR_ALIGN;
    gdr::StepArgs a = {};
    a.p.B = N; a.p.T = T; a.p.H = H; a.p.HV = HV; a.p.dk = dk; a.p.dv = dv; a.p.dtype = dtype; a.p.g_dtype = g_dtype;
    a.p.flags = flags; a.p.scale = scale;
    a.p.q = q; a.p.k = k; a.p.v = v; a.p.g = g; a.p.beta = beta; a.p.A_log = A_log; a.p.dt_bias = dt_bias; a.p.o = o;
    a.state_in = state_in; a.state_out = state_out;
    a.vec = (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) & (dtype == KDA_DTYPE_F32 ? 15 : 7)) == 0;
    const cudaError_t e = dtype == KDA_DTYPE_F32 ? gdr::launch_sizes<float>(a, (cudaStream_t)stream)
                                                 : gdr::launch_sizes<__nv_bfloat16>(a, (cudaStream_t)stream);
    return e == cudaSuccess ? KDA_OK : fail_cuda(e);
}
