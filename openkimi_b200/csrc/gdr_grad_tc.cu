// Gated delta rule, backward: the gradients of a chunk on tcgen05, from the records that the transposed walks leave (gdr_tc.cu).  The
// formulas stand in gdr_grad.cu; here
//   F^T = S0 do^T   E^T = S0 Y^T   H^T = dS V'^T  [128 x 64]      dA^T = V' do^T   dL^T = V' Y^T  [64 x 64]
// are products over the 128 value columns in K-steps of 16, and then
//   dq^T = F^T scaled + k^T Z^T       dk^T = E^T and H^T scaled + k^T X^T + k^T X + q^T Z
// with the key channels as the 128 lanes, so that products with the states run at M = 128.  What L2 norm's gradient needs of q . dq and
// k . dk comes from the same sums as dG: q . F, k . E, k . H, and rows and columns of Z (q k^T) and X (k k^T).
//
// One CTA per SM walks the (chunk, value head) units.  Eight warps read the records, take <S0, dS> and leave three BF16 parts in a ring
// of two K-steps (a warp asks L2 for the next unit's meanwhile); one issues the products; one brings the next unit's rows; sixteen do
// the rest of a unit while the next unit's accumulators fill; one the gradients of gate and beta.  16 x 2048 tokens of 6 heads take
// 350 us (732 on mma.sync): 375 KB of records, rows and gradients per unit, 3.3 TB/s, half of the copy's rate.  What bounds it is the
// pipe of shared memory and L1: the records in, their parts out (1.5 times the bytes), the MMAs' operands, the exchange of rows and
// columns and the main warps' spills; twice the warps for either part gained nothing, 88 registers instead of 80 for the main ones 5 %.
// An MMA whose A operand lies in shared memory takes N / 2 + 43 cycles here (M = 128; M = 64: N / 2 + 27), so do and the parts of Y lie
// side by side and go through as one operand of up to 192 columns.  Loads from tensor memory wait for the MMAs issued before them, so a
// unit's accumulators are read at once, before the next unit's first K-step, and the last products of a unit slip in between two
// K-steps of the next.
// Records of two BF16 parts take the same bytes and no conversion, but dg is a difference of larger sums: 2e-5 off for 15 tokens.
#include "gdr.cuh"

namespace kda {
namespace gdr {

namespace gt {
constexpr int MAIN = 512, CONV = 256, NTHR = 896, RING = 2, K = 128;
constexpr int W_CONV = MAIN / 32, W_MMA = W_CONV + CONV / 32, W_ROWS = W_MMA + 1, W_COPY = W_ROWS + 1;  // the other warps; the last is the gate's
// registers of the main, converting and other warps; 16 x 88 + 8 x 56 + 4 x 40 = 28 x 72 a lane
constexpr int REG_MAIN = 88, REG_CONV = 56, REG_REST = 40;
constexpr uint32_t MAT = SQ * 2;
// the rows of a unit: q, k as two halves of 64 columns with 128-byte swizzle
constexpr uint32_t Q = 0, KK = 16384, AU = 32768, TILE = AU + AUX * 4;
// a K-step: three parts each of S0, dS [16][128]; of V' the parts side by side [16][3 x 64]; do and the parts of Y one after the other
// [4 x 64][16], all in core-matrix order
constexpr uint32_t SPART = 4096, YPART = 2048, S0 = 0, DS = 3 * SPART, V = 6 * SPART, B = V + 6144, STAGE = B + 4 * YPART;
// Z^T, X^T: two parts each in core-matrix order, then dq and dk as rows
constexpr uint32_t R0 = 2 * TILE, Z = R0 + RING * STAGE, X = Z + 2 * MAT, RED = X + 2 * MAT, DOTS = RED + 12 * C * 4,
                   SUMN = DOTS + 12 * C * 4, TOTAL = SUMN + 8 * C * 8;
static_assert(TOTAL <= 232448 - 1024 && TILE % 1024 == 0, "fits");
// tensor memory columns; E^T in two halves that are added up (products with the first and the second part of Y)
constexpr uint32_t T_F = 0, T_E = 64, T_H = 192, T_DA = 256, T_DL = 320, T_DQ = 384, T_DK = 448;
// sums over 64 x 64 matrices with rows i, columns j: over rows i by block of j: Z qk^T (4), dL KKD (4); diagonals of Z qk^T and of
// Y V'^T; the factors of q and k in the gradient of the L2 norm
enum { R_ZQ = 0, R_B = 4, R_DZ = 8, R_DY = 9, R_CQ = 10, R_CK = 11 };
// the same in 64 bits: of N over columns j by block of i (4), over rows i by block of j (4).  In dG's running sum a pair of rows cancels
// between its row and its column: with sums in FP32 their rounding was left, 4e-6 of dA_log's terms at decays of e^-0.3 to e^-32.
enum { N_COL = 0, N_ROW = 4 };
}  // namespace gt

// 16 lanes x 16 consecutive columns as fragments: f[i] is (row g, columns 8 i + 2 t, + 1), (row g + 8, the same)
__device__ __forceinline__ void tmem_frag2(uint32_t at, float (&f)[2][4]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(f[0][0]), "=f"(f[0][1]), "=f"(f[0][2]), "=f"(f[0][3]), "=f"(f[1][0]), "=f"(f[1][1]), "=f"(f[1][2]), "=f"(f[1][3])
                 : "r"(at)
                 : "memory");
}
// 16 consecutive columns of this thread's lane
__device__ __forceinline__ void tmem_row16(uint32_t at, float (&x)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]), "=f"(x[8]), "=f"(x[9]),
                   "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
                 : "r"(at)
                 : "memory");
}
// val[i] summed over the 32 lanes; lanes 2 i and 2 i + 1 end with value i in val[0]: the number of values a lane carries halves at
// every step
template <int M = 16, int O = 16>
__device__ __forceinline__ void lanes_total(float* val, int lane) {
    if constexpr (M > 1) {
        const bool up = lane & O;
#pragma unroll
        for (int i = 0; i < M / 2; ++i) {
            const float keep = up ? val[M / 2 + i] : val[i], send = up ? val[i] : val[M / 2 + i];
            val[i] = keep + __shfl_xor_sync(0xffffffffu, send, O);
        }
        lanes_total<M / 2, O / 2>(val, lane);
    } else {
        val[0] += __shfl_xor_sync(0xffffffffu, val[0], O);
    }
}
// A and B fragments of 16 rows from `row` on of a [64][128] tile with 128-byte swizzle, channels c..c + 15 (a_frag, b_frag)
__device__ __forceinline__ void swz_a_frag(uint32_t (&f)[4], uint32_t x, int row, int c, int lane) {
    ldsm(f, x + 2 * swz_bf16(row + (lane & 15), c + (lane >> 4) * 8));
}
__device__ __forceinline__ void swz_b_frag(uint32_t (&f)[4], uint32_t x, int row, int c, int lane) {
    ldsm(f, x + 2 * swz_bf16(row + (lane & 7) + (lane >> 4) * 8, c + ((lane >> 3) & 1) * 8));
}
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__global__ void __launch_bounds__(gt::NTHR, 1) gdr_grad_tc_kernel(const KdaGdrParams p, const Layout lay) {
    using namespace gt;
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t full[RING], empty[RING], tfull[2], tempty[2], accbar, accfree, zready, dqbar, dqfree, sums, gatefree;
    __shared__ uint32_t tmem_s;
    __shared__ float ss[2][CONV / 32];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (warp == 0) {
        tmem_alloc(&tmem_s, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < RING; ++i) {
            mbar_init(&full[i], CONV / 32);
            mbar_init(&empty[i], 1);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 3 + MAIN / 32);  // the last products, the gate's warp, the one that asks L2, the main ones
        }
        mbar_init(&accbar, 1 + CONV / 32);
        mbar_init(&accfree, MAIN / 32);
        mbar_init(&zready, MAIN / 32);
        mbar_init(&dqbar, 1);
        mbar_init(&dqfree, MAIN / 32);
        mbar_init(&sums, MAIN / 32);
        mbar_init(&gatefree, 1);
        mbar_fence_init();
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem0 = tmem_s;
    const int units = p.NT * p.HV, stride = gridDim.x, grp = p.HV / p.H;
    const char* ws = static_cast<const char*>(p.workspace);
    char* sc = static_cast<char*>(p.bwd_scratch);
    float* red = reinterpret_cast<float*>(dyn + RED);
    float* dots = reinterpret_cast<float*>(dyn + DOTS);  // q.F, k.E, k.H: [3][4 blocks of channels][64]
    auto dot = [&](int which, int r) {
        const float* x = dots + which * 4 * C + r;
        return (x[0] + x[C]) + (x[2 * C] + x[3 * C]);
    };
    double* sumN = reinterpret_cast<double*>(dyn + SUMN);
    auto rows = [&](const auto* of, int r) {  // sum over row r, the blocks of columns up to its own
        auto s = of[r];
#pragma unroll
        for (int j = 1; j < 4; ++j)
            if (j <= r >> 4) s += of[j * C + r];
        return s;
    };
    auto cols = [&](int r) {  // sum of N over column r, the blocks of rows from its own on
        double s = sumN[(N_COL + 3) * C + r];
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i >= r >> 4) s += sumN[(N_COL + i) * C + r];
        return s;
    };
    bool ok = true;
    if (warp < W_CONV) registers_up<REG_MAIN>();  // (one instruction for the four warps of a group)
    else if (warp < W_MMA) registers_down<REG_CONV>();
    else registers_down<REG_REST>();

    if (warp < MAIN / 32) {
        const int rb = warp & 3, ib = warp >> 2, g = lane >> 2, t = lane & 3, d = tid & 127, t0 = 16 * ib;
        const uint32_t tm = tmem0 + ((uint32_t)(rb * 32) << 16);
        bf16 *sZ = reinterpret_cast<bf16*>(dyn + Z), *sX = reinterpret_cast<bf16*>(dyn + X);
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV, kh = h / grp;
            const unsigned char* b = dyn + tb * TILE;
            const float* aux = reinterpret_cast<const float*>(b + AU);
            const float *be = aux + A_BETA * C, *rq = aux + A_RQ * C, *rk = aux + A_RK * C, *ghi = aux + A_GHI * C, *glo = aux + A_GLO * C;
            const bf16 *sq = reinterpret_cast<const bf16*>(b + Q), *sk = reinterpret_cast<const bf16*>(b + KK);
            const ChunkInfo ci = chunk_info(p, c);
            ok = mbar_wait(&tfull[tb], (it >> 1) & 1, p, 1 << 12) && ok;
            ok = bar_and(1, MAIN, ok);  // (also: the unit before is done with Z, X and the sums)
            if (!ok) break;
            // (a wait below that gives up finishes the unit with what there is, for the barriers' sake)
            const bool any = ib >= rb;  // rows j = 16 rb.. meet columns i = 16 ib.. from the diagonal on
            const bool tiny = __any_sync(0xffffffffu, (2 * lane < ci.len && fabsf(be[2 * lane]) <= 1e-18f) || (2 * lane + 1 < ci.len && fabsf(be[2 * lane + 1]) <= 1e-18f));
            float qk[2][4], kk[2][4];  // k_j . q_i, k_j . k_i
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) qk[j][i] = kk[j][i] = 0.f;
            if (any)
#pragma unroll 2
                for (int k = 0; k < K; k += 16) {
                    uint32_t fk[4], bq[4], bk[4];
                    swz_a_frag(fk, smem_u32(sk), 16 * rb, k, lane);
                    swz_b_frag(bq, smem_u32(sq), t0, k, lane);
                    swz_b_frag(bk, smem_u32(sk), t0, k, lane);
                    mma(qk[0], fk, bq[0], bq[1]);
                    mma(qk[1], fk, bq[2], bq[3]);
                    mma(kk[0], fk, bk[0], bk[1]);
                    mma(kk[1], fk, bk[2], bk[3]);
                }
            ok = mbar_wait(&accbar, it & 1, p, 1 << 13) && ok;
            tc_fence_after();
            // ---- everything out of the accumulators
            float fq[16], fk[16], hh[16], dA[2][4], dL[2][4];
            {
                tmem_row16(tm + T_E + t0, fk);
                tmem_row16(tm + T_E + 64 + t0, hh);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) fk[j] += hh[j];
                tmem_row16(tm + T_F + t0, fq);
                tmem_row16(tm + T_H + t0, hh);
                tmem_frag2(tm + T_DA + t0, dA);
                tmem_frag2(tm + T_DL + t0, dL);
                tmem_wait_ld();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&accfree);
            if (it > 0) ok = mbar_wait(&gatefree, (it - 1) & 1, p, 1 << 11) && ok;  // the sums of the unit before have been used
            if (any) {  // ---- pairs of rows: 16 rows j x 16 columns i
                const int r0 = 16 * rb + g;
                const float gj[2] = {ghi[r0], ghi[r0 + 8]}, lj[2] = {glo[r0], glo[r0 + 8]}, kj[2] = {rk[r0], rk[r0 + 8]};
                double cn[2] = {0.0, 0.0};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    double rn[2] = {0.0, 0.0};
                    float rz[2] = {0.f, 0.f}, rl[2] = {0.f, 0.f};
                    const int i0 = t0 + 8 * j + 2 * t;
                    const float2 gi = load2(ghi + i0), li = load2(glo + i0), qi = load2(rq + i0), ki = load2(rk + i0), bi = load2(be + i0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int jj = r0 + 8 * i;
                        float z[2], x[2];
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const int ii = i0 + y;
                            // e^(G_i - G_j) / |k_j|
                            const float e = ii >= jj ? expf((y ? gi.y : gi.x) - gj[i] + ((y ? li.y : li.x) - lj[i])) * kj[i] : 0.f;
                            const float b = y ? bi.y : bi.x;
                            z[y] = dA[j][2 * i + y] * (p.scale * (y ? qi.y : qi.x)) * e;
                            const float l = ii > jj ? -dL[j][2 * i + y] * (y ? ki.y : ki.x) * e : 0.f;
                            x[y] = l * b;
                            const float zq = z[y] * qk[j][2 * i + y], lk = l * kk[j][2 * i + y];
                            const float nn = ii > jj ? fmaf(b, lk, zq) : 0.f;
                            rz[y] += zq;
                            rl[y] += lk;
                            rn[y] += nn;
                            cn[i] += nn;
                            if (ii == jj) {
                                red[R_DZ * C + ii] = zq;
                                red[R_DY * C + ii] = dL[j][2 * i + y];
                            }
                        }
                        put<2>(sZ, SQ, cm_idx(jj, i0, C), z[0], z[1]);
                        put<2>(sX, SQ, cm_idx(jj, i0, C), x[0], x[1]);
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            rn[y] += __shfl_xor_sync(0xffffffffu, rn[y], o);
                            rz[y] += __shfl_xor_sync(0xffffffffu, rz[y], o);
                        }
                        if (g == 0) {
                            sumN[(N_ROW + rb) * C + i0 + y] = rn[y];
                            red[(R_ZQ + rb) * C + i0 + y] = rz[y];
                        }
                        if (tiny) {
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) rl[y] += __shfl_xor_sync(0xffffffffu, rl[y], o);
                            if (g == 0) red[(R_B + rb) * C + i0 + y] = rl[y];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) cn[i] += __shfl_xor_sync(0xffffffffu, cn[i], o);
                    if (t == 0) sumN[(N_COL + ib) * C + r0 + 8 * i] = cn[i];
                }
                fence_async_smem();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&zready);
            // ---- the products with the states: lane d, 16 rows
            uint32_t qk_d[16];  // q and k of this lane's channel
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int at = swz_bf16(t0 + j, d);
                qk_d[j] = reinterpret_cast<const uint16_t*>(sq)[at] | (uint32_t)reinterpret_cast<const uint16_t*>(sk)[at] << 16;
            }
            {   // one sum after the other: what is live is F, E, H, the rows and one sum's terms
                float s[16], *to = dots + rb * C + t0 + (lane >> 1);
                auto scaled = [&](float (&x)[16], int factor) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(aux + factor * C + t0 + j);
                        x[j] *= f.x; x[j + 1] *= f.y; x[j + 2] *= f.z; x[j + 3] *= f.w;
                    }
                };
                auto total = [&](int which) {
                    lanes_total(s, lane);
                    if (!(lane & 1)) to[which * 4 * C] = s[0];
                };
                scaled(fq, A_OQ);
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = fq[j] * __uint_as_float(qk_d[j] << 16);
                total(0);
                scaled(fk, A_GK);  // k.E
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = fk[j] * __uint_as_float(qk_d[j] & 0xffff0000u);
                total(1);
                scaled(hh, A_FK);  // k.H
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = hh[j] * __uint_as_float(qk_d[j] & 0xffff0000u);
                total(2);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(be + t0 + j);
                    fk[j] = hh[j] - f.x * fk[j]; fk[j + 1] = hh[j + 1] - f.y * fk[j + 1];
                    fk[j + 2] = hh[j + 2] - f.z * fk[j + 2]; fk[j + 3] = hh[j + 3] - f.w * fk[j + 3];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sums);
            bar_sync(1, MAIN);
            {   // these rows' factors in the gradient of the L2 norm (a row shorter than 1e-6 is divided by that, whatever its length); the
                // four warps of a block of rows write the same
                const int r = t0 + (lane & 15);
                float cq = 0.f, ck = 0.f;
                if (grp == 1 && (p.flags & KDA_FLAG_QK_L2NORM)) {
                    const float z = rows(red + R_ZQ * C, r), dz = red[R_DZ * C + r];
                    if (rq[r] < 1e6f) cq = rq[r] * rq[r] * (dot(0, r) + z);
                    if (rk[r] < 1e6f) ck = rk[r] * rk[r] * (dot(2, r) - be[r] * dot(1, r) + ((float)rows(sumN + N_ROW * C, r) - (z - dz)) + (float)cols(r) + dz);
                }
                red[R_CQ * C + r] = cq;
                red[R_CK * C + r] = ck;
                __syncwarp();
            }
            // ---- the other products
            ok = mbar_wait(&dqbar, it & 1, p, 1 << 14) && ok;
            tc_fence_after();
            {
                float s[16];
                tmem_row16(tm + T_DQ + t0, s);
                tmem_row16(tm + T_DK + t0, hh);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&dqfree);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 cq = *reinterpret_cast<const float4*>(red + R_CQ * C + t0 + j), ck = *reinterpret_cast<const float4*>(red + R_CK * C + t0 + j);
                    const float *a = &cq.x, *e = &ck.x;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        fq[j + x] += s[j + x] - a[x] * __uint_as_float(qk_d[j + x] << 16);
                        fk[j + x] += hh[j + x] - e[x] * __uint_as_float(qk_d[j + x] & 0xffff0000u);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[tb]);
            if (grp > 1) {  // the group's value heads are added up, and the L2 norm follows, in gdr_heads_kernel (R_CQ, R_CK are 0 then)
                float* out = reinterpret_cast<float*>(sc + lay.dqk) + (size_t)u * 2 * C * K + d;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    out[(t0 + j) * K] = fq[j];
                    out[C * K + (t0 + j) * K] = fk[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    sZ[(t0 + j) * K + d] = __float2bfloat16_rn(fq[j]);
                    sX[(t0 + j) * K + d] = __float2bfloat16_rn(fk[j]);
                }
                bar_sync(1, MAIN);
                const size_t row = ((size_t)ci.tok0 * p.H + kh) * K;
#pragma unroll
                for (int i = tid; i < 2 * C * 16; i += MAIN) {
                    const int r = (i >> 4) & (C - 1), cc = (i & 15) * 8;
                    bf16* dst = static_cast<bf16*>(i < C * 16 ? p.grad_q : p.grad_k) + row + (size_t)r * p.H * K + cc;
                    if (r < ci.len) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>((i < C * 16 ? sZ : sX) + r * K + cc);
                }
            }
        }
    } else if (warp < (MAIN + CONV) / 32) {
        const int t = tid - MAIN, t7 = t & 127, row = t7 >> 1, e8 = (t7 & 1) * 8;
        const bool first = t < 128;  // of V' (the others: of Y and do)
        float x[3][8];  // pieces of eight values: S0, dS, V' or Y
        uint4 od;       // of do
        const bf16* dsrc = nullptr;
        auto request = [&](int u, int k) {
            load8(reinterpret_cast<const float*>(ws + lay.S0) + (size_t)u * K * 128 + k * 16 * K + 8 * t, x[0]);
            load8(reinterpret_cast<const float*>(sc + lay.dS) + (size_t)u * K * 128 + k * 16 * K + 8 * t, x[1]);
            if (first) {
                load8(reinterpret_cast<const float*>(ws + lay.Vn) + (size_t)u * C * 128 + k * 16 * C + 8 * t, x[2]);
            } else {
                load8(reinterpret_cast<const float*>(sc + lay.Y) + ((size_t)u * C + row) * 128 + k * 16 + e8, x[2]);
                if (k == 0) {
                    const ChunkInfo ci = chunk_info(p, u / p.HV);
                    dsrc = row < ci.len ? static_cast<const bf16*>(p.grad_o) + (((size_t)ci.tok0 + row) * p.HV + u % p.HV) * 128 + e8 : nullptr;
                }
                od = dsrc ? *reinterpret_cast<const uint4*>(dsrc + k * 16) : make_uint4(0, 0, 0, 0);
            }
        };
        auto leave = [&](unsigned char* at, uint32_t part, const float (&v)[8]) {
            uint32_t w[4][3];
#pragma unroll
            for (int i = 0; i < 4; ++i) split(v[2 * i], v[2 * i + 1], w[i]);
#pragma unroll
            for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(at + i * part) = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
        };
        int step = 0;
        if ((int)blockIdx.x < units) request(blockIdx.x, 0);
        for (int u = blockIdx.x, it = 0; u < units && ok; u += stride, ++it) {
            float s = 0.f;
            for (int k = 0; k < 8; ++k, ++step) {
                const int st = step % RING;
                if (step >= RING) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((step / RING) & 1) ^ 1, p, 1 << 15));
                if (!ok) break;
                unsigned char* b = dyn + R0 + st * STAGE;
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(x[0][i], x[1][i], s);
                leave(b + S0 + 16 * t, SPART, x[0]);
                leave(b + DS + 16 * t, SPART, x[1]);
                if (first) {
                    leave(b + V + (t >> 6) * (3 * 1024) + 16 * (t & 63), 1024, x[2]);
                } else {
                    unsigned char* rows = b + gt::B + (row >> 3) * 256 + (t & 1) * 128 + (row & 7) * 16;
                    *reinterpret_cast<uint4*>(rows) = od;
                    leave(rows + YPART, YPART, x[2]);
                }
                if (k < 7) request(u, k + 1);
                else if (u + stride < units) request(u + stride, 0);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[st]);
            }
            s = warp_sum(s);
            if (lane == 0) {
                ss[it & 1][warp - W_CONV] = s;
                mbar_arrive(&accbar);
            }
            __syncwarp();
        }
    } else if (warp == W_MMA) {
        constexpr uint32_t id192 = make_idesc(128, 192, true, false), id128 = make_idesc(128, 128, true, false), id64 = make_idesc(128, 64, true, false),
                           idH = make_idesc(128, 64, true, true), idA = make_idesc(64, 128, true, false), idL = make_idesc(64, 64, true, false);
        auto wait = [&](uint64_t* bar, uint32_t parity, int what) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, p, what));
            tc_fence_after();
            return ok;
        };
        // the last products of unit `it`.  Z^T and X^T are upper triangular: as [K = j][N = i] K-step s meets columns from its own block
        // on, as [N = j][K = i] rows up to it.
        auto finish = [&](int it) {
            if ((it > 0 && !wait(&dqfree, (it - 1) & 1, 1 << 19)) || !wait(&zready, it & 1, 1 << 20)) return;
            const uint32_t tile = smem_u32(dyn + (it & 1) * TILE), z = smem_u32(dyn + Z), x = smem_u32(dyn + X);
            if (elect_one()) {
#pragma unroll
                for (int i = 1; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint64_t k_s = make_desc_sw128(tile + KK + s * 2048, 8192, 1024);
                        const uint32_t id = make_idesc(128, 64 - 16 * s, true, true);
                        mma_ss(tmem0 + T_DQ + 16 * s, k_s, make_desc(z + i * MAT + s * 2048 + s * 256, 1024, 128), id, i < 1 || s > 0);
                        mma_ss(tmem0 + T_DK + 16 * s, k_s, make_desc(x + i * MAT + s * 2048 + s * 256, 1024, 128), id, i < 1 || s > 0);
                    }
#pragma unroll
                for (int i = 1; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint32_t id = make_idesc(128, 16 * (s + 1), true, false);
                        mma_ss(tmem0 + T_DK, make_desc_sw128(tile + KK + s * 2048, 8192, 1024), make_desc(x + i * MAT + s * 256, 128, 1024), id, true);
                        mma_ss(tmem0 + T_DK, make_desc_sw128(tile + Q + s * 2048, 8192, 1024), make_desc(z + i * MAT + s * 256, 128, 1024), id, true);
                    }
                mma_commit(&dqbar);
                mma_commit(&tempty[it & 1]);
            }
            __syncwarp();
        };
        int step = 0, it = 0;
        for (int u = blockIdx.x; u < units && ok; u += stride, ++it) {
            if (it > 0 && !wait(&accfree, (it - 1) & 1, 1 << 17)) break;
            for (int k = 0; k < 8 && ok; ++k, ++step) {
                const int st = step % RING;
                if (k == 3 && it > 0) finish(it - 1);  // by now its pairs are there
                if (!wait(&full[st], (step / RING) & 1, 1 << 18)) break;
                const uint32_t b = smem_u32(dyn + R0 + st * STAGE);
                if (elect_one()) {
                    uint64_t S[3], D[3], W[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        S[i] = make_desc(b + S0 + i * SPART, 2048, 128);
                        D[i] = make_desc(b + DS + i * SPART, 2048, 128);
                        W[i] = make_desc(b + V + i * 1024, 3 * 1024, 128);
                    }
                    const uint64_t dO = make_desc(b + gt::B, 128, 256), Y0 = make_desc(b + gt::B + YPART, 128, 256),
                                   Y1 = make_desc(b + gt::B + 2 * YPART, 128, 256), Y2 = make_desc(b + gt::B + 3 * YPART, 128, 256);
                    const bool acc = k > 0;
                    // [do | Y0 | Y1] and [do | Y0] are read from dO on; products of the smallest parts first
                    mma_ss(tmem0 + T_F, S[1], dO, id192, acc);
                    mma_ss(tmem0 + T_F, S[2], dO, id128, true);
                    mma_ss(tmem0 + T_E + 64, S[0], Y2, id64, true);
                    mma_ss(tmem0 + T_F, S[0], dO, id192, true);
                    mma_ss(tmem0 + T_H, D[2], W[0], idH, acc);
                    mma_ss(tmem0 + T_H, D[1], W[1], idH, true);
                    mma_ss(tmem0 + T_H, D[0], W[2], idH, true);
                    mma_ss(tmem0 + T_H, D[1], W[0], idH, true);
                    mma_ss(tmem0 + T_H, D[0], W[1], idH, true);
                    mma_ss(tmem0 + T_H, D[0], W[0], idH, true);
                    mma_ss(tmem0 + T_DA, W[2], dO, idA, acc);
                    mma_ss(tmem0 + T_DL, W[1], Y1, idL, true);
                    mma_ss(tmem0 + T_DL, W[0], Y2, idL, true);
                    mma_ss(tmem0 + T_DA, W[1], dO, idA, true);
                    mma_ss(tmem0 + T_DL, W[0], Y1, idL, true);
                    mma_ss(tmem0 + T_DA, W[0], dO, idA, true);
                    mma_commit(&empty[st]);
                    if (k == 7) mma_commit(&accbar);
                }
                __syncwarp();
            }
        }
        if (ok && it > 0) finish(it - 1);
    } else if (warp == W_ROWS) {
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV, kh = h / grp;
            unsigned char* b = dyn + tb * TILE;
            const ChunkInfo ci = chunk_info(p, c);
            if (it > 1) ok = __all_sync(0xffffffffu, mbar_wait(&tempty[tb], ((it >> 1) & 1) ^ 1, p, 1 << 21));
            if (!ok) break;
            const size_t qrow = ((size_t)ci.tok0 * p.H + kh) * K;
            load_cm<K, 32, true>(reinterpret_cast<bf16*>(b + Q), static_cast<const bf16*>(p.q) + qrow, (size_t)p.H * K, ci.len, lane);
            load_cm<K, 32, true>(reinterpret_cast<bf16*>(b + KK), static_cast<const bf16*>(p.k) + qrow, (size_t)p.H * K, ci.len, lane);
            load_words<32>(reinterpret_cast<bf16*>(b + AU), reinterpret_cast<const bf16*>(ws + lay.aux + (size_t)u * AUX * 4), AUX * 4 / 16, lane);
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tfull[tb]);
        }
    } else if (warp == W_COPY) {  // hints only, a unit ahead of the converters; counted in tempty, or it might miss a phase of tfull
        if (lane == 0)
            for (int u = blockIdx.x, it = 0; u + stride < units; u += stride, ++it) {
                ok = mbar_wait(&tfull[it & 1], (it >> 1) & 1, p, 1 << 9);
                if (!ok) break;
                mbar_arrive(&tempty[it & 1]);
                const size_t n = (size_t)u + stride;
                l2_prefetch_bulk(ws + lay.S0 + n * K * 512, K * 512);
                l2_prefetch_bulk(sc + lay.dS + n * K * 512, K * 512);
                l2_prefetch_bulk(ws + lay.Vn + n * C * 512, C * 512);
                l2_prefetch_bulk(sc + lay.Y + n * C * 512, C * 512);
            }
    } else {  // gradients of the gate and of beta, two neighbouring rows per lane
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV;
            const float *aux = reinterpret_cast<const float*>(dyn + tb * TILE + AU), *be = aux + A_BETA * C;
            const ChunkInfo ci = chunk_info(p, c);
            ok = __all_sync(0xffffffffu, mbar_wait(&sums, it & 1, p, 1 << 8));
            if (!ok) break;
            const float last = aux[A_LAST * C], total = ((ss[tb][0] + ss[tb][1]) + (ss[tb][2] + ss[tb][3])) + ((ss[tb][4] + ss[tb][5]) + (ss[tb][6] + ss[tb][7]));
            double dG[2], h1[2];
            float db[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 2 * lane + i;
                const float e = dot(1, r);
                dG[i] = rows(sumN + N_ROW * C, r) - cols(r) + dot(0, r) - (double)be[r] * e;
                h1[i] = dot(2, r);
                // Y_i . V'_i / beta_i; where beta_i is 0, or so small that the quotient means nothing, Y_i . v_i less what the chunk
                // predicts for v_i
                if (fabsf(be[r]) > 1e-18f) {
                    db[i] = red[R_DY * C + r] / be[r];
                } else {
                    const float* y = reinterpret_cast<const float*>(sc + lay.Y) + ((size_t)u * C + r) * 128;
                    float yv = 0.f;
                    if (r < ci.len) {
                        for (int x = 0; x < 128; ++x) yv = fmaf(y[x], ldf(static_cast<const bf16*>(p.v) + (((size_t)ci.tok0 + r) * p.HV + h) * 128 + x), yv);
                        yv += rows(red + R_B * C, r) - e;
                    }
                    db[i] = yv;
                }
            }
            const float2 dg = decay_gradients(dG, h1, (double)last * total, lane);
            gate_gradients(p, lay, ci, (size_t)u, h, dg.x, dg.y, db[0], db[1], be[2 * lane], be[2 * lane + 1], lane);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&gatefree);
                mbar_arrive(&tempty[tb]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem0, 512);
}

cudaError_t grad_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    cudaError_t e = allow_smem(gdr_grad_tc_kernel, gt::TOTAL);
    if (e != cudaSuccess) return e;
    const int units = p.NT * p.HV, sms = sm_count();
    return launch_dependent(gdr_grad_tc_kernel, units < sms ? units : sms, gt::NTHR, gt::TOTAL, s, p, l);
}

}  // namespace gdr
}  // namespace kda
