// Gated delta rule, backward: the gradients of a chunk on tcgen05, from the records that the transposed walks leave (gdr_tc.cu).  The
// formulas stand in gdr_grad.cu; here
//   F^T = S0 do^T   E^T = S0 Y^T   H^T = dS V'^T  [128 x 64]      dA = do V'^T   dL = Y V'^T  [64 x 64]
// are products over the 128 value columns in K-steps of 16, and then
//   dq^T = F^T scaled + k^T Z^T       dk^T = E^T and H^T scaled + k^T X^T + k^T X + q^T Z
// with the key channels as the 128 lanes, so that products with the states run at M = 128.  What L2 norm's gradient needs of q . dq and
// k . dk comes from the same sums as dG: q . F, k . E, k . H, and rows and columns of Z (q k^T) and X (k k^T).
//
// One CTA per SM walks the (chunk, value head) units.  What bounds it: 256 KB of records and rows per unit, 5.9 us of an SM's share
// of HBM, so everything runs beside the loads: four warps read the records (FP32, in the order in which a K-step wants them), take
// <S0, dS> and leave three BF16 parts in a ring of two K-steps; a warp issues the products; two bring the next unit's rows; eight do
// the rest of a unit while the next unit's accumulators fill.  Records of two BF16 parts take the same bytes and no conversion, but
// dg is a difference of larger sums: 2e-5 off for 15 tokens.
#include "gdr.cuh"

namespace kda {
namespace gdr {

namespace gt {
constexpr int MAIN = 256, CONV = 128, ROWS = 64, NTHR = MAIN + CONV + 32 + ROWS, RING = 2, K = 128;
constexpr uint32_t MAT = SQ * 2;
// the rows of a unit: q, k, do as two halves of 64 columns with 128-byte swizzle
constexpr uint32_t Q = 0, KK = 16384, DO = 32768, AU = 49152, TILE = AU + AUX * 4;
// a K-step: three parts each of S0, dS [16][128] and V', Y [16][64] in core-matrix order
constexpr uint32_t SPART = 4096, VPART = 2048, S0 = 0, DS = 3 * SPART, V = 6 * SPART, Y = V + 3 * VPART, STAGE = Y + 3 * VPART;
// Z, X: two parts each in core-matrix order, then dq and dk as rows
constexpr uint32_t R0 = 2 * TILE, Z = R0 + RING * STAGE, X = Z + 2 * MAT, RED = X + 2 * MAT, DOTS = RED + 14 * C * 4, TOTAL = DOTS + 12 * C * 4;
static_assert(TOTAL <= 231000 && TILE % 1024 == 0, "fits");
// tensor memory columns; q k^T and k k^T lie where dq and dk go later
constexpr uint32_t T_F = 0, T_E = 64, T_H = 128, T_DA = 192, T_DL = 256, T_DQ = 320, T_DK = 384;
// sums over rows or columns of the 64 x 64 matrices: of N (row halves 0, 1), Z qk^T (2), dL KKD (2); columns of N by row block (4);
// diagonals of Z qk^T and of Y V'^T; then the factors of q and k in the gradient of the L2 norm
enum { R_N = 0, R_ZQ = 2, R_B = 4, R_COL = 6, R_DZ = 10, R_DY = 11, R_CQ = 12, R_CK = 13 };
}  // namespace gt

// 16 lanes x 32 consecutive columns as fragments: registers 4 i .. 4 i + 3 are (row g, columns 8 i + 2 t, + 1), (row g + 8, the same)
__device__ __forceinline__ void tmem_frag4(uint32_t at, float (&f)[4][4]) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at)
                 : "memory");
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i][j] = __uint_as_float(r[4 * i + j]);
}
// 32 consecutive columns of this thread's lane
__device__ __forceinline__ void tmem_row32(uint32_t at, float (&x)[32]) {
    uint32_t r[2][16];
    tmem_ld16(at, r[0]);
    tmem_ld16(at + 16, r[1]);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(r[j >> 4][j & 15]);
}
// val[i] summed over the 32 lanes; lane l ends with value l in val[0]: the number of values a lane carries halves at every step
template <int M, int O = 16>
__device__ __forceinline__ void lanes_total(float* val, int lane) {
    if constexpr (O > 0) {
        const bool up = lane & O;
#pragma unroll
        for (int i = 0; i < M / 2; ++i) {
            const float keep = up ? val[M / 2 + i] : val[i], send = up ? val[i] : val[M / 2 + i];
            val[i] = keep + __shfl_xor_sync(0xffffffffu, send, O);
        }
        lanes_total<M / 2, O / 2>(val, lane);
    }
}
// K-major operand with 128-byte swizzle: rows of 64 elements (128 bytes), eight rows 1024 bytes; 16 elements along K are 32 bytes
__device__ __forceinline__ uint64_t desc_rows(uint32_t at, int kstep) { return make_desc_sw128(at + (kstep >> 2) * 8192 + (kstep & 3) * 32, 16, 1024); }

__global__ void __launch_bounds__(gt::NTHR, 1) gdr_grad_tc_kernel(const KdaGdrParams p, const Layout lay) {
    using namespace gt;
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t full[RING], empty[RING], tfull[2], tempty[2], accbar, accfree, zready, dqbar, dqfree;
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
            mbar_init(&tfull[i], ROWS / 32);
            mbar_init(&tempty[i], 1 + MAIN / 32);
        }
        mbar_init(&accbar, 1 + CONV / 32);
        mbar_init(&accfree, MAIN / 32);
        mbar_init(&zready, MAIN / 32);
        mbar_init(&dqbar, 1);
        mbar_init(&dqfree, MAIN / 32);
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
    bool ok = true;

    if (warp < MAIN / 32) {
        const int rb = warp & 3, half = warp >> 2, g = lane >> 2, t = lane & 3, d = tid & 127, t0 = 32 * half;
        const uint32_t tm = tmem0 + ((uint32_t)(rb * 32) << 16);
        float* red = reinterpret_cast<float*>(dyn + RED);
        float* dots = reinterpret_cast<float*>(dyn + DOTS);  // q.F, k.E, k.H: [3][4 blocks of channels][64]
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
            ok = mbar_wait(&accbar, it & 1, p, 1 << 13) && ok;
            tc_fence_after();
            {   // ---- pairs of rows: 16 rows x 32 columns
                float dA[4][4], dL[4][4], qk[4][4], kk[4][4];
                const bool any = 2 * half <= rb;
                if (any) {
                    tmem_frag4(tm + T_DA + 32 * half, dA);
                    tmem_frag4(tm + T_DL + 32 * half, dL);
                    tmem_frag4(tm + T_DQ + 32 * half, qk);
                    tmem_frag4(tm + T_DK + 32 * half, kk);
                }
                const int r0 = 16 * rb + g;
                float rn[2] = {0.f, 0.f}, rz[2] = {0.f, 0.f}, rl[2] = {0.f, 0.f};
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
                            const float e = r >= cc ? expf(ghi[r] - ghi[cc] + (glo[r] - glo[cc])) * rk[cc] : 0.f;
                            z[y] = r >= cc ? dA[j][2 * i + y] * p.scale * rq[r] * e : 0.f;
                            const float l = r > cc ? -dL[j][2 * i + y] * rk[r] * e : 0.f;
                            x[y] = l * be[r];
                            const float zq = z[y] * qk[j][2 * i + y], lk = l * kk[j][2 * i + y];
                            const float nn = r > cc ? fmaf(be[r], lk, zq) : 0.f;
                            rz[i] += zq;
                            rl[i] += lk;
                            rn[i] += nn;
                            col[y] += nn;
                            if (r == cc) {
                                red[R_DZ * C + r] = zq;
                                red[R_DY * C + r] = dL[j][2 * i + y];
                            }
                        }
                        put<2>(sZ, SQ, cm_idx(r, j0, C), z[0], z[1]);
                        put<2>(sX, SQ, cm_idx(r, j0, C), x[0], x[1]);
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) col[y] += __shfl_xor_sync(0xffffffffu, col[y], o);
                        if (g == 0) red[(R_COL + rb) * C + j0 + y] = col[y];
                    }
                }
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&zready);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        rn[i] += __shfl_xor_sync(0xffffffffu, rn[i], o);
                        rz[i] += __shfl_xor_sync(0xffffffffu, rz[i], o);
                        rl[i] += __shfl_xor_sync(0xffffffffu, rl[i], o);
                    }
                    if (t == 0) {
                        red[(R_N + half) * C + r0 + 8 * i] = rn[i];
                        red[(R_ZQ + half) * C + r0 + 8 * i] = rz[i];
                        red[(R_B + half) * C + r0 + 8 * i] = rl[i];
                    }
                }
            }
            // ---- the products with the states: lane d, 32 rows
            float fq[32], fk[32];
            {
                float s[32];
                tmem_row32(tm + T_F + t0, fq);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    fq[j] *= aux[A_OQ * C + t0 + j];
                    s[j] = fq[j] * __bfloat162float(sq[swz_bf16(t0 + j, d)]);
                }
                lanes_total<32>(s, lane);
                dots[rb * C + t0 + lane] = s[0];
                tmem_row32(tm + T_E + t0, fk);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    fk[j] *= aux[A_GK * C + t0 + j];
                    s[j] = fk[j] * __bfloat162float(sk[swz_bf16(t0 + j, d)]);
                    fk[j] *= -be[t0 + j];
                }
                lanes_total<32>(s, lane);
                dots[(4 + rb) * C + t0 + lane] = s[0];
                tmem_row32(tm + T_H + t0, s);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&accfree);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    s[j] *= aux[A_FK * C + t0 + j];
                    fk[j] += s[j];
                    s[j] *= __bfloat162float(sk[swz_bf16(t0 + j, d)]);
                }
                lanes_total<32>(s, lane);
                dots[(8 + rb) * C + t0 + lane] = s[0];
            }
            bar_sync(1, MAIN);
            auto dot = [&](int which, int r) {
                const float* x = dots + which * 4 * C + r;
                return (x[0] + x[C]) + (x[2 * C] + x[3 * C]);
            };
            auto cols = [&](int r) {  // column r of N: the row blocks from its own on
                float s = 0.f;
                for (int i = r >> 4; i < 4; ++i) s += red[(R_COL + i) * C + r];
                return s;
            };
            if (warp < 2) {  // a row shorter than 1e-6 is divided by that, whatever its length
                const int r = tid;
                const float n = red[R_N * C + r] + red[(R_N + 1) * C + r], z = red[R_ZQ * C + r] + red[(R_ZQ + 1) * C + r], dz = red[R_DZ * C + r];
                const bool l2 = p.flags & KDA_FLAG_QK_L2NORM;
                red[R_CQ * C + r] = l2 && rq[r] < 1e6f ? rq[r] * rq[r] * (dot(0, r) + z) : 0.f;
                red[R_CK * C + r] = l2 && rk[r] < 1e6f ? rk[r] * rk[r] * (dot(2, r) - be[r] * dot(1, r) + (n - (z - dz)) + cols(r) + dz) : 0.f;
            } else if (warp == 2) {  // the gate's and beta's gradients, two neighbouring rows per lane
                const float last = aux[A_LAST * C], total = (ss[tb][0] + ss[tb][1]) + (ss[tb][2] + ss[tb][3]);
                double dG[2], hsum = 0.0;
                float db[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = 2 * lane + i;
                    const float n = red[R_N * C + r] + red[(R_N + 1) * C + r], e = dot(1, r), hh = dot(2, r);
                    dG[i] = (double)n - cols(r) + dot(0, r) - (double)be[r] * e - hh;
                    hsum += hh;
                    // Y_i . V'_i / beta_i; where beta_i is 0, or so small that the quotient means nothing, Y_i . v_i less what the chunk
                    // predicts for v_i
                    if (fabsf(be[r]) > 1e-18f) {
                        db[i] = red[R_DY * C + r] / be[r];
                    } else {
                        const float* y = reinterpret_cast<const float*>(sc + lay.Y) + (size_t)u * C * 128;
                        float yv = 0.f;
                        if (r < ci.len)
                            for (int x = 0; x < 128; ++x)
                                yv = fmaf(y[rec_idx(x, r, C)], ldf(static_cast<const bf16*>(p.v) + (((size_t)ci.tok0 + r) * p.HV + h) * 128 + x), yv);
                        db[i] = yv - e + red[R_B * C + r] + red[(R_B + 1) * C + r];
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) hsum += __shfl_xor_sync(0xffffffffu, hsum, o);
                double run = dG[0] + dG[1];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double dn = __shfl_down_sync(0xffffffffu, run, o);
                    if (lane + o < 32) run += dn;
                }
                run += (double)last * total + hsum;
                gate_gradients(p, lay, ci, (size_t)u, h, (float)run, (float)(run - dG[0]), db[0], db[1], be[2 * lane], be[2 * lane + 1], lane);
            }
            bar_sync(1, MAIN);
            // ---- the other products
            ok = mbar_wait(&dqbar, it & 1, p, 1 << 14) && ok;
            tc_fence_after();
            {
                float s[32];
                tmem_row32(tm + T_DQ + t0, s);
#pragma unroll
                for (int j = 0; j < 32; ++j) fq[j] += s[j] - red[R_CQ * C + t0 + j] * __bfloat162float(sq[swz_bf16(t0 + j, d)]);
                tmem_row32(tm + T_DK + t0, s);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&dqfree);
#pragma unroll
                for (int j = 0; j < 32; ++j) fk[j] += s[j] - red[R_CK * C + t0 + j] * __bfloat162float(sk[swz_bf16(t0 + j, d)]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[tb]);
            if (grp > 1) {  // the group's value heads are added up, and the L2 norm follows, in gdr_heads_kernel (R_CQ, R_CK are 0 then)
                float* out = reinterpret_cast<float*>(sc + lay.dqk) + (size_t)u * 2 * C * K + d;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    out[(t0 + j) * K] = fq[j];
                    out[C * K + (t0 + j) * K] = fk[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
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
        const int t = tid - MAIN;
        float x[6][8];  // pieces of eight values: S0 and dS two each, V' and Y
        auto request = [&](int u, int k) {
            const float* a = reinterpret_cast<const float*>(ws + lay.S0) + (size_t)u * K * 128 + k * 16 * K + 8 * t;
            const float* e = reinterpret_cast<const float*>(sc + lay.dS) + (size_t)u * K * 128 + k * 16 * K + 8 * t;
            load8(a, x[0]);
            load8(a + 8 * CONV, x[1]);
            load8(e, x[2]);
            load8(e + 8 * CONV, x[3]);
            load8(reinterpret_cast<const float*>(ws + lay.Vn) + (size_t)u * C * 128 + k * 16 * C + 8 * t, x[4]);
            load8(reinterpret_cast<const float*>(sc + lay.Y) + (size_t)u * C * 128 + k * 16 * C + 8 * t, x[5]);
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
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) s = fmaf(x[j][i], x[2 + j][i], s);
                    leave(b + S0 + 16 * (t + CONV * j), SPART, x[j]);
                    leave(b + DS + 16 * (t + CONV * j), SPART, x[2 + j]);
                }
                leave(b + V + 16 * t, VPART, x[4]);
                leave(b + Y + 16 * t, VPART, x[5]);
                if (k < 7) request(u, k + 1);
                else if (u + stride < units) request(u + stride, 0);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[st]);
            }
            s = warp_sum(s);
            if (lane == 0) {
                ss[it & 1][warp - MAIN / 32] = s;
                mbar_arrive(&accbar);
            }
            __syncwarp();
        }
    } else if (warp == (MAIN + CONV) / 32) {
        constexpr uint32_t idF = make_idesc(128, 64, true, false), idE = make_idesc(128, 64, true, true), idA = make_idesc(64, 64, false, true),
                           idL = make_idesc(64, 64, true, true), idQ = make_idesc(64, 64, false, false);
        auto wait = [&](uint64_t* bar, uint32_t parity, int what) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, p, what));
            tc_fence_after();
            return ok;
        };
        int step = 0;
        const uint32_t z = smem_u32(dyn + Z), x = smem_u32(dyn + X);
        for (int u = blockIdx.x, it = 0; u < units && ok; u += stride, ++it) {
            if (!wait(&tfull[it & 1], (it >> 1) & 1, 1 << 16) || (it > 0 && !wait(&accfree, (it - 1) & 1, 1 << 17))) break;
            const uint32_t tile = smem_u32(dyn + (it & 1) * TILE);
            for (int k = 0; k < 8 && ok; ++k, ++step) {
                const int st = step % RING;
                if (!wait(&full[st], (step / RING) & 1, 1 << 18)) break;
                const uint32_t b = smem_u32(dyn + R0 + st * STAGE);
                if (elect_one()) {
                    const uint64_t dO = desc_rows(tile + DO, k);
                    uint64_t S[3], D[3], W[3], G[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        S[i] = make_desc(b + S0 + i * SPART, 2048, 128);
                        D[i] = make_desc(b + DS + i * SPART, 2048, 128);
                        W[i] = make_desc(b + V + i * VPART, 1024, 128);
                        G[i] = make_desc(b + Y + i * VPART, 1024, 128);
                    }
                    const bool acc = k > 0;
#pragma unroll
                    for (int i = 2; i >= 0; --i) {
                        mma_ss(tmem0 + T_DA, dO, W[i], idA, acc || i < 2);
                        mma_ss(tmem0 + T_F, S[i], dO, idF, acc || i < 2);
                    }
#pragma unroll
                    for (int o = 2; o >= 0; --o)
#pragma unroll
                        for (int i = o; i >= 0; --i) {
                            const bool more = acc || o < 2 || i < o;
                            mma_ss(tmem0 + T_DL, G[i], W[o - i], idL, more);
                            mma_ss(tmem0 + T_E, S[i], G[o - i], idE, more);
                            mma_ss(tmem0 + T_H, D[i], W[o - i], idE, more);
                        }
                    mma_commit(&empty[st]);
                }
                __syncwarp();
            }
            if (!ok || (it > 0 && !wait(&dqfree, (it - 1) & 1, 1 << 19))) break;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    mma_ss(tmem0 + T_DQ, desc_rows(tile + Q, k), desc_rows(tile + KK, k), idQ, k > 0);
                    mma_ss(tmem0 + T_DK, desc_rows(tile + KK, k), desc_rows(tile + KK, k), idQ, k > 0);
                }
                mma_commit(&accbar);
            }
            __syncwarp();
            if (!wait(&zready, it & 1, 1 << 20)) break;
            if (elect_one()) {  // Z and X are lower triangular: K-step s meets rows (or columns) from its own block on (or up to it)
#pragma unroll
                for (int i = 1; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint64_t k_s = make_desc_sw128(tile + KK + s * 2048, 8192, 1024);
                        const uint32_t id = make_idesc(128, 64 - 16 * s, true, false);
                        mma_ss(tmem0 + T_DQ + 16 * s, k_s, make_desc(z + i * MAT + s * 256 + s * 2048, 128, 1024), id, i < 1 || s > 0);
                        mma_ss(tmem0 + T_DK + 16 * s, k_s, make_desc(x + i * MAT + s * 256 + s * 2048, 128, 1024), id, i < 1 || s > 0);
                    }
#pragma unroll
                for (int i = 1; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const uint32_t id = make_idesc(128, 16 * (s + 1), true, true);
                        mma_ss(tmem0 + T_DK, make_desc_sw128(tile + KK + s * 2048, 8192, 1024), make_desc(x + i * MAT + s * 2048, 1024, 128), id, true);
                        mma_ss(tmem0 + T_DK, make_desc_sw128(tile + Q + s * 2048, 8192, 1024), make_desc(z + i * MAT + s * 2048, 1024, 128), id, true);
                    }
                mma_commit(&dqbar);
                mma_commit(&tempty[it & 1]);
            }
            __syncwarp();
        }
    } else {
        const int rt = tid - MAIN - CONV - 32;
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV, kh = h / grp;
            unsigned char* b = dyn + tb * TILE;
            const ChunkInfo ci = chunk_info(p, c);
            if (it > 1) ok = __all_sync(0xffffffffu, mbar_wait(&tempty[tb], ((it >> 1) & 1) ^ 1, p, 1 << 21));
            if (!ok) break;
            if (rt == 0 && u + stride < units) {  // the next unit's records on their way into L2
                const size_t n = (size_t)u + stride;
                l2_prefetch_bulk(ws + lay.S0 + n * K * 512, K * 512);
                l2_prefetch_bulk(sc + lay.dS + n * K * 512, K * 512);
                l2_prefetch_bulk(ws + lay.Vn + n * C * 512, C * 512);
                l2_prefetch_bulk(sc + lay.Y + n * C * 512, C * 512);
            }
            __syncwarp();
            const size_t qrow = ((size_t)ci.tok0 * p.H + kh) * K;
            load_cm<K, ROWS, true>(reinterpret_cast<bf16*>(b + DO), static_cast<const bf16*>(p.grad_o) + ((size_t)ci.tok0 * p.HV + h) * 128, (size_t)p.HV * 128, ci.len, rt);
            load_cm<K, ROWS, true>(reinterpret_cast<bf16*>(b + Q), static_cast<const bf16*>(p.q) + qrow, (size_t)p.H * K, ci.len, rt);
            load_cm<K, ROWS, true>(reinterpret_cast<bf16*>(b + KK), static_cast<const bf16*>(p.k) + qrow, (size_t)p.H * K, ci.len, rt);
            load_words<ROWS>(reinterpret_cast<bf16*>(b + AU), reinterpret_cast<const bf16*>(ws + lay.aux + (size_t)u * AUX * 4), AUX * 4 / 16, rt);
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tfull[tb]);
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
