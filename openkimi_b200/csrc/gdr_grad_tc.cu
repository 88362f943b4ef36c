// Gated delta rule, backward: the gradients of a chunk on tcgen05, from the records that the transposed walks leave (gdr_tc.cu).  The
// formulas stand in gdr_grad.cu; here
//   F = do S0^T   E = Y S0^T   H = V' dS^T  [64 x dk]      dA = do V'^T   dL = Y V'^T  [64 x 64]
// are products over the 128 value columns, M = 64 rows, in K-steps of 16 columns.
//
// One CTA per SM walks the (chunk, value head) units.  What bounds it: 256 KB of records and rows per unit, 5.9 us of an SM's share
// of HBM, so everything runs beside the loads: four warps read the records (FP32, in the order in which a K-step wants them), take
// <S0, dS> and leave three BF16 parts in a ring of two K-steps; a warp issues the products; a warp brings the next unit's rows; eight
// warps do the rest of a unit (pairs, gate, the products with q and k on mma.sync with operands that they have in shared memory)
// while the next unit's accumulators fill.  Records of two BF16 parts take the same bytes and no conversion, but dg is a
// difference of larger sums: 2e-5 off for 15 tokens.
#include "gdr_grad.cuh"

namespace kda {
namespace gdr {

namespace gt {
constexpr int MAIN = 256, CONV = 128, NTHR = MAIN + CONV + 64, RING = 2;  // then a warp each: products, rows
template <int K>
struct Map {
    static constexpr uint32_t LDK = K + 8, ROWS = C * LDK * 2;
    static constexpr uint32_t Q = 0, KK = ROWS, DO = 2 * ROWS, AU = DO + C * 256, YV = AU + 8 * C * 4, TILE = YV + C * 4;
    static constexpr uint32_t SPART = 32 * K, VPART = 2048, S0 = 0, DS = 3 * SPART, V = 6 * SPART, Y = V + 3 * VPART, STAGE = Y + 3 * VPART;  // a K-step: three parts each
    static constexpr uint32_t R0 = 2 * TILE, ZPART = C * gr::LDZ * 2, Z = R0 + RING * STAGE, X = Z + 2 * ZPART, RED = X + 2 * ZPART,
                              TOTAL = RED + gr::RED * C * 4;
    static constexpr uint32_t F = 0, E = K, H = 2 * K, DA = 3 * K, DL = DA + 64;  // tensor memory columns
    static_assert(TOTAL <= 231000 && DL + 64 <= 512, "fits");
};
}  // namespace gt

// 16 lanes x 8 N consecutive columns as fragments: registers 4 i .. 4 i + 3 are (row g, columns 8 i + 2 t, + 1), (row g + 8, the same)
__device__ __forceinline__ void tmem_frag4(uint32_t at, float (*f)[4]) {  // 32 columns
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

template <int K>
__global__ void __launch_bounds__(gt::NTHR, 1) gdr_grad_tc_kernel(const KdaGdrParams p, const Layout lay) {
    using namespace gt;
    using M = Map<K>;
    constexpr int NK = K / 16;
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t full[RING], empty[RING], tfull[2], tempty[2], accbar, accfree;
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
            mbar_init(&tempty[i], 1 + MAIN / 32);
        }
        mbar_init(&accbar, 1 + CONV / 32);
        mbar_init(&accfree, MAIN / 32);
        mbar_fence_init();
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem0 = tmem_s;
    const int units = p.NT * p.HV, stride = gridDim.x, grp = p.HV / p.H;
    const char* ws = static_cast<const char*>(p.workspace);
    const char* sc = static_cast<const char*>(p.bwd_scratch);
    bool ok = true;

    if (warp < MAIN / 32) {
        const int rb = warp & 3, half = warp >> 2;
        const uint32_t tm = tmem0 + ((uint32_t)(rb * 32) << 16);
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV, kh = h / grp;
            unsigned char* b = dyn + tb * M::TILE;
            float* aux = reinterpret_cast<float*>(b + M::AU);
            const GradRows<bf16, K> m = {reinterpret_cast<bf16*>(b + M::Q), reinterpret_cast<bf16*>(b + M::KK), smem_u32(b + M::Q), smem_u32(b + M::KK),
                                         reinterpret_cast<bf16*>(dyn + M::Z), reinterpret_cast<bf16*>(dyn + M::X), smem_u32(dyn + M::Z), smem_u32(dyn + M::X),
                                         aux, aux + C, aux + 2 * C, aux + 3 * C, aux + 4 * C, aux + 5 * C, aux + 6 * C,
                                         reinterpret_cast<float*>(dyn + M::RED), 0.f};
            GradRows<bf16, K> mm = m;
            const ChunkInfo ci = chunk_info(p, c);
            ok = mbar_wait(&tfull[tb], (it >> 1) & 1, p, 1 << 12) && ok;
            ok = bar_and(1, MAIN, ok);  // (also: the unit before is done with Z, X and the sums)
            if (!ok) break;
            mm.last = aux[A_LAST * C];
            if (tid < C) mm.red[gr::R_Y * C + tid] = reinterpret_cast<const float*>(b + M::YV)[tid];
            float F[NK][4], E[NK][4];
            {
                float qk[4][4], kk[4][4], dA[4][4], dL[4][4];
                grad_rows_products(mm, rb, half, lane, qk, kk);
                ok = mbar_wait(&accbar, it & 1, p, 1 << 13) && ok;  // (given up: the unit is finished with what there is, with its barriers)
                tc_fence_after();
                tmem_frag4(tm + M::DA + 32 * half, dA);
                tmem_frag4(tm + M::DL + 32 * half, dL);
                grad_pairs(mm, p.scale, rb, half, lane, dA, dL, qk, kk);
            }
            {
                float H[NK][4];
#pragma unroll
                for (int i = 0; i < NK; i += 4) {
                    tmem_frag4(tm + M::F + half * (K / 2) + 8 * i, F + i);
                    tmem_frag4(tm + M::E + half * (K / 2) + 8 * i, E + i);
                    tmem_frag4(tm + M::H + half * (K / 2) + 8 * i, H + i);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&accfree);
                grad_scale(mm, p.scale, rb, half, lane, F, E, H);
            }
            const float total = (ss[tb][0] + ss[tb][1]) + (ss[tb][2] + ss[tb][3]);
            grad_finish(p, lay, mm, ci, (size_t)u, h, kh, grp, total, F, E, warp, lane, [] { bar_sync(1, MAIN); });
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[tb]);
        }
    } else if (warp < (MAIN + CONV) / 32) {
        const int t = tid - MAIN;
        constexpr int NS = K / 64;  // pieces of eight values of a state that a thread has in a K-step; of Y and V' it is one
        float4 x[2 * (2 * NS + 2)];
        auto request = [&](int u, int k) {
            const float* S0 = reinterpret_cast<const float*>(ws + lay.S0) + (size_t)u * K * 128 + k * 16 * K;
            const float* dS = reinterpret_cast<const float*>(sc + lay.dS) + (size_t)u * K * 128 + k * 16 * K;
            const float* V = reinterpret_cast<const float*>(ws + lay.Vn) + (size_t)u * C * 128 + k * 16 * C;
            const float* Y = reinterpret_cast<const float*>(sc + lay.Y) + (size_t)u * C * 128 + k * 16 * C;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    x[2 * j + i] = __ldcs(reinterpret_cast<const float4*>(S0 + 8 * (t + CONV * j) + 4 * i));
                    x[2 * (NS + j) + i] = __ldcs(reinterpret_cast<const float4*>(dS + 8 * (t + CONV * j) + 4 * i));
                }
                x[4 * NS + i] = __ldcs(reinterpret_cast<const float4*>(V + 8 * t + 4 * i));
                x[4 * NS + 2 + i] = __ldcs(reinterpret_cast<const float4*>(Y + 8 * t + 4 * i));
            }
        };
        auto leave = [&](unsigned char* at, uint32_t part, const float4& a, const float4& c) {
            uint32_t w[4][3];
            split(a.x, a.y, w[0]);
            split(a.z, a.w, w[1]);
            split(c.x, c.y, w[2]);
            split(c.z, c.w, w[3]);
#pragma unroll
            for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(at + i * part) = make_uint4(w[0][i], w[1][i], w[2][i], w[3][i]);
        };
        int step = 0;
        if ((int)blockIdx.x < units) request(blockIdx.x, 0);
        for (int u = blockIdx.x, it = 0; u < units && ok; u += stride, ++it) {
            float s = 0.f;
            for (int k = 0; k < 8; ++k, ++step) {
                const int st = step % RING;
                if (step >= RING) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ((step / RING) & 1) ^ 1, p, 1 << 14));
                if (!ok) break;
                unsigned char* b = dyn + M::R0 + st * M::STAGE;
#pragma unroll
                for (int j = 0; j < NS; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4 &a = x[2 * j + i], &d = x[2 * (NS + j) + i];
                        s = fmaf(a.x, d.x, fmaf(a.y, d.y, fmaf(a.z, d.z, fmaf(a.w, d.w, s))));
                    }
                    leave(b + M::S0 + 16 * (t + CONV * j), M::SPART, x[2 * j], x[2 * j + 1]);
                    leave(b + M::DS + 16 * (t + CONV * j), M::SPART, x[2 * (NS + j)], x[2 * (NS + j) + 1]);
                }
                leave(b + M::V + 16 * t, M::VPART, x[4 * NS], x[4 * NS + 1]);
                leave(b + M::Y + 16 * t, M::VPART, x[4 * NS + 2], x[4 * NS + 3]);
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
        constexpr uint32_t idF = make_idesc(64, K, false, true), idE = make_idesc(64, K, true, true), idA = make_idesc(64, 64, false, true),
                           idL = make_idesc(64, 64, true, true);
        int st = 0, ph = 0;
        for (int u = blockIdx.x, it = 0; u < units && ok; u += stride, ++it) {
            ok = __all_sync(0xffffffffu, mbar_wait(&tfull[it & 1], (it >> 1) & 1, p, 1 << 15));
            if (ok && it > 0) ok = __all_sync(0xffffffffu, mbar_wait(&accfree, (it - 1) & 1, p, 1 << 16));
            const uint32_t od = smem_u32(dyn + (it & 1) * M::TILE + M::DO);
            for (int k = 0; k < 8 && ok; ++k) {
                ok = __all_sync(0xffffffffu, mbar_wait(&full[st], ph, p, 1 << 17));
                if (!ok) break;
                tc_fence_after();
                const uint32_t b = smem_u32(dyn + M::R0 + st * M::STAGE);
                if (elect_one()) {
                    const uint64_t dO = make_desc(od + k * 256, 128, 2048);
                    uint64_t S[3], D[3], V[3], Y[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        S[i] = make_desc(b + M::S0 + i * M::SPART, K * 16, 128);
                        D[i] = make_desc(b + M::DS + i * M::SPART, K * 16, 128);
                        V[i] = make_desc(b + M::V + i * M::VPART, 1024, 128);
                        Y[i] = make_desc(b + M::Y + i * M::VPART, 1024, 128);
                    }
                    const bool acc = k > 0;
#pragma unroll
                    for (int i = 2; i >= 0; --i) {
                        mma_ss(tmem0 + M::DA, dO, V[i], idA, acc || i < 2);
                        mma_ss(tmem0 + M::F, dO, S[i], idF, acc || i < 2);
                    }
#pragma unroll
                    for (int o = 2; o >= 0; --o)
#pragma unroll
                        for (int i = o; i >= 0; --i) {
                            const bool more = acc || o < 2 || i < o;
                            mma_ss(tmem0 + M::DL, Y[i], V[o - i], idL, more);
                            mma_ss(tmem0 + M::E, Y[i], S[o - i], idE, more);
                            mma_ss(tmem0 + M::H, V[i], D[o - i], idE, more);
                        }
                    mma_commit(&empty[st]);
                    if (k == 7) {
                        mma_commit(&accbar);
                        mma_commit(&tempty[it & 1]);
                    }
                }
                __syncwarp();
                if (++st == RING) st = 0, ph ^= 1;
            }
        }
    } else {
        for (int u = blockIdx.x, it = 0; u < units; u += stride, ++it) {
            const int tb = it & 1, c = u / p.HV, h = u - c * p.HV, kh = h / grp;
            unsigned char* b = dyn + tb * M::TILE;
            const ChunkInfo ci = chunk_info(p, c);
            if (it > 1) ok = __all_sync(0xffffffffu, mbar_wait(&tempty[tb], ((it >> 1) & 1) ^ 1, p, 1 << 19));
            if (!ok) break;
            if (lane == 0 && u + stride < units) {  // the next unit's records on their way into L2
                const size_t n = (size_t)u + stride;
                l2_prefetch_bulk(ws + lay.S0 + n * K * 512, K * 512);
                l2_prefetch_bulk(sc + lay.dS + n * K * 512, K * 512);
                l2_prefetch_bulk(ws + lay.Vn + n * C * 512, C * 512);
                l2_prefetch_bulk(sc + lay.Y + n * C * 512, C * 512);
            }
            const size_t qrow = (size_t)ci.tok0 * p.H + kh;
            load_tile<K, K + 8, 32>(reinterpret_cast<bf16*>(b + M::Q), static_cast<const bf16*>(p.q) + qrow * K, (size_t)p.H * K, ci.len, lane);
            load_tile<K, K + 8, 32>(reinterpret_cast<bf16*>(b + M::KK), static_cast<const bf16*>(p.k) + qrow * K, (size_t)p.H * K, ci.len, lane);
            load_cm<128, 32>(reinterpret_cast<bf16*>(b + M::DO), static_cast<const bf16*>(p.grad_o) + ((size_t)ci.tok0 * p.HV + h) * 128,
                             (size_t)p.HV * 128, ci.len, lane);
            load_words<32>(reinterpret_cast<bf16*>(b + M::AU), reinterpret_cast<const bf16*>(ws + lay.aux + (size_t)u * AUX * 4), 8 * C * 4 / 16, lane);
            load_words<32>(reinterpret_cast<bf16*>(b + M::YV), reinterpret_cast<const bf16*>(sc + lay.yv + (size_t)u * C * 4), C * 4 / 16, lane);
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

template <int K>
static cudaError_t launch(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    constexpr int bytes = gt::Map<K>::TOTAL;
    cudaError_t e = allow_smem(gdr_grad_tc_kernel<K>, bytes);
    if (e != cudaSuccess) return e;
    const int units = p.NT * p.HV, sms = sm_count();
    return launch_dependent(gdr_grad_tc_kernel<K>, units < sms ? units : sms, gt::NTHR, bytes, s, p, l);
}

cudaError_t grad_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s) { return p.dk == 64 ? launch<64>(p, l, s) : launch<128>(p, l, s); }

}  // namespace gdr
}  // namespace kda
