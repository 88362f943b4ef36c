// Gated delta rule, the walks along the chunks on tcgen05 (BF16, 128 value columns; gdr_state.cu has the other sizes and FP32).
//
// One CTA per (sequence, value head).  Everything is transposed, value column e = TMEM lane e, so that the 128 lanes are full:
//   P^T = S^T k^T    R^T = -e^G / |k| P^T    V'^T = (v^T + R^T) T'^T    W^T = e^(G_last-G) / |k| V'^T          T' = T diag(beta)
//   S^T <- e^G_last S^T + W^T k              o^T = scale e^G / |q| (S^T q^T) + V'^T A^T
// The state stays in registers in FP32 (256 threads: lane e, half of the key channels).  A computed operand goes to tensor memory in
// three BF16 parts and multiplies q, k, T, A from shared memory, where T and A have three parts too; products of the smallest
// parts are accumulated first, so that the accumulator's truncation falls on small sums.  The update is accumulated from zero and
// added to the decayed state in FP32.
// Bound by the chain of a chunk: split S - S k - R - R T - V' - W k - S.  Everything else is off it: two producer warps bring the next
// chunk's rows (core-matrix order) and records, one warp issues all products, four warps turn finished outputs into rows.  A chunk of
// 64 tokens takes 4.5 us with few CTAs, 5.8 forward and 6.5 backward with 96 that save their records (16 x 2048 tokens of 6 heads: 185
// and 207 us, 3 TB/s of records and rows); on mma.sync, in panels of 32 columns on 384 CTAs, 479 and 494.  At 128 registers a thread the
// forward spills 52 bytes and the backward 212.
#include "gdr.cuh"

namespace kda {
namespace gdr {

namespace ft {
constexpr int MAIN = 256, OUT = 128, PROD = 64, NTHR = MAIN + OUT + PROD + 32, K = 128, DH = K / 2;  // DH: key channels of a main thread
struct Map {
    static constexpr uint32_t ROWS = C * K * 2, MAT = SQ * 2;
    static constexpr uint32_t KK = 0, Q = ROWS, V = 2 * ROWS, TM = V + C * 256, AM = TM + 3 * MAT, AU = AM + 2 * MAT, STAGE = AU + AUX * 4;
    static constexpr uint32_t OT = 2 * STAGE, TOTAL = OT + C * 256;
    // tensor memory columns.  S parts: per half three blocks of DH / 2; over them, once S k and S q are done, the update (DH columns).
    // W and then V' A^T over R, the parts of V' over V' itself, each half of the rows over its own columns.
    static constexpr uint32_t SP = 0, HB = 3 * DH / 2, KS = 2 * HB, QS = KS + 64, VA = QS + 64, R = VA + 64, AV = R, COLS = R + 96;
    static_assert(COLS <= 512 && TOTAL <= 232448, "fits");
};
}  // namespace ft

// 16 consecutive values as P parts: 8 TMEM columns each, `stride` columns apart
template <int P>
__device__ __forceinline__ void st_parts(uint32_t at, uint32_t stride, const float (&x)[16]) {
    uint32_t w[P][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        uint32_t s[P];
        split(x[2 * j], x[2 * j + 1], s);
#pragma unroll
        for (int i = 0; i < P; ++i) w[i][j] = s[i];
    }
#pragma unroll
    for (int i = 0; i < P; ++i) tmem_st8(at + i * stride, w[i]);
}
// N consecutive columns of a record's row (col a multiple of 8)
template <int N>
__device__ __forceinline__ void store_record(float* rec, int e, int col, int cols, const float* x) {
#pragma unroll
    for (int j = 0; j < N; j += 8) store8(rec + rec_idx(e, col + j, cols), x + j);
}
// DH key channels from d0 on of column e: states [dk][dv], or [dv][dk] (rows); src NULL: zero
__device__ __forceinline__ void load_state(const float* src, bool rows, int e, int d0, float (&S)[ft::DH]) {
#pragma unroll
    for (int j = 0; j < ft::DH; j += 4) {
        if (!src) {
            S[j] = S[j + 1] = S[j + 2] = S[j + 3] = 0.f;
        } else if (rows) {
            const float4 x = *reinterpret_cast<const float4*>(src + (size_t)e * ft::K + d0 + j);
            S[j] = x.x; S[j + 1] = x.y; S[j + 2] = x.z; S[j + 3] = x.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) S[j + i] = src[(d0 + j + i) * 128 + e];
        }
    }
}
__device__ __forceinline__ void store_state(float* dst, bool rows, int e, int d0, const float (&S)[ft::DH]) {
#pragma unroll
    for (int j = 0; j < ft::DH; ++j) dst[rows ? e * ft::K + d0 + j : (d0 + j) * 128 + e] = S[j];
}
__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + j);
        x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
    }
}
// this warp has read what the products waiting for `bar` may not hold up: loads from tensor memory wait for the MMAs issued before them,
// so products that are not on the chain are issued behind a load, beside the conversion that follows it
__device__ __forceinline__ void signal(uint64_t* bar, int lane) {
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// last segment that a sequence of nc chunks reaches (however long it is: the count is a hint's)
__device__ __forceinline__ int last_segment(int nc, const Layout& l) { return l.segs == 1 ? 0 : max(0, min(l.segs, (nc + l.seg_len - 1) / l.seg_len) - 1); }

// What a CTA walks: chunks cb..ce of a sequence for one value head.
//   pass 0  whole sequences
//   pass 1  segments of sequences, for the state they end in: blockIdx.y 0, from zero (the first: from the sequence's own start),
//           1: from the identity and without values, what the segment makes of the state that it is entered with; the last
//           segment is walked neither way: nothing follows it, and the backward starts behind it
//   pass 2  segments from the states that gdr_borders_kernel has made of that
// The backward's segments run from their ends to their starts; its pass 1 takes the transitions of the forward.
struct Walk {
    int n, h, kh, c0, cb, ce, seg, last;  // last: the sequence's last segment, of those that it reaches
    long long tok_begin, tok_end;
    // index of the segment: blockIdx.x is (sequence, head, segment) with `count` segments from `first` on
    __device__ __forceinline__ void init(const KdaGdrParams& p, const Layout& l, int first, int count) {
        const int w = blockIdx.x / count;
        seg = first + blockIdx.x % count;
        h = w % p.HV; n = w / p.HV; kh = h / (p.HV / p.H);
        int nc;
        seq_chunks(p, n, c0, nc);
        seq_tokens(p, n, tok_begin, tok_end);
        last = last_segment(nc, l);
        cb = min((long long)seg * l.seg_len, (long long)nc);
        ce = seg == last ? nc : min((long long)(seg + 1) * l.seg_len, (long long)nc);
    }
    // the segment's matrix in a segment buffer
    __device__ __forceinline__ size_t slot(const KdaGdrParams& p, const Layout& l, int s) const { return (((size_t)n * p.HV + h) * l.segs + s) * 16384; }
    __device__ __forceinline__ long long tok(int c) const { return tok_begin + (long long)c * C; }
    __device__ __forceinline__ int rows(int c) const { return (int)min((long long)C, tok_end - tok(c)); }
};

// SAVE: records for the backward; OUT: outputs (pass 1 has none)
template <bool SAVE, bool OUT>
__global__ void __launch_bounds__(ft::NTHR, 1) gdr_fwd_tc_kernel(const KdaGdrParams p, const Layout lay, const int pass) {
    using ft::MAIN;
    using ft::PROD;
    using ft::K;
    using ft::DH;
    using M = ft::Map;
    constexpr int OUTW = ft::OUT;
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t full[2], empty[2], sready, ksbar, rready, vbar, wready, sibar, obar, ofree, ksread, vread, siread;
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    Walk wk;
    wk.init(p, lay, pass == 1 && blockIdx.y, pass == 1 ? lay.segs - 1 : lay.segs);
    const int nc = wk.ce - wk.cb;
    const bool values = pass != 1 || blockIdx.y == 0;
    if (wk.seg > wk.last || (pass == 1 && wk.seg == wk.last)) return;  // (segments that the sequence does not reach)
    wk.c0 += wk.cb;
    wk.tok_begin += (long long)wk.cb * C;
    if (warp == 0) {
        tmem_alloc(&tmem_s, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], 1 + PROD / 32);
            mbar_init(&empty[i], OUT ? OUTW / 32 : MAIN / 32);
        }
        mbar_init(&sready, MAIN / 32);
        mbar_init(&rready, MAIN / 32);
        mbar_init(&wready, MAIN / 32);
        mbar_init(&ksread, MAIN / 32);
        mbar_init(&vread, MAIN / 32);
        mbar_init(&siread, MAIN / 32);
        mbar_init(&ksbar, 1);
        mbar_init(&vbar, 1);
        mbar_init(&sibar, 1);
        mbar_init(&obar, 1);
        mbar_init(&ofree, OUTW / 32);
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem0 = tmem_s;
    const char* ws = static_cast<const char*>(p.workspace);
    bool ok = true;

    if (warp < MAIN / 32) {
        const int e = tid & 127, half = warp >> 2, d0 = half * DH, t0 = half * 32;
        const uint32_t tm = tmem0 + ((uint32_t)((warp & 3) * 32) << 16);
        const size_t sbase = (size_t)(wk.n * (size_t)p.HV + wk.h) * K * 128;
        const bool vf = p.flags & KDA_FLAG_STATE_V_FIRST;
        float* const ends = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.segE);
        float S[DH];
        {   // the state that the walk starts from
            const bool begin = wk.seg == 0, own = begin || pass != 1;
            const float* src = !values || !own ? nullptr : begin ? p.h0 ? p.h0 + sbase : nullptr : ends + wk.slot(p, lay, wk.seg - 1);
            load_state(src, begin && vf, e, d0, S);
            if (!values)
#pragma unroll
                for (int j = 0; j < DH; ++j) S[j] = d0 + j == e ? 1.f : 0.f;
        }
        for (int c = 0; c < nc; ++c) {
            const int stage = c & 1, ph = c & 1;
            const unsigned char* b = dyn + stage * M::STAGE;
            const float* aux = reinterpret_cast<const float*>(b + M::AU);
            const size_t unit = (size_t)(wk.c0 + c) * p.HV + wk.h;
#pragma unroll
            for (int g = 0; g < DH / 16; ++g) {
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = S[16 * g + j];
                st_parts<3>(tm + M::SP + half * M::HB + 8 * g, DH / 2, x);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sready);
            if (SAVE) store_record<DH>(reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.S0) + unit * K * 128, e, d0, K, S);
            // ---- R
            ok = mbar_wait(&full[stage], (c >> 1) & 1, p, 1 << 12) && ok;
            const float last = aux[A_LAST * C];
            ok = mbar_wait(&ksbar, ph, p, 1 << 13) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            uint32_t r[2][16];
            tmem_ld16(tm + M::KS + t0, r[0]);
            tmem_ld16(tm + M::KS + t0 + 16, r[1]);
            tmem_wait_ld();
            signal(&ksread, lane);
            if (OUT && c > 0) ok = mbar_wait(&ofree, ph ^ 1, p, 1 << 11) && ok;  // V' A^T of the chunk before has left R's place
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[16];
                load16(aux + A_GK * C + t0 + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) f[j] *= -__uint_as_float(r[g][j]);
                st_parts<3>(tm + M::R + half * 16 + 8 * g, 32, f);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&rready);
            // ---- V'
            ok = mbar_wait(&vbar, ph, p, 1 << 14) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            tmem_ld16(tm + M::VA + t0, r[0]);
            tmem_ld16(tm + M::VA + t0 + 16, r[1]);
            tmem_wait_ld();
            signal(&vread, lane);
            float x[2][16];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[16];
                load16(aux + A_FK * C + t0 + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    x[g][j] = __uint_as_float(r[g][j]);
                    f[j] *= x[g][j];
                }
                st_parts<3>(tm + M::R + half * 16 + 8 * g, 32, f);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&wready);
            if (OUT) {  // for V' A^T, which waits for siread
#pragma unroll
                for (int g = 0; g < 2; ++g) st_parts<2>(tm + M::VA + half * 32 + 8 * g, 16, x[g]);
                tmem_wait_st();
            }
            if (SAVE) {
                float* V = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.Vn) + unit * C * 128;
#pragma unroll
                for (int g = 0; g < 2; ++g) store_record<16>(V, e, t0 + 16 * g, C, x[g]);
            }
            // ---- the state at the end of the chunk
            ok = mbar_wait(&sibar, ph, p, 1 << 15) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            if (!OUT && lane == 0) mbar_arrive(&empty[stage]);
#pragma unroll
            for (int g = 0; g < DH / 16; g += 2) {
                tmem_ld16(tm + M::SP + half * M::HB + 16 * g, r[0]);
                tmem_ld16(tm + M::SP + half * M::HB + 16 * g + 16, r[1]);
                tmem_wait_ld();
                if (g == DH / 16 - 2) signal(&siread, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[16 * (g + i) + j] = fmaf(last, S[16 * (g + i) + j], __uint_as_float(r[i][j]));
            }
        }
        if (ok) {
            if (pass == 1) store_state((values ? ends : reinterpret_cast<float*>(static_cast<char*>(p.workspace) + lay.segX)) + wk.slot(p, lay, wk.seg), false, e, d0, S);
            else if (p.ht && wk.seg == wk.last) store_state(p.ht + sbase, vf, e, d0, S);
        }
    } else if (warp < (MAIN + OUTW) / 32) {
        const int e = tid & 127;
        const uint32_t tm = tmem0 + ((uint32_t)((warp & 3) * 32) << 16);
        bf16* tile = reinterpret_cast<bf16*>(dyn + M::OT);
        for (int c = 0; c < (OUT ? nc : 0); ++c) {
            const int stage = c & 1;
            const float* oq = reinterpret_cast<const float*>(dyn + stage * M::STAGE + M::AU) + A_OQ * C;
            ok = mbar_wait(&obar, c & 1, p, 1 << 16) && ok;
            ok = bar_and(2, OUTW, ok);  // (also: the tile of the previous chunk has been stored)
            if (!ok) break;
            tc_fence_after();
            uint32_t o[C / 2];
#pragma unroll
            for (int g = 0; g < C / 16; ++g) {
                uint32_t a[16], q[16];
                tmem_ld16(tm + M::QS + 16 * g, q);
                tmem_ld16(tm + M::AV + 16 * g, a);
                tmem_wait_ld();
                float f[16];
                load16(oq + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                    o[8 * g + j / 2] = pack_bf16(fmaf(f[j], __uint_as_float(q[j]), __uint_as_float(a[j])),
                                                 fmaf(f[j + 1], __uint_as_float(q[j + 1]), __uint_as_float(a[j + 1])));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ofree);
                mbar_arrive(&empty[stage]);
            }
#pragma unroll
            for (int j = 0; j < C / 2; ++j) {
                reinterpret_cast<uint16_t*>(tile)[(2 * j) * 128 + e] = (uint16_t)o[j];
                reinterpret_cast<uint16_t*>(tile)[(2 * j + 1) * 128 + e] = (uint16_t)(o[j] >> 16);
            }
            bar_sync(2, OUTW);
            const int rows = wk.rows(c);
            bf16* dst = static_cast<bf16*>(p.o) + ((size_t)wk.tok(c) * p.HV + wk.h) * 128;
#pragma unroll
            for (int i = e; i < C * 16; i += OUTW) {
                const int rr = i >> 4, cc = (i & 15) * 8;
                if (rr < rows) *reinterpret_cast<uint4*>(dst + (size_t)rr * p.HV * 128 + cc) = *reinterpret_cast<const uint4*>(tile + rr * 128 + cc);
            }
        }
    } else if (warp < (MAIN + OUTW + PROD) / 32) {
        const int pt = tid - MAIN - OUTW;
        int c = 0;
        for (; c < nc; ++c) {
            const int stage = c & 1;
            unsigned char* b = dyn + stage * M::STAGE;
            if (c > 1) ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], ((c >> 1) & 1) ^ 1, p, 1 << 17));
            if (!ok) break;
            const size_t unit = (size_t)(wk.c0 + c) * p.HV + wk.h;
            const int rows = wk.rows(c);
            if (pt == 0) {
                mbar_expect_tx(&full[stage], (OUT ? 5 : 3) * M::MAT + AUX * 4);
                tma_load_1d(b + M::TM, ws + lay.T + unit * 3 * M::MAT, 3 * M::MAT, &full[stage]);
                tma_load_1d(b + M::AU, ws + lay.aux + unit * AUX * 4, AUX * 4, &full[stage]);
                if (OUT) tma_load_1d(b + M::AM, ws + lay.A + unit * 3 * M::MAT, 2 * M::MAT, &full[stage]);
            }
            __syncwarp();
            const size_t krow = ((size_t)wk.tok(c) * p.H + wk.kh) * K;
            load_cm<K, PROD>(reinterpret_cast<bf16*>(b + M::KK), static_cast<const bf16*>(p.k) + krow, (size_t)p.H * K, rows, pt);
            if (OUT) load_cm<K, PROD>(reinterpret_cast<bf16*>(b + M::Q), static_cast<const bf16*>(p.q) + krow, (size_t)p.H * K, rows, pt);
            if (values) load_cm<128, PROD>(reinterpret_cast<bf16*>(b + M::V), static_cast<const bf16*>(p.v) + ((size_t)wk.tok(c) * p.HV + wk.h) * 128,
                               (size_t)p.HV * 128, rows, pt);
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
        }
        // given up: the records on their way land before the CTA's memory goes
        for (int i = max(c - 2, 0); !ok && i < c; ++i) mbar_wait(&full[i & 1], (i >> 1) & 1, p, 1 << 17);
    } else {
        constexpr uint32_t id64 = make_idesc(128, 64, false, false), idu = make_idesc(128, DH, false, true);
        for (int c = 0; c < nc && ok; ++c) {
            const int stage = c & 1, ph = c & 1;
            const uint32_t b = smem_u32(dyn + stage * M::STAGE);
            auto wait = [&](uint64_t* bar, uint32_t parity, int what) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, p, what));
                tc_fence_after();
                return ok;
            };
            if (!wait(&full[stage], (c >> 1) & 1, 1 << 18)) break;
            auto with_rows = [&](uint32_t acc, uint32_t rows_at, int parts) {  // S parts times rows, K-major
#pragma unroll
                for (int i = parts - 1; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < K / 16; ++s)
                        mma_ts(tmem0 + acc, tmem0 + M::SP + (s / (DH / 16)) * M::HB + i * (DH / 2) + (s % (DH / 16)) * 8,
                               make_desc(b + rows_at + s * 256, 128, K * 16), id64, i < parts - 1 || s > 0);
            };
            // (+)= x M^T, M lower triangular: K-step s of x's part i is at a(i, s)
            auto with_matrix = [&](uint32_t acc, auto a, uint32_t mat, int parts, bool first) {
#pragma unroll
                for (int o = parts - 1; o >= 0; --o)
#pragma unroll
                    for (int i = o; i >= 0; --i) {
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            mma_ts(tmem0 + acc + 16 * s, tmem0 + a(i, s), make_desc(b + mat + (o - i) * M::MAT + s * 256 + s * 2048, 128, 1024),
                                   make_idesc(128, 64 - 16 * s, false, false), !first || s > 0);
                        first = false;
                    }
            };
            if (!wait(&sready, ph, 1 << 19)) break;
            if (elect_one()) {
                with_rows(M::KS, M::KK, 3);
                mma_commit(&ksbar);
            }
            __syncwarp();
            if (!wait(&ksread, ph, 1 << 20)) break;
            // v^T T'^T (the parts of V' that were here have been used: their products are done)
            if (values && elect_one())
#pragma unroll
                for (int i = 2; i >= 0; --i)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        mma_ss(tmem0 + M::VA + 16 * s, make_desc(b + M::V + s * 4096, 2048, 128), make_desc(b + M::TM + i * M::MAT + s * 256 + s * 2048, 128, 1024),
                               make_idesc(128, 64 - 16 * s, true, false), i < 2 || s > 0);
            __syncwarp();
            if (!wait(&rready, ph, 1 << 21)) break;
            if (elect_one()) {
                with_matrix(M::VA, [](int i, int s) { return M::R + i * 32 + s * 8; }, M::TM, 3, !values);
                mma_commit(&vbar);
            }
            __syncwarp();
            if (OUT) {  // (the accumulator of the chunk before has been read: R could not have been stored)
                if (!wait(&vread, ph, 1 << 10)) break;
                if (elect_one()) with_rows(M::QS, M::Q, 2);
                __syncwarp();
            }
            if (!wait(&wready, ph, 1 << 22)) break;
            if (elect_one()) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 2; i >= 0; --i)
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            mma_ts(tmem0 + M::SP + h * M::HB, tmem0 + M::R + i * 32 + s * 8,
                                   make_desc(b + M::KK + h * (DH / 8) * 128 + s * 2 * (K / 8) * 128, (K / 8) * 128, 128), idu, i < 2 || s > 0);
                mma_commit(&sibar);
            }
            __syncwarp();
            if (OUT) {
                if (!wait(&siread, ph, 1 << 9)) break;
                if (elect_one()) {
                    with_matrix(M::AV, [](int i, int s) { return M::VA + (s >> 1) * 32 + i * 16 + (s & 1) * 8; }, M::AM, 2, true);
                    mma_commit(&obar);
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem0, 512);
}

// ---- backward: dS^T in registers, from the last chunk to the first -------------------------------------------------------
//   dV'^T = e^(G_last-G) / |k| dS^T k^T + do^T A      Y^T = dV'^T T      X^T = -beta e^G / |k| Y^T      dv = beta Y
//   dS^T <- e^G_last dS^T + (scale e^G / |q| do)^T q + X^T k
// The products with do only are issued beside the chain dS - dS k - dV' - dV' T - X - X k - dS.
namespace bt {
using ft::K;
using ft::DH;
struct Map {
    static constexpr uint32_t ROWS = C * K * 2, MAT = SQ * 2;
    static constexpr uint32_t KK = 0, Q = ROWS, DO = 2 * ROWS, TM = DO + C * 256, AM = TM + 3 * MAT, AU = AM + 3 * MAT, STAGE = AU + AUX * 4;
    static constexpr uint32_t OT = 2 * STAGE, TOTAL = OT + C * 256;
    // tensor memory: the parts of dS, over them the update; of the scaled do; of dV', over them X; dS k^T, over it Y; do^T A
    static constexpr uint32_t SP = 0, HB = 3 * DH / 2, DOS = 2 * HB, DV = DOS + 96, KD = DV + 96, AD = KD + 64, COLS = AD + 64;
    static_assert(COLS <= 512 && TOTAL <= 232448 && STAGE % 1024 == 0, "fits");
};
}  // namespace bt

// OUT: dv and the records (pass 1 has none)
template <bool OUT>
__global__ void __launch_bounds__(ft::NTHR, 1) gdr_bwd_tc_kernel(const KdaGdrParams p, const Layout lay, const int pass) {
    using ft::MAIN;
    using ft::PROD;
    using ft::K;
    using ft::DH;
    using M = bt::Map;
    constexpr int OUTW = ft::OUT;
    extern __shared__ __align__(1024) unsigned char dyn[];
    __shared__ uint64_t full[2], empty[2], sready, kdbar, dosready, dvready, ybar, xready, sibar, ofree, kdread, siread;
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    pdl_wait();
    Walk wk;
    wk.init(p, lay, pass == 1, pass == 1 ? lay.segs - 1 : lay.segs);
    const int nc = wk.ce - wk.cb;
    if (wk.seg > wk.last) return;  // (a segment that the sequence does not reach)
    wk.c0 += wk.cb;
    wk.tok_begin += (long long)wk.cb * C;
    if (warp == 0) {
        tmem_alloc(&tmem_s, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], 1 + PROD / 32);
            mbar_init(&empty[i], (MAIN + (OUT ? OUTW : 0)) / 32);
        }
        mbar_init(&sready, MAIN / 32);
        mbar_init(&dosready, MAIN / 32);
        mbar_init(&dvready, MAIN / 32);
        mbar_init(&xready, MAIN / 32);
        mbar_init(&kdread, MAIN / 32);
        mbar_init(&siread, MAIN / 32);
        mbar_init(&kdbar, 1);
        mbar_init(&ybar, 1);
        mbar_init(&sibar, 1);
        mbar_init(&ofree, OUTW / 32);
        mbar_fence_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem0 = tmem_s;
    const char* ws = static_cast<const char*>(p.workspace);
    char* sc = static_cast<char*>(p.bwd_scratch);
    bool ok = true;

    // step i is chunk nc - 1 - i
    if (warp < MAIN / 32) {
        const int e = tid & 127, half = warp >> 2, d0 = half * DH, t0 = half * 32;
        const uint32_t tm = tmem0 + ((uint32_t)((warp & 3) * 32) << 16);
        const size_t sbase = (size_t)(wk.n * (size_t)p.HV + wk.h) * K * 128;
        const bool vf = p.flags & KDA_FLAG_STATE_V_FIRST, end = wk.seg == wk.last;
        float* const starts = reinterpret_cast<float*>(sc + lay.segF);
        float S[DH];
        load_state(end ? p.grad_ht ? p.grad_ht + sbase : nullptr : pass == 1 ? nullptr : starts + wk.slot(p, lay, wk.seg + 1), end && vf, e, d0, S);
        for (int i = 0; i < nc; ++i) {
            const int c = nc - 1 - i, stage = i & 1, ph = i & 1;
            const unsigned char* b = dyn + stage * M::STAGE;
            const float* aux = reinterpret_cast<const float*>(b + M::AU);
            const size_t unit = (size_t)(wk.c0 + c) * p.HV + wk.h;
#pragma unroll
            for (int g = 0; g < DH / 16; ++g) {
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = S[16 * g + j];
                st_parts<3>(tm + M::SP + half * M::HB + 8 * g, DH / 2, x);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sready);
            // ---- scaled rows of do
            ok = mbar_wait(&full[stage], (i >> 1) & 1, p, 1 << 12) && ok;
            const float last = aux[A_LAST * C];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[16];
                load16(aux + A_OQ * C + t0 + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) f[j] *= __bfloat162float(reinterpret_cast<const bf16*>(b + M::DO)[swz_bf16(t0 + 16 * g + j, e)]);
                st_parts<3>(tm + M::DOS + half * 16 + 8 * g, 32, f);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&dosready);
            if (OUT) store_record<DH>(reinterpret_cast<float*>(sc + lay.dS) + unit * K * 128, e, d0, K, S);
            // ---- dV'
            ok = mbar_wait(&kdbar, ph, p, 1 << 13) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            uint32_t r[2][16], ad[2][16];
            tmem_ld16(tm + M::KD + t0, r[0]);
            tmem_ld16(tm + M::KD + t0 + 16, r[1]);
            tmem_ld16(tm + M::AD + t0, ad[0]);
            tmem_ld16(tm + M::AD + t0 + 16, ad[1]);
            tmem_wait_ld();
            signal(&kdread, lane);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[16];
                load16(aux + A_FK * C + t0 + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) f[j] = fmaf(f[j], __uint_as_float(r[g][j]), __uint_as_float(ad[g][j]));
                st_parts<3>(tm + M::DV + half * 16 + 8 * g, 32, f);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&dvready);
            // ---- X
            ok = mbar_wait(&ybar, ph, p, 1 << 14) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            tmem_ld16(tm + M::KD + t0, r[0]);
            tmem_ld16(tm + M::KD + t0 + 16, r[1]);
            tmem_wait_ld();
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                float f[16];
                load16(aux + A_BGK * C + t0 + 16 * g, f);
#pragma unroll
                for (int j = 0; j < 16; ++j) f[j] *= -__uint_as_float(r[g][j]);
                st_parts<3>(tm + M::DV + half * 16 + 8 * g, 32, f);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&xready);
            // ---- dS at the start of the chunk
            ok = mbar_wait(&sibar, ph, p, 1 << 15) && ok;
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            if (lane == 0) mbar_arrive(&empty[stage]);
#pragma unroll
            for (int g = 0; g < DH / 16; g += 2) {
                tmem_ld16(tm + M::SP + half * M::HB + 16 * g, r[0]);
                tmem_ld16(tm + M::SP + half * M::HB + 16 * g + 16, r[1]);
                tmem_wait_ld();
                if (g == DH / 16 - 2) signal(&siread, lane);
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[16 * (g + x) + j] = fmaf(last, S[16 * (g + x) + j], __uint_as_float(r[x][j]));
            }
        }
        if (ok) {
            if (pass == 1) store_state(starts + wk.slot(p, lay, wk.seg), false, e, d0, S);
            else if (p.grad_h0 && wk.seg == 0) store_state(p.grad_h0 + sbase, vf, e, d0, S);
        }
    } else if (warp < (MAIN + OUTW) / 32) {
        const int e = tid & 127;
        const uint32_t tm = tmem0 + ((uint32_t)((warp & 3) * 32) << 16);
        bf16* tile = reinterpret_cast<bf16*>(dyn + M::OT);
        for (int i = 0; i < (OUT ? nc : 0); ++i) {
            const int c = nc - 1 - i, stage = i & 1;
            const float* be = reinterpret_cast<const float*>(dyn + stage * M::STAGE + M::AU) + A_BETA * C;
            const size_t unit = (size_t)(wk.c0 + c) * p.HV + wk.h;
            ok = mbar_wait(&ybar, i & 1, p, 1 << 16) && ok;
            ok = bar_and(2, OUTW, ok);
            if (!ok) break;
            tc_fence_after();
            uint32_t y[C / 16][16];
#pragma unroll
            for (int g = 0; g < C / 16; ++g) tmem_ld16(tm + M::KD + 16 * g, y[g]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ofree);
            float* Y = reinterpret_cast<float*>(sc + lay.Y) + unit * C * 128 + e;  // [64][128]
#pragma unroll
            for (int g = 0; g < C / 16; ++g) {
                float f[16];
                load16(be + 16 * g, f);
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    x[j] = __uint_as_float(y[g][j]);
                    tile[(16 * g + j) * 128 + e] = __float2bfloat16_rn(f[j] * x[j]);
                    Y[(16 * g + j) * 128] = x[j];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
            bar_sync(2, OUTW);
            const int rows = wk.rows(c);
            bf16* dst = static_cast<bf16*>(p.grad_v) + ((size_t)wk.tok(c) * p.HV + wk.h) * 128;
#pragma unroll
            for (int x = e; x < C * 16; x += OUTW) {
                const int rr = x >> 4, cc = (x & 15) * 8;
                if (rr < rows) *reinterpret_cast<uint4*>(dst + (size_t)rr * p.HV * 128 + cc) = *reinterpret_cast<const uint4*>(tile + rr * 128 + cc);
            }
        }
    } else if (warp < (MAIN + OUTW + PROD) / 32) {
        const int pt = tid - MAIN - OUTW;
        int i = 0;
        for (; i < nc; ++i) {
            const int c = nc - 1 - i, stage = i & 1;
            unsigned char* b = dyn + stage * M::STAGE;
            if (i > 1) ok = __all_sync(0xffffffffu, mbar_wait(&empty[stage], ((i >> 1) & 1) ^ 1, p, 1 << 17));
            if (!ok) break;
            const size_t unit = (size_t)(wk.c0 + c) * p.HV + wk.h;
            const int rows = wk.rows(c);
            if (pt == 0) {
                mbar_expect_tx(&full[stage], 6 * M::MAT + AUX * 4);
                tma_load_1d(b + M::AM, ws + lay.A + unit * 3 * M::MAT, 3 * M::MAT, &full[stage]);
                tma_load_1d(b + M::AU, ws + lay.aux + unit * AUX * 4, AUX * 4, &full[stage]);
                tma_load_1d(b + M::TM, ws + lay.Tb + unit * 3 * M::MAT, 3 * M::MAT, &full[stage]);
            }
            __syncwarp();
            const size_t krow = ((size_t)wk.tok(c) * p.H + wk.kh) * K;
            load_cm<K, PROD>(reinterpret_cast<bf16*>(b + M::KK), static_cast<const bf16*>(p.k) + krow, (size_t)p.H * K, rows, pt);
            load_cm<128, PROD, true>(reinterpret_cast<bf16*>(b + M::DO), static_cast<const bf16*>(p.grad_o) + ((size_t)wk.tok(c) * p.HV + wk.h) * 128,
                           (size_t)p.HV * 128, rows, pt);
            load_cm<K, PROD>(reinterpret_cast<bf16*>(b + M::Q), static_cast<const bf16*>(p.q) + krow, (size_t)p.H * K, rows, pt);
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
        }
        for (int x = max(i - 2, 0); !ok && x < i; ++x) mbar_wait(&full[x & 1], (x >> 1) & 1, p, 1 << 17);
    } else {
        constexpr uint32_t id64 = make_idesc(128, 64, false, false), idu = make_idesc(128, DH, false, true);
        for (int i = 0; i < nc && ok; ++i) {
            const int stage = i & 1, ph = i & 1;
            const uint32_t b = smem_u32(dyn + stage * M::STAGE);
            auto wait = [&](uint64_t* bar, uint32_t parity, int what) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, p, what));
                tc_fence_after();
                return ok;
            };
            // columns j of x M for lower triangular M: block s of the inner index reaches columns up to 16 (s + 1)
            auto update = [&](uint32_t parts_at, uint32_t rows_at, bool first) {  // update (+)= parts times rows
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 2; x >= 0; --x)
#pragma unroll
                        for (int s = 0; s < 4; ++s)
                            mma_ts(tmem0 + M::SP + h * M::HB, tmem0 + parts_at + x * 32 + s * 8,
                                   make_desc(b + rows_at + h * (DH / 8) * 128 + s * 2 * (K / 8) * 128, (K / 8) * 128, 128), idu,
                                   !first || x < 2 || s > 0);
            };
            if (!wait(&full[stage], (i >> 1) & 1, 1 << 18) || (i > 0 && !wait(&siread, ph ^ 1, 1 << 9))) break;
            if (elect_one()) {
#pragma unroll
                for (int x = 2; x >= 0; --x)
#pragma unroll
                    for (int s = 3; s >= 0; --s)
                        mma_ss(tmem0 + M::AD, make_desc_sw128(b + M::DO + s * 2048, 8192, 1024),
                               make_desc(b + M::AM + x * M::MAT + s * 2048, 1024, 128), make_idesc(128, 16 * (s + 1), true, true), x < 2 || s < 3);
            }
            __syncwarp();
            if (!wait(&sready, ph, 1 << 19) || (OUT && i > 0 && !wait(&ofree, ph ^ 1, 1 << 20))) break;
            if (elect_one()) {
#pragma unroll
                for (int x = 2; x >= 0; --x)
#pragma unroll
                    for (int s = 0; s < K / 16; ++s)
                        mma_ts(tmem0 + M::KD, tmem0 + M::SP + (s / (DH / 16)) * M::HB + x * (DH / 2) + (s % (DH / 16)) * 8,
                               make_desc(b + M::KK + s * 256, 128, K * 16), id64, x < 2 || s > 0);
                mma_commit(&kdbar);
            }
            __syncwarp();
            if (!wait(&dosready, ph, 1 << 21) || !wait(&kdread, ph, 1 << 22)) break;  // (the parts of dS have been used)
            if (elect_one()) update(M::DOS, M::Q, true);
            __syncwarp();
            if (!wait(&dvready, ph, 1 << 23)) break;
            if (elect_one()) {
                bool first = true;
#pragma unroll
                for (int o = 2; o >= 0; --o)
#pragma unroll
                    for (int x = o; x >= 0; --x) {
#pragma unroll
                        for (int s = 3; s >= 0; --s)
                            mma_ts(tmem0 + M::KD, tmem0 + M::DV + x * 32 + s * 8, make_desc(b + M::TM + (o - x) * M::MAT + s * 2048, 1024, 128),
                                   make_idesc(128, 16 * (s + 1), false, true), !first || s < 3);
                        first = false;
                    }
                mma_commit(&ybar);
            }
            __syncwarp();
            if (!wait(&xready, ph, 1 << 24)) break;
            if (elect_one()) {
                update(M::DV, M::KK, false);
                mma_commit(&sibar);
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem0, 512);
}

// States at the segments' borders, 8 columns of one (sequence, head) per CTA: forward, E_j <- X_j E_{j-1} + E_j for j = 1, 2, ..; backward
// (TR), F_j <- X_j^T F_{j+1} + F_j for j = segs - 2 downwards.  FP32 multiply-adds; the X of the next two segments arrive meanwhile.
// 2.6 us a border (8 heads); with 512 threads, two to a sum, 3.5.
constexpr int LDX = 132, XBUF = 3;  // floats per row of X, its copies
template <bool TR>
__global__ void __launch_bounds__(256) gdr_borders_kernel(const KdaGdrParams p, const Layout lay, float* M, const float* X) {
    extern __shared__ __align__(16) float sm[];  // X three times, then the columns [128][8]
    float* cols = sm + XBUF * 128 * LDX;
    const int tid = threadIdx.x, d = tid >> 1, c4 = (tid & 1) * 4, c0 = (blockIdx.x & 15) * 8;
    const size_t base = (size_t)(blockIdx.x >> 4) * lay.segs * 16384;
    pdl_wait();
    int first_chunk, nc;
    seq_chunks(p, (blockIdx.x >> 4) / p.HV, first_chunk, nc);
    const int last = last_segment(nc, lay), steps = last - 1;  // (segment 0 of the forward, the last of the backward are done)
    if (steps < 1) return;
    auto seg = [&](int i) { return TR ? last - 1 - i : 1 + i; };
    auto request = [&](int i) {
        const float* x = X + base + (size_t)seg(i) * 16384;
        if (i < steps)
            for (int q = tid; q < 4096; q += 256) cp_async16_z(sm + i % XBUF * 128 * LDX + (q >> 5) * LDX + (q & 31) * 4, x + 4 * q, true);
        cp_async_commit();
    };
    auto at = [&](int s) { return reinterpret_cast<float4*>(M + base + (size_t)s * 16384 + d * 128 + c0 + c4); };
    for (int i = 0; i < XBUF - 1; ++i) request(i);
    float4 next = *at(seg(0));
    *reinterpret_cast<float4*>(cols + d * 8 + c4) = *at(TR ? last : 0);
    for (int i = 0; i < steps; ++i) {
        float4 acc = next;
        cp_async_wait<XBUF - 2>();
        __syncthreads();
        request(i + XBUF - 1);  // (into what the step before read)
        if (i + 1 < steps) next = *at(seg(i + 1));
        const float* x = sm + i % XBUF * 128 * LDX;
#pragma unroll 8
        for (int k = 0; k < 128; k += 4) {
            float w[4];
            if (TR) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = x[(k + j) * LDX + d];
            } else {
                const float4 v = *reinterpret_cast<const float4*>(x + d * LDX + k);
                w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 s = *reinterpret_cast<const float4*>(cols + (k + j) * 8 + c4);
                acc.x = fmaf(w[j], s.x, acc.x); acc.y = fmaf(w[j], s.y, acc.y); acc.z = fmaf(w[j], s.z, acc.z); acc.w = fmaf(w[j], s.w, acc.w);
            }
        }
        __syncthreads();
        *reinterpret_cast<float4*>(cols + d * 8 + c4) = acc;
        *at(seg(i)) = acc;
    }
}

template <class Kernel>
static cudaError_t walk(Kernel* k, dim3 grid, int bytes, const KdaGdrParams& p, const Layout& l, int pass, cudaStream_t s) {
    const cudaError_t e = allow_smem(k, bytes);
    return e == cudaSuccess ? launch_dependent(k, grid, ft::NTHR, bytes, s, p, l, pass) : e;
}
template <bool TR>
static cudaError_t borders(const KdaGdrParams& p, const Layout& l, float* m, cudaStream_t s) {
    constexpr int bytes = (XBUF * 128 * LDX + 128 * 8) * 4;
    if (l.segs < 3) return cudaSuccess;
    const cudaError_t e = allow_smem(gdr_borders_kernel<TR>, bytes);
    const float* x = reinterpret_cast<const float*>(static_cast<const char*>(p.workspace) + l.segX);
    return e == cudaSuccess ? launch_dependent(gdr_borders_kernel<TR>, p.N * p.HV * 16, 256, bytes, s, p, l, m, x) : e;
}

cudaError_t fwd_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    const unsigned walks = (unsigned)(p.N * p.HV);
    const bool save = !(p.flags & KDA_FLAG_NO_SAVE);
    cudaError_t e = cudaSuccess;
    if (l.segs > 1) {
        // (two segments need no transition: the first starts from the sequence's own state, the last's nobody needs)
        e = walk(gdr_fwd_tc_kernel<false, false>, dim3(walks * (l.segs - 1), l.segs > 2 ? 2 : 1), ft::Map::TOTAL, p, l, 1, s);
        if (e == cudaSuccess) e = borders<false>(p, l, reinterpret_cast<float*>(static_cast<char*>(p.workspace) + l.segE), s);
    }
    if (e != cudaSuccess) return e;
    const dim3 grid(walks * l.segs);
    const int pass = l.segs > 1 ? 2 : 0;
    return save ? walk(gdr_fwd_tc_kernel<true, true>, grid, ft::Map::TOTAL, p, l, pass, s) : walk(gdr_fwd_tc_kernel<false, true>, grid, ft::Map::TOTAL, p, l, pass, s);
}

cudaError_t bwd_tc(const KdaGdrParams& p, const Layout& l, cudaStream_t s) {
    const unsigned walks = (unsigned)(p.N * p.HV);
    cudaError_t e = cudaSuccess;
    if (l.segs > 1) {
        e = walk(gdr_bwd_tc_kernel<false>, dim3(walks * (l.segs - 1)), bt::Map::TOTAL, p, l, 1, s);
        if (e == cudaSuccess) e = borders<true>(p, l, reinterpret_cast<float*>(static_cast<char*>(p.bwd_scratch) + l.segF), s);
    }
    if (e != cudaSuccess) return e;
    return walk(gdr_bwd_tc_kernel<true>, dim3(walks * l.segs), bt::Map::TOTAL, p, l, l.segs > 1 ? 2 : 0, s);
}

}  // namespace gdr
}  // namespace kda
