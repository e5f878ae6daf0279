// Softmax cross entropy of a linear layer over a large vocabulary, with its gradients, without the logits in memory.
//
//   z = x W^T + b      lse_i = log sum_j exp z_ij      loss_i = lse_i - (1 - e) z_i,t(i) - e/V sum_j z_ij
//   dz_ij = p_ij - (1 - e) [j = t(i)] - e/V            dx = g dz W      dW = g dz^T x      db = g sum_i dz_i
//
// x bf16 [T, D], W bf16 [V, D].  The rows are worked through in blocks whose size the workspace bounds; per block
//   1. x W^T tile by tile (lx_gemm_kernel, NT).  The epilogue takes a tile's logits in fp32 from the accumulators: per row and 64
//      columns their maximum m and s = sum exp(z - m) go to a small table; exp(z - m) itself, in [0, 1], goes to the block's
//      matrix P in fp16 (11 bits; bf16 would round it 8 times as far; what falls below fp16's 6e-8 of its maximum is below what the
//      later bf16 rounding of its larger neighbours leaves).  Loss alone: only the table is written.
//   2. one workgroup per row (lx_row_kernel): lse from the table, the target's logit as a dot product of its own, the row's loss, and
//      P -> dz in place, now bf16: the one rounding of the gradient's factor.  g is not in it: a constant such as 1 / count would be
//      rounded 1 part in 256 in the same direction everywhere; it multiplies the fp32 sums of the next step.
//   3. dx = dz W (NN) and dW = dz^T x (TN) with the same kernel, and the column sums for db.
// 6 T V D floating-point operations: nothing is computed twice.  Keeping one 16-bit factor per logit of a block costs 4 bytes of
// traffic per logit for step 2, where computing the logits again for the gradients would cost 2 D operations.
#include "common.h"
#include "gemm_nt.h"

#define LX_BK 64
#define LX_TILE 256
#define LX_ELEMS (LX_TILE * LX_BK)                            // elements per operand tile
#define LX_LDS (4 * LX_ELEMS * 2 + 8 * 16 * 64 * 4)           // two buffers of both tiles, 4 KB of epilogue staging per wave
#define LX_STAT 64                                            // columns per entry of the statistics table

enum { LX_NT = 0, LX_NN = 1, LX_TN = 2 };
enum { LX_OUT = 0, LX_XENT = 1 };

// 512 bytes of zeros (never written): what rows and columns behind the contraction's end are read from
__device__ __attribute__((aligned(512))) unsigned lx_zero_row[128];

struct LxGemmParams {
    const bf16_t* A; const bf16_t* B;       // NT: A [M][KA], B [N][KB];  NN: B [KB][N];  TN: A [KA][M], B [KB][N]
    long long lda, ldb;
    int M, N;
    int KA, KB;             // valid extent of the contraction in each operand; behind it zeros are read
    int steps;              // 64-deep steps over the whole contraction
    int tiles_m, tiles_n, band, splits;
    // LX_OUT: out[m][n] = scale[0] * acc (+ add[m][n]), bf16 or fp32; or slab[split][m][n] = acc
    const float* scale;
    const float* add;
    void* out; long long ldo; int out_f32;
    float* slab;
    // LX_XENT
    const void* bias; int bias_type;        // 0 fp32, 1 bf16, null: none
    float2* stats; int stat_cols;           // [M][stat_cols]: (m, s) of 64 columns
    float* zsum;                            // [M][stat_cols] sums of the logits, null: not wanted (no smoothing)
    _Float16* P; long long ldp;             // null: loss alone
};

static __device__ __forceinline__ int lx_swz(int m) { return (((m >> 3) & 1) << 3) | ((m & 3) << 1); }
static __device__ __forceinline__ bf16x8 lx_tr(const bf16_t* lo, const bf16_t* hi) {
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)lo);
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)hi);
    return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
static __device__ __forceinline__ unsigned lx_pack_h(float a, float b) {
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
}

// One 512-thread workgroup per compute unit works through 256 x 256 tiles of the output, 8 waves (2 x 4) of 128 x 64 = 128 accumulator
// registers each, 64-deep steps.  Operands go from memory to LDS by DMA, two steps ahead across tile borders, into a double buffer;
// fragments are read one phase of 16 matrix instructions before their use.  An operand whose rows run along the contraction sits in LDS as
// [256][64] (16-byte chunks XOR-swizzled by the row) and is read with ds_read_b128; one whose rows run along the output as [64][256]
// and is read with the transposing ds_read_b64_tr_b16: no transposed copy of W or dz is made.  The matrix instruction's operands are
// swapped, so a lane holds four consecutive columns of one output row.  Tiles are dealt by number (no counters: a captured graph may be
// replayed on any stream); a tile order in bands of 8 column tiles keeps what the 32 workgroups of an XCD read at a time to 4 row panels
// and 8 column panels.
template <int LAY, int EPI>
__global__ __launch_bounds__(512) void lx_gemm_kernel(const LxGemmParams p) {
    constexpr bool AT = LAY == LX_TN, BT = LAY != LX_NT;        // operand stored with the contraction as its slow dimension
    extern __shared__ __attribute__((aligned(16))) bf16_t lsm[];   // [2 buffers][A tile | B tile], [8 waves][16][64] fp32

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int lr = lane & 15, lg = lane >> 4;
    const int lq = lr >> 2, lp = lr & 3;
    const unsigned lds_base = __builtin_amdgcn_readfirstlane(lds_addr(lsm));
    const unsigned lds_stage = (unsigned)(wave * 4 * 1024);

    const int tiles = p.tiles_m * p.tiles_n, items = tiles * p.splits, G = gridDim.x;

    // ---- staging: where the next step's operands come from
    // [256][64] image: wave w, piece j: rows (4 w + j) * 8 + lane / 8; LDS position lane % 8 receives chunk (lane % 8) ^ (row & 7)
    // [64][256] image: wave w, piece j: rows (4 w + j) * 2 + lane / 32; LDS position lane % 32 receives chunk (lane % 32) ^ lx_swz(row)
    const int srow = lane >> 3, sch = (lane & 7) ^ srow;
    const int shalf = lane >> 5, spos = lane & 31;
    int sv = blockIdx.x, sk = 0, sk_end = 0;
    const bf16_t* sA = p.A;
    const bf16_t* sB = p.B;
    unsigned voA[4], voB[4];
    auto locate = [&](int v, int& split, int& m0, int& n0) {
        const int id = xcd_remap(v, items);
        split = id / tiles;
        const int tile = id - split * tiles;
        const int full = p.tiles_m * p.band;
        const int blk = tile / full;
        const int rem = tile - blk * full;
        const int c0 = blk * p.band;
        const int width = p.tiles_n - c0 < p.band ? p.tiles_n - c0 : p.band;
        const int tm = rem / width;
        // the divisions run on the vector unit: say that their results are the same in every lane
        split = __builtin_amdgcn_readfirstlane(split);
        m0 = __builtin_amdgcn_readfirstlane(tm * LX_TILE);
        n0 = __builtin_amdgcn_readfirstlane((c0 + rem - tm * width) * LX_TILE);
    };
    // split s of S takes steps [s * steps / S, (s + 1) * steps / S): q = steps / S each, the first steps % S one more
    const int sq = __builtin_amdgcn_readfirstlane(p.steps / p.splits), sr = p.steps - sq * p.splits;
    auto first_step = [&](int split) { return split * sq + (split < sr ? split : sr); };
    auto aim = [&](int v) {
        int split, m0, n0;
        locate(v, split, m0, n0);
        sk = first_step(split);
        sk_end = first_step(split + 1);
        sA = p.A + (AT ? (size_t)m0 : (size_t)m0 * p.lda);
        sB = p.B + (BT ? (size_t)n0 : (size_t)n0 * p.ldb);
        // rows and columns behind the edge of the output read the last valid ones: their results are not stored
        const int ma = p.M - 1 - m0, mb = p.N - 1 - n0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (AT) {
                const int r = (wave * 4 + j) * 2 + shalf;
                voA[j] = (unsigned)((r * p.lda + (spos ^ lx_swz(r)) * 8) * 2);      // A's rows are padded to a multiple of 256
            } else {
                const int r = (wave * 4 + j) * 8 + srow;
                voA[j] = (unsigned)(((r < ma ? r : ma) * p.lda + sch * 8) * 2);
            }
            if (BT) {
                const int r = (wave * 4 + j) * 2 + shalf;
                const int c = (spos ^ lx_swz(r)) * 8;
                voB[j] = (unsigned)((r * p.ldb + (n0 + c < p.N ? c : p.N - 8 - n0)) * 2);
            } else {
                const int r = (wave * 4 + j) * 8 + srow;
                voB[j] = (unsigned)(((r < mb ? r : mb) * p.ldb + sch * 8) * 2);
            }
        }
    };
    // one operand's 64-deep step kstep -> LDS; what lies behind the contraction's end K comes from the zero row
    auto stage = [&](const bf16_t* base, const unsigned (&vo)[4], bool slow, long long ld, int K, int kstep, unsigned dst) {
        const bf16_t* src = base + (slow ? (size_t)kstep * LX_BK * ld : (size_t)kstep * LX_BK);
        if ((kstep + 1) * LX_BK <= K) {
#pragma unroll
            for (int j = 0; j < 4; ++j) glds16(src, vo[j], dst + j * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = kstep * LX_BK + (slow ? (wave * 4 + j) * 2 + shalf : sch * 8);
                const void* z = (const char*)lx_zero_row + (lane & 31) * 16;
                glds16_v(k < K ? (const void*)((const char*)src + vo[j]) : z, dst + j * 1024);
            }
        }
    };
    auto stageA = [&](int par) { stage(sA, voA, AT, p.lda, p.KA, sk, lds_base + (unsigned)(par * 2 * LX_ELEMS * 2) + lds_stage); };
    auto stageB = [&](int par) { stage(sB, voB, BT, p.ldb, p.KB, sk, lds_base + (unsigned)((par * 2 + 1) * LX_ELEMS * 2) + lds_stage); };
    auto advance = [&]() {
        if (++sk == sk_end) {
            sv += G;
            if (sv < items) aim(sv);
        }
    };

    // ---- fragments
    int offA[2], offB[2];
    int preA = 0, preB = 0, rbase = 0;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int x = ((ks * 4 + lg) ^ (lr & 7)) << 3;
        offA[ks] = (wm * 128 + lr) * LX_BK + x;
        offB[ks] = (wn * 64 + lr) * LX_BK + x;
    }
    if (AT || BT) {
        const int sw = lx_swz(8 * lg + lq);
        preA = ((wm * 16) | (lp >> 1)) ^ sw;
        preB = ((wn * 8) | (lp >> 1)) ^ sw;
        rbase = (8 * lg + lq) * 256 + (lp & 1) * 4;
    }
    f32x4 acc[8][4];
    bf16x8 faE[4], faO[4], fbE[4], fbO[4];
    auto ldA = [&](bf16x8 (&f)[4], const bf16_t* cA, int ks, int h) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (AT) {
                const bf16_t* q = cA + ks * 32 * 256 + rbase + ((preA ^ (2 * (4 * h + t))) << 3);
                f[t] = lx_tr(q, q + 4 * 256);
            } else {
                f[t] = *reinterpret_cast<const bf16x8*>(cA + offA[ks] + (4 * h + t) * 16 * LX_BK);
            }
        }
    };
    auto ldB = [&](bf16x8 (&f)[4], const bf16_t* cB, int ks) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (BT) {
                const bf16_t* q = cB + ks * 32 * 256 + rbase + ((preB ^ (2 * t)) << 3);
                f[t] = lx_tr(q, q + 4 * 256);
            } else {
                f[t] = *reinterpret_cast<const bf16x8*>(cB + offB[ks] + t * 16 * LX_BK);
            }
        }
    };
    auto mma = [&](const bf16x8 (&fa)[4], const bf16x8 (&fb)[4], int h) {
#pragma unroll
        for (int tm = 0; tm < 4; ++tm)
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
                acc[4 * h + tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[tn], fa[tm], acc[4 * h + tm][tn], 0, 0, 0);
    };
    // interleave a phase's 16 matrix instructions with its LDS reads
    constexpr int RA = AT ? 8 : 4, RAB = (AT ? 8 : 4) + (BT ? 8 : 4);
#define LX_MIX(reads)                                                                 \
    _Pragma("unroll") for (int i = 0; i < (reads); ++i) {                             \
        __builtin_amdgcn_sched_group_barrier(0x008, 16 / (reads), 0);                 \
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                            \
    }                                                                                 \
    __builtin_amdgcn_sched_barrier(0)

    if (sv >= items) return;
    int v = sv;
    aim(sv);
    stageA(0);
    stageB(0);
    advance();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (sv < items) { stageA(1); stageB(1); advance(); }
    ldB(fbE, lsm + LX_ELEMS, 0);
    ldA(faE, lsm, 0, 0);
    int par = 0;
    bool pend = false;          // the A half of a step is on its way into buffer par ^ 1, the B half is not yet requested

    for (; v < items; v += G) {
        int split, m0, n0;
        locate(v, split, m0, n0);
        const int nk = first_step(split + 1) - first_step(split);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int kt = 0; kt < nk; ++kt) {
            const bf16_t* cA = lsm + par * 2 * LX_ELEMS;
            const bf16_t* cB = cA + LX_ELEMS;
            const bf16_t* nA = lsm + (par ^ 1) * 2 * LX_ELEMS;
            const bf16_t* nB = nA + LX_ELEMS;
            if (pend) { stageB(par ^ 1); advance(); pend = false; }
            mma(faE, fbE, 0);
            ldA(faO, cA, 0, 1);
            LX_MIX(RA);
            mma(faO, fbE, 1);
            ldB(fbO, cB, 1);
            ldA(faE, cA, 1, 0);
            LX_MIX(RAB);
            mma(faE, fbO, 0);
            ldA(faO, cA, 1, 1);
            LX_MIX(RA);
            // every wave has read the current buffer; the next step has landed: publish it, refill the current buffer
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (sv < items) { stageA(par); pend = true; }
            mma(faO, fbO, 1);
            ldB(fbE, nB, 0);
            ldA(faE, nA, 0, 0);
            LX_MIX(RAB);
            par ^= 1;
        }
        if (pend) { stageB(par ^ 1); advance(); pend = false; }

        if constexpr (EPI == LX_OUT) {
            // accumulators -> rows of 64 columns through the wave's 4 KB of LDS, so that a store covers whole lines
            float* stg = reinterpret_cast<float*>(lsm + 4 * LX_ELEMS) + wave * (16 * 64);
            const int n = n0 + wn * 64 + (lane & 7) * 8;
            const float sc = p.scale != nullptr ? p.scale[0] : 1.0f;
#pragma unroll
            for (int tm = 0; tm < 8; ++tm) {
#pragma unroll
                for (int tn = 0; tn < 4; ++tn)
                    *reinterpret_cast<f32x4*>(stg + lr * 64 + (((tn * 4 + lg) ^ (lr & 7)) << 2)) = acc[tm][tn];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = half * 8 + srow;
                    f32x4 lo = *reinterpret_cast<const f32x4*>(stg + r * 64 + (((2 * (lane & 7)) ^ srow) << 2));
                    f32x4 hi = *reinterpret_cast<const f32x4*>(stg + r * 64 + (((2 * (lane & 7) + 1) ^ srow) << 2));
                    const int m = m0 + wm * 128 + tm * 16 + r;
                    if (m < p.M && n < p.N) {
                        if (p.slab != nullptr) {
                            float* q = p.slab + ((size_t)split * p.M + m) * p.N + n;
                            __builtin_nontemporal_store(lo, reinterpret_cast<f32x4*>(q));
                            __builtin_nontemporal_store(hi, reinterpret_cast<f32x4*>(q + 4));
                        } else {
                            lo *= sc;
                            hi *= sc;
                            if (p.add != nullptr) {
                                const float* q = p.add + (size_t)m * p.N + n;
                                lo += *reinterpret_cast<const f32x4*>(q);
                                hi += *reinterpret_cast<const f32x4*>(q + 4);
                            }
                            if (p.out_f32) {
                                float* q = reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n;
                                *reinterpret_cast<f32x4*>(q) = lo;
                                *reinterpret_cast<f32x4*>(q + 4) = hi;
                            } else {
                                const u32x4 o = {pack2bf(lo[0], lo[1]), pack2bf(lo[2], lo[3]), pack2bf(hi[0], hi[1]), pack2bf(hi[2], hi[3])};
                                __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(reinterpret_cast<bf16_t*>(p.out) + (size_t)m * p.ldo + n));
                            }
                        }
                    }
                }
            }
        } else {
            bf16_t* stg = reinterpret_cast<bf16_t*>(reinterpret_cast<float*>(lsm + 4 * LX_ELEMS) + wave * (16 * 64));
            // bias of the lane's 16 columns; columns behind the vocabulary count as logits of -inf
            float bias[4][4];
            bool in[4][4];
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = n0 + wn * 64 + tn * 16 + 4 * lg + j;
                    in[tn][j] = n < p.N;
                    const int nc = in[tn][j] ? n : p.N - 1;
                    bias[tn][j] = 0.f;
                    if (p.bias != nullptr) bias[tn][j] = p.bias_type == 1 ? bf2f(reinterpret_cast<const bf16_t*>(p.bias)[nc]) : reinterpret_cast<const float*>(p.bias)[nc];
                }
            const int sc = (n0 >> 6) + wn;
#pragma unroll
            for (int tm = 0; tm < 8; ++tm) {
                const int m = m0 + wm * 128 + tm * 16 + lr;
                float z[4][4], mx = -INFINITY, zs = 0.f;
#pragma unroll
                for (int tn = 0; tn < 4; ++tn)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float u = acc[tm][tn][j] + bias[tn][j];
                        zs += in[tn][j] ? u : 0.f;
                        z[tn][j] = in[tn][j] ? u : -INFINITY;
                        mx = fmaxf(mx, z[tn][j]);
                    }
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float ref = mx == -INFINITY ? 0.f : mx;        // a row of -inf only: exp(-inf - 0) = 0
                float s = 0.f;
#pragma unroll
                for (int tn = 0; tn < 4; ++tn)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        z[tn][j] = __builtin_amdgcn_exp2f((z[tn][j] - ref) * 1.44269504088896340736f);
                        s += z[tn][j];
                    }
                s += __shfl_xor(s, 16, 64);
                s += __shfl_xor(s, 32, 64);
                if (lg == 0 && m < p.M) p.stats[(size_t)m * p.stat_cols + sc] = make_float2(mx, s);
                if (p.zsum != nullptr) {
                    zs += __shfl_xor(zs, 16, 64);
                    zs += __shfl_xor(zs, 32, 64);
                    if (lg == 0 && m < p.M) p.zsum[(size_t)m * p.stat_cols + sc] = zs;
                }
                if (p.P != nullptr) {
#pragma unroll
                    for (int tn = 0; tn < 4; ++tn) {
                        uint2 w;
                        w.x = lx_pack_h(z[tn][0], z[tn][1]);
                        w.y = lx_pack_h(z[tn][2], z[tn][3]);
                        *reinterpret_cast<uint2*>(stg + lr * 64 + (((tn * 2 + (lg >> 1)) ^ (lr & 7)) << 3) + (lg & 1) * 4) = w;
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int r = half * 8 + srow;
                        const u32x4 o = *reinterpret_cast<const u32x4*>(stg + r * 64 + (((lane & 7) ^ srow) << 3));
                        const int mr = m0 + wm * 128 + tm * 16 + r;
                        if (mr < p.M)
                            __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(p.P + (size_t)mr * p.ldp + n0 + wn * 64 + (lane & 7) * 8));
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- rows
struct LxRowParams {
    const bf16_t* x; long long ldx;
    const bf16_t* w; long long ldw;
    const void* bias; int bias_type;
    const long long* target; long long ignore_index;
    const float2* stats; const float* zsum; int stat_cols;
    bf16_t* P; long long ldp;          // fp16 on entry, bf16 dz on exit; null: loss alone
    float* rows;
    int V, D;
    float smoothing;
};

static __device__ __forceinline__ float lx_block_max(float v, float* sh) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}
static __device__ __forceinline__ float lx_block_sum(float v, float* sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__global__ __launch_bounds__(256) void lx_row_kernel(const LxRowParams p) {
    __shared__ float sh[4];
    const int row = blockIdx.x;
    const long long t64 = p.target[row];
    bf16_t* P = p.P != nullptr ? p.P + (size_t)row * p.ldp : nullptr;
    const int chunks = (int)(p.ldp / 8);
    if (t64 == p.ignore_index) {
        if (threadIdx.x == 0) p.rows[row] = 0.f;
        if (P != nullptr)
            for (int c = threadIdx.x; c < chunks; c += 256) reinterpret_cast<u32x4*>(P)[c] = (u32x4){0u, 0u, 0u, 0u};
        return;
    }
    // a label outside [0, V) never becomes an address: the row's loss and gradient are NaN
    const bool valid = t64 >= 0 && t64 < (long long)p.V;
    const int t = valid ? (int)t64 : 0;
    const float2* st = p.stats + (size_t)row * p.stat_cols;
    float mx = -INFINITY;
    for (int c = threadIdx.x; c < p.stat_cols; c += 256) mx = fmaxf(mx, st[c].x);
    mx = lx_block_max(mx, sh);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float s = 0.f, zs = 0.f;
    for (int c = threadIdx.x; c < p.stat_cols; c += 256) {
        const float2 v = st[c];
        s += v.y * (v.x == -INFINITY ? 1.f : __expf(v.x - ref));         // an all -inf entry has s = 0, or NaN where a logit was NaN
        if (p.smoothing > 0.f) zs += p.zsum[(size_t)row * p.stat_cols + c];
    }
    s = lx_block_sum(s, sh);
    // the target's logit
    const bf16_t* xr = p.x + (size_t)row * p.ldx;
    const bf16_t* wr = p.w + (size_t)t * p.ldw;
    float dot = 0.f;
    for (int c = threadIdx.x; c < p.D / 8; c += 256) {
        float a[8], b[8];
        load8(xr + c * 8, a);
        load8(wr + c * 8, b);
#pragma unroll
        for (int k = 0; k < 8; ++k) dot = __builtin_fmaf(a[k], b[k], dot);
    }
    dot = lx_block_sum(dot, sh);
    if (p.smoothing > 0.f) zs = lx_block_sum(zs, sh);
    if (p.bias != nullptr) dot += p.bias_type == 1 ? bf2f(reinterpret_cast<const bf16_t*>(p.bias)[t]) : reinterpret_cast<const float*>(p.bias)[t];
    const float lse = ref + logf(s);
    if (threadIdx.x == 0) {
        float l = lse - dot;
        if (p.smoothing > 0.f) l = (1.f - p.smoothing) * l + p.smoothing * (lse - zs / (float)p.V);
        p.rows[row] = valid ? l : __builtin_nanf("");
    }
    if (P == nullptr) return;
    const float u = p.smoothing / (float)p.V, hit = 1.f - p.smoothing;
    for (int c = threadIdx.x; c < chunks; c += 256) {
        const u32x4 r = reinterpret_cast<const u32x4*>(P)[c];
        const float f = __expf(st[c >> 3].x - lse);
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned word = r[k];         // (a bit cast of the vector's element itself reads element 0)
            const f16x2 h = __builtin_bit_cast(f16x2, word);
            v[2 * k] = (float)h[0] * f - u;
            v[2 * k + 1] = (float)h[1] * f - u;
        }
        const int n = c * 8;
        if ((t >> 3) == c) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (n + k == t) v[k] -= hit;
        }
        if (!valid) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __builtin_nanf("");
        }
        if (n + 8 > p.V) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (n + k >= p.V) v[k] = 0.f;
        }
        const u32x4 o = {pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
        reinterpret_cast<u32x4*>(P)[c] = o;
    }
}

// count of the counted rows, the scale of the gradients (1 / count, or 1 for a sum; 0 without a counted row) and the loss, by one workgroup
__global__ __launch_bounds__(1024) void lx_loss_kernel(const long long* __restrict__ target, long long ignore_index, const float* __restrict__ rows, int T,
                                                       int mean, float* __restrict__ scale, float* __restrict__ loss) {
    __shared__ double sh[16];
    __shared__ int shc[16];
    double s = 0.0;
    int n = 0;
    for (int i = threadIdx.x; i < T; i += 1024) {
        if (target[i] != ignore_index) ++n;
        if (rows != nullptr) s += (double)rows[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); n += __shfl_xor(n, o, 64); }
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = s; shc[threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) { s += sh[w]; n += shc[w]; }
        if (scale != nullptr) *scale = n == 0 ? 0.f : mean ? (float)(1.0 / (double)n) : 1.f;
        if (loss != nullptr) *loss = (float)(n == 0 ? 0.0 : mean ? s / (double)n : s);
    }
}

// out = scale * sum over the splits of slab[s] (+ add), fixed order; N % 4 == 0
__global__ __launch_bounds__(256) void lx_reduce_kernel(const float* __restrict__ slab, int splits, int M, int N, const float* __restrict__ scale,
                                                        const float* __restrict__ add, void* __restrict__ out, long long ldo, int out_f32) {
    const size_t total = (size_t)M * N / 4, stride = (size_t)M * N;
    const float sc = scale != nullptr ? scale[0] : 1.0f;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const float* q = slab + i * 4;
        f32x4 s = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(q));
#pragma unroll 4
        for (int k = 1; k < splits; ++k) s += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(q + k * stride));
        s *= sc;
        if (add != nullptr) s += *reinterpret_cast<const f32x4*>(add + i * 4);
        const size_t m = i * 4 / N, n = i * 4 - m * N;
        if (out_f32) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(out) + m * ldo + n) = s;
        } else {
            uint2 o;
            o.x = pack2bf(s[0], s[1]);
            o.y = pack2bf(s[2], s[3]);
            *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(out) + m * ldo + n) = o;
        }
    }
}

// db: column sums of dz.  A block sums 512 columns over a range of rows into partial[range][ldp]; the second kernel adds the ranges in order.
__global__ __launch_bounds__(256) void lx_colsum_kernel(const bf16_t* __restrict__ dz, long long ldp, int T, int rows_per_range, float* __restrict__ partial) {
    __shared__ float sh[4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long col = (long long)blockIdx.x * 512 + lane * 8;
    const int r0 = blockIdx.y * rows_per_range, r1 = r0 + rows_per_range < T ? r0 + rows_per_range : T;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col < ldp) {
#pragma unroll 4
        for (int r = r0 + wave; r < r1; r += 4) {
            float v[8];
            load8(dz + (size_t)r * ldp + col, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += v[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sh[wave][lane * 8 + k] = acc[k];
    __syncthreads();
    for (int c = threadIdx.x; c < 512; c += 256) {
        const long long n = (long long)blockIdx.x * 512 + c;
        if (n < ldp) partial[(size_t)blockIdx.y * ldp + n] = (sh[0][c] + sh[1][c]) + (sh[2][c] + sh[3][c]);
    }
}
__global__ __launch_bounds__(256) void lx_colsum_final_kernel(const float* __restrict__ partial, long long ldp, int ranges, int V, const float* __restrict__ scale,
                                                              float* __restrict__ sum, int first, void* __restrict__ db, int db_f32) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= V) return;
    float s = first ? 0.f : sum[n];
    for (int r = 0; r < ranges; ++r) s += partial[(size_t)r * ldp + n];
    if (db == nullptr) { sum[n] = s; return; }
    s *= scale[0];
    if (db_f32) reinterpret_cast<float*>(db)[n] = s;
    else reinterpret_cast<bf16_t*>(db)[n] = f2bf(s);
}

// ---------------------------------------------------------------------------------------------------- host
#define LX_RANGES 64

static int lx_cus() {
    static int cache[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (cache[dev] == 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) { (void)hipGetLastError(); n = 256; }
        cache[dev] = n >= 8 ? n & ~7 : n;
    }
    return cache[dev];
}
static size_t lx_up(size_t n) { return (n + 255) & ~(size_t)255; }

// how the rows are cut and where everything lies in the workspace
struct LxPlan {
    long long ldp, stat_cols;
    int block, blocks;              // rows per block, blocks
    int dx_splits;
    size_t scale, stats, zsum, P, acc, slab, colpart, colsum, total;
};
// dx = dz W has few output tiles and a long contraction: it is cut so that about every compute unit has a share, at least 8 steps each
static int lx_dx_splits(int rows, int V, int D) {
    const long long tiles = (long long)((rows + LX_TILE - 1) / LX_TILE) * ((D + LX_TILE - 1) / LX_TILE);
    const long long steps = (V + LX_BK - 1) / LX_BK;
    long long s = 256 / tiles;
    if (s > steps / 8) s = steps / 8;
    return (int)(s < 1 ? 1 : s);
}
static LxPlan lx_plan(long long T, int V, int D, int grad, int smoothing, int dw_f32, int bias, size_t block_bytes) {
    LxPlan q = {};
    q.ldp = ((long long)V + LX_TILE - 1) / LX_TILE * LX_TILE;
    q.stat_cols = q.ldp / LX_STAT;
    const size_t row = (grad ? (size_t)q.ldp * 2 : 0) + (size_t)q.stat_cols * (smoothing ? 12 : 8);
    long long rows = (long long)(block_bytes / row) / LX_TILE * LX_TILE;
    if (rows < LX_TILE) rows = LX_TILE;
    if (rows > (1 << 22)) rows = 1 << 22;
    if (rows > T) rows = T;
    q.blocks = (int)((T + rows - 1) / rows);
    // equal blocks: the last one is not a remnant
    rows = (T + q.blocks - 1) / q.blocks;
    if (q.blocks > 1) rows = (rows + LX_TILE - 1) / LX_TILE * LX_TILE;
    q.block = (int)rows;
    q.blocks = (int)((T + rows - 1) / rows);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += lx_up(n); return here; };
    q.scale = take(16);
    q.stats = take((size_t)rows * q.stat_cols * sizeof(float2));
    q.zsum = smoothing ? take((size_t)rows * q.stat_cols * sizeof(float)) : 0;
    if (grad) {
        q.P = take((size_t)rows * q.ldp * 2);
        if (q.blocks > 1 && !dw_f32) q.acc = take((size_t)V * D * sizeof(float));
        q.dx_splits = lx_dx_splits((int)rows, V, D);
        if (q.dx_splits > 1) q.slab = take((size_t)q.dx_splits * rows * D * sizeof(float));
        if (bias) {
            q.colpart = take((size_t)LX_RANGES * q.ldp * sizeof(float));
            q.colsum = take((size_t)V * sizeof(float));
        }
    }
    q.total = at;
    return q;
}

template <int LAY, int EPI>
static int lx_launch(const LxGemmParams& p, hipStream_t s, const char* what) {
    static VitkLdsOnce once = {};
    if (int rc = vitk_lds_once(once, (const void*)lx_gemm_kernel<LAY, EPI>, LX_LDS, what)) return rc;
    const long long items = (long long)p.tiles_m * p.tiles_n * p.splits;
    const int cus = lx_cus();
    const int grid = items < cus ? (int)items : cus;
    lx_gemm_kernel<LAY, EPI><<<grid, 512, LX_LDS, s>>>(p);
    return vitk_check_launch(what);
}

extern "C" {

size_t vitk_linear_xent_workspace(int64_t T, int V, int D, int want_grad, int smoothing, int dw_f32, int bias, size_t block_bytes) {
    if (T <= 0 || T > 0x7fffffff || V <= 0 || V > (1 << 22) || D <= 0 || D > (1 << 20)) return 0;
    return lx_plan(T, V, D, want_grad, smoothing, dw_f32, bias, block_bytes).total;
}

int vitk_linear_xent(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_type, const int64_t* target, int64_t T, int V, int D,
                     float smoothing, int64_t ignore_index, int mean, float* loss, float* rows, void* dx, int64_t lddx, void* dw, int64_t lddw, int dw_f32,
                     void* db, int db_f32, void* workspace, size_t workspace_bytes, size_t block_bytes, void* stream) {
    VITK_REQUIRE(T > 0 && T <= 0x7fffffff && V > 0 && V <= (1 << 22) && D > 0 && D <= (1 << 20), "linear_xent: bad shape T=%lld V=%d D=%d", (long long)T, V, D);
    VITK_REQUIRE(x && w && target && loss && rows && workspace, "linear_xent: null pointer");
    VITK_REQUIRE(D % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && ldx >= D && ldw >= D && ldx < (1 << 22) && ldw < (1 << 22),
                 "linear_xent: D and the row strides must be multiples of 8, strides from D to 2^22 (D=%d ldx=%lld ldw=%lld)", D, (long long)ldx, (long long)ldw);
    VITK_REQUIRE(vitk_aligned(x, 16) && vitk_aligned(w, 16) && vitk_aligned(workspace, 256) && vitk_aligned(target, 8), "linear_xent: rows must be 16-byte aligned");
    VITK_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, "linear_xent: smoothing %g outside [0, 1]", (double)smoothing);
    VITK_REQUIRE(!bias || bias_type == 0 || bias_type == 1, "linear_xent: bias types are 0 (fp32) and 1 (bf16)");
    VITK_REQUIRE((dx != nullptr) == (dw != nullptr), "linear_xent: dx and dw go together");
    const bool grad = dx != nullptr;
    VITK_REQUIRE(!grad || (lddx % 8 == 0 && lddx >= D && lddw % 8 == 0 && lddw >= D && vitk_aligned(dx, 16) && vitk_aligned(dw, 16)),
                 "linear_xent: gradient rows must be 16-byte aligned with strides that are multiples of 8 (lddx=%lld lddw=%lld)", (long long)lddx, (long long)lddw);
    VITK_REQUIRE(!db || (grad && bias), "linear_xent: db needs a bias and the other gradients");
    const LxPlan q = lx_plan(T, V, D, grad, smoothing > 0.f, dw_f32, db != nullptr, block_bytes);
    VITK_REQUIRE(!grad || !dw_f32 || q.blocks == 1 || lddw == D, "linear_xent: an fp32 dw over several blocks of rows must be contiguous");
    if (workspace_bytes < q.total) {
        vitk_set_error("linear_xent: workspace %zu < %zu", workspace_bytes, q.total);
        return VITK_ENOSPC;
    }
    hipStream_t s = (hipStream_t)stream;
    char* ws = (char*)workspace;
    float* scale = (float*)(ws + q.scale);
    const long long* tg = (const long long*)target;
    if (q.blocks > 1 && grad) {
        lx_loss_kernel<<<1, 1024, 0, s>>>(tg, ignore_index, nullptr, (int)T, mean, scale, nullptr);
        if (int rc = vitk_check_launch("linear_xent_count")) return rc;
    }
    for (int b = 0; b < q.blocks; ++b) {
        const long long r0 = (long long)b * q.block;
        const int n = (int)(T - r0 < q.block ? T - r0 : q.block);
        const bool last = b == q.blocks - 1;
        LxGemmParams g = {};
        g.A = (const bf16_t*)x + r0 * ldx; g.lda = ldx; g.B = (const bf16_t*)w; g.ldb = ldw;
        g.M = n; g.N = V; g.KA = g.KB = D; g.steps = (D + LX_BK - 1) / LX_BK;
        g.tiles_m = (n + LX_TILE - 1) / LX_TILE; g.tiles_n = (int)(q.ldp / LX_TILE); g.band = 8; g.splits = 1;
        g.bias = bias; g.bias_type = bias_type;
        g.stats = (float2*)(ws + q.stats); g.stat_cols = (int)q.stat_cols; g.zsum = smoothing > 0.f ? (float*)(ws + q.zsum) : nullptr;
        g.P = grad ? (_Float16*)(ws + q.P) : nullptr; g.ldp = q.ldp;
        if (int rc = lx_launch<LX_NT, LX_XENT>(g, s, "linear_xent_logits")) return rc;
        LxRowParams r = {};
        r.x = g.A; r.ldx = ldx; r.w = g.B; r.ldw = ldw; r.bias = bias; r.bias_type = bias_type; r.target = tg + r0; r.ignore_index = ignore_index;
        r.stats = g.stats; r.zsum = g.zsum; r.stat_cols = g.stat_cols; r.P = (bf16_t*)g.P; r.ldp = q.ldp; r.rows = rows + r0; r.V = V; r.D = D; r.smoothing = smoothing;
        lx_row_kernel<<<n, 256, 0, s>>>(r);
        if (int rc = vitk_check_launch("linear_xent_rows")) return rc;
        if (last) {
            lx_loss_kernel<<<1, 1024, 0, s>>>(tg, ignore_index, rows, (int)T, mean, q.blocks > 1 ? nullptr : scale, loss);
            if (int rc = vitk_check_launch("linear_xent_loss")) return rc;
        }
        if (!grad) continue;
        const bf16_t* dz = (const bf16_t*)(ws + q.P);
        // dx = dz W: dz is zero behind the vocabulary up to its row stride
        LxGemmParams d = {};
        d.A = dz; d.lda = q.ldp; d.B = (const bf16_t*)w; d.ldb = ldw; d.M = n; d.N = D; d.KA = (int)q.ldp; d.KB = V; d.steps = (V + LX_BK - 1) / LX_BK;
        d.tiles_m = (n + LX_TILE - 1) / LX_TILE; d.tiles_n = (D + LX_TILE - 1) / LX_TILE; d.band = 8; d.splits = q.dx_splits;
        d.scale = scale; d.out = (bf16_t*)dx + r0 * lddx; d.ldo = lddx; d.slab = q.dx_splits > 1 ? (float*)(ws + q.slab) : nullptr;
        if (int rc = lx_launch<LX_NN, LX_OUT>(d, s, "linear_xent_dx")) return rc;
        if (d.slab != nullptr) {
            const long long total = (long long)n * D / 4;
            const int grid = (int)((total + 255) / 256 < 2048 ? (total + 255) / 256 : 2048);
            lx_reduce_kernel<<<grid, 256, 0, s>>>(d.slab, d.splits, n, D, scale, nullptr, d.out, lddx, 0);
            if (int rc = vitk_check_launch("linear_xent_dx_sum")) return rc;
        }
        // dW = dz^T x, summed over the blocks in fp32
        LxGemmParams e = {};
        e.A = dz; e.lda = q.ldp; e.B = g.A; e.ldb = ldx; e.M = V; e.N = D; e.KA = e.KB = n; e.steps = (n + LX_BK - 1) / LX_BK;
        e.tiles_m = (V + LX_TILE - 1) / LX_TILE; e.tiles_n = (D + LX_TILE - 1) / LX_TILE; e.band = 8; e.splits = 1;
        e.scale = scale;
        float* acc = dw_f32 ? (float*)dw : (float*)(ws + q.acc);
        e.add = b > 0 ? acc : nullptr;
        if (last) { e.out = dw; e.ldo = lddw; e.out_f32 = dw_f32; }
        else { e.out = acc; e.ldo = D; e.out_f32 = 1; }
        if (int rc = lx_launch<LX_TN, LX_OUT>(e, s, "linear_xent_dw")) return rc;
        if (db != nullptr) {
            float* part = (float*)(ws + q.colpart);
            int per = (n + LX_RANGES - 1) / LX_RANGES;
            if (per < 32) per = 32;
            const int ranges = (n + per - 1) / per;
            lx_colsum_kernel<<<dim3((unsigned)((q.ldp + 511) / 512), ranges), 256, 0, s>>>(dz, q.ldp, n, per, part);
            lx_colsum_final_kernel<<<(V + 255) / 256, 256, 0, s>>>(part, q.ldp, ranges, V, scale, (float*)(ws + q.colsum), b == 0, last ? db : nullptr, db_f32);
            if (int rc = vitk_check_launch("linear_xent_db")) return rc;
        }
    }
    return VITK_OK;
}

}  // extern "C"
