// Softmax cross entropy of a linear layer over a large vocabulary, with its gradients.  The logits stay in registers; what the gradients need of
// them is kept in 2 bytes each, for a block of rows at a time.
//
//   z = x W^T + b      lse_i = log sum_j exp z_ij      loss_i = lse_i - (1 - e) z_i,t(i) - e/V sum_j z_ij
//   dz_ij = p_ij - (1 - e) [j = t(i)] - e/V            dx = g dz W      dW = g dz^T x      db = g sum_i dz_i
//
// x bf16 [T, D], W bf16 [V, D].  The rows are worked through in blocks whose size the workspace bounds; per block
//   1. x W^T tile by tile (lx_logits_kernel).  The epilogue takes a tile's logits in fp32 from the accumulators: per row and 64
//      columns their maximum m and s = sum exp(z - m) go to a small table; exp(z - m) itself, in [0, 1], goes to the block's
//      matrix P in 16 bits of its own: no sign, 6 bits of exponent, 10 of fraction, from 1 down to 2^-62 (lx_pack_p).  fp16 has the same 11 bits
//      but ends at 6e-8 of the piece's maximum, and a class that stays 18 powers of e below a neighbour would lose its row of dW and its
//      db, which have no larger neighbour in their sums; bf16 would round 8 times as far.  Loss alone: only the table is written.
//   2. one workgroup per row (lx_row_kernel): lse from the table, the target's logit as a dot product of its own, the row's loss, and
//      P -> dz in place, now bf16: the one rounding of the gradient's factor.  Constants are kept out of it, because each would be rounded
//      by up to 1 part in 256 in the same direction everywhere: dz is divided by g and by a number that makes 1 - e a bf16 number and
//      e/V nearly one (lx_factor); both multiply the fp32 sums of the next step.
//      Where dW is wanted it also copies x, with zeros for the rows that are not counted: their dz is zero, but zero times what such a row may
//      hold (infinities, NaN) would not be.  2 T D bytes written beside the 4 T V of P: 0.3 to 1.4 % of a call.
//   3. dx = dz W and dW = dz^T x (lx_grad_kernel), and the column sums for db, to which each target's dz adds what its rounding took (near
//      -(1 - e) a probability of less than 2^-9 vanishes).
// 6 T V D floating-point operations: nothing is computed twice.  Keeping one 16-bit factor per logit of a block costs 4 bytes of
// traffic per logit for step 2, where computing the logits again for the gradients would cost 2 D operations.
#include "common.h"
#include "gemm_nt.h"

#define LX_BK 64
#define LX_TILE 256
#define LX_ELEMS (LX_TILE * LX_BK)                            // elements per operand tile
#define LX_LDS (4 * LX_ELEMS * 2 + 8 * 16 * 64 * 4)           // two buffers of both tiles, 4 KB of epilogue staging per wave
#define LX_GRAD_LDS (4 * LX_ELEMS * 2 + 4 * 16 * 64 * 4)
#define LX_STAT 64                                            // columns per entry of the statistics table

enum { LX_NT = 0, LX_NN = 1, LX_TN = 2 };
enum { LX_OUT = 0, LX_XENT = 1, LX_XENT_BIAS = 2 };       // LX_XENT_BIAS: with a bias or the sums of the logits

// 512 bytes of zeros (never written): what rows and columns behind the contraction's end are read from
__device__ __attribute__((aligned(512))) unsigned lx_zero_row[128];

struct LxGemmParams {
    const bf16_t* A; const bf16_t* B;       // NT: A [M][KA], B [N][KB];  NN: B [KB][N];  TN: A [KA][M], B [KB][N]
    int lda, ldb;
    int M, N;
    int KA, KB;             // valid extent of the contraction in each operand; behind it zeros are read (lx_grad_kernel: A holds them)
    int steps;              // 64-deep steps over the whole contraction
    int tiles_m, tiles_n;
    // work, LX_XENT*: workgroup g of G takes the tiles g, g + G, ... (in bands of 8 column tiles)
    // work, LX_OUT: see LxDeal
    int width, teams, whole, rest, ranges;
    int splits;             // the small kernel: ranges of steps
    // LX_OUT: out[m][n] = scale[0] * acc (+ add[m][n]), bf16 or fp32
    const float* scale;
    const float* add;
    void* out; long long ldo; int out_f32;
    float* slab;
    // LX_XENT
    const void* bias; int bias_type;        // 0 fp32, 1 bf16, null: none
    float2* stats; int stat_cols;           // [M][stat_cols]: (m, s) of 64 columns
    float* zsum;                            // [M][stat_cols] sums of the logits, null: not wanted (no smoothing)
    unsigned short* P; long long ldp;       // (lx_pack_p) null: loss alone
    unsigned* ticket;                       // zeroed here for the kernels that follow
};

static __device__ __forceinline__ int lx_swz(int m) { return (((m >> 3) & 1) << 3) | ((m & 3) << 1); }
static __device__ __forceinline__ bf16x8 lx_tr(const bf16_t* lo, const bf16_t* hi) {
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)lo);
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)hi);
    return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// P's numbers, at most 1.  Times 2^-64 their fp32 exponent field ends at 63 (6 bits); 10 bits of the fraction are kept, to nearest.  Read back, the 16
// bits in place are that number again (its subnormals too: exponent field 0), and 2^64 goes into the factor it is multiplied with.  (2^-64 within
// the exponential's argument saves the product, but rounds the argument to 4e-6 there: the row sums of few classes were twice as far off.)
static __device__ __forceinline__ unsigned lx_pack_p(float a, float b) {
    const unsigned x = (__float_as_uint(a * 0x1p-64f) + 0x1000u) << 3, y = (__float_as_uint(b * 0x1p-64f) + 0x1000u) << 3;
    return __builtin_amdgcn_perm(y, x, 0x07060302u);        // the upper halves of both
}
static __device__ __forceinline__ float lx_unpack_p(unsigned v) { return __uint_as_float(v << 13); }

// v combined over the four lanes that share a row (lane ^ 16, lane ^ 32), by the lane swaps of the vector unit: no trip through LDS
template <class F>
static __device__ __forceinline__ float lx_over_row(float v, F&& f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The loss's epilogue of a wave that holds FM * 16 rows (from m0) by 64 columns (from n0) of logits: lane (lr, lg) has columns 16 tn + 4 lg + j
// of row 16 tm + lr.  stg: 2 KB of LDS of the wave's own, through which P leaves in rows of 64 columns so that a store covers whole lines.
// EXTRA: with a bias or the sums of the logits.  WANT_P, FULL (every row is one of the matrix): so that the code of the rows has no branch and the
// rows' chains of maximum, exponentials and sum overlap (a branch per row and the sums through LDS cost 2 % of the logits at 8192 x 100003 x
// 2048, 4 % at 2047 x 50021 x 1024).
template <int FM, bool EXTRA, bool WANT_P, bool FULL>
static __device__ __forceinline__ void lx_loss_rows(const LxGemmParams& p, f32x4 (&acc)[FM][4], int m0, int n0, bf16_t* stg) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));          // what is derived from it is not to be kept in registers over the main loop
    const int lr = lane & 15, lg = lane >> 4, srow = lane >> 3;
    const int room = p.N - n0 - 4 * lg;              // the lane's columns with 16 tn + j < room are columns of the vocabulary
    float mxs[FM], sums[FM], zsums[FM];
#pragma unroll
    for (int tm = 0; tm < FM; ++tm) {
        float z[4][4], mx = acc[tm][0][0];
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
            for (int j = 0; j < 4; ++j) mx = fmaxf(mx, acc[tm][tn][j]);
        if constexpr (EXTRA) {
            float q[4];
#pragma unroll
            for (int tn = 0; tn < 4; ++tn) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = tn * 16 + j < room ? acc[tm][tn][j] : 0.f;
                q[tn] = (v[0] + v[1]) + (v[2] + v[3]);
            }
            zsums[tm] = lx_over_row((q[0] + q[1]) + (q[2] + q[3]), [](float a, float b) { return a + b; });
        }
        mx = lx_over_row(mx, [](float a, float b) { return fmaxf(a, b); });
        // The maximum is taken off before the product with log2(e), so that the largest gives 1 exactly however large the logits are.  (With
        // z * log2(e) - fl(m * log2(e)) as one fma a logit saves an instruction, 0.5 to 1 % of a call, but from logits of 10^7 on the product's
        // rounding is whole powers of two; a second form for those, behind a branch, spills the accumulators.)
        const float off = mx == -INFINITY ? 0.f : mx;         // a row of -inf only: 2^(-inf) = 0
        float q[4];
#pragma unroll
        for (int tn = 0; tn < 4; ++tn) {
#pragma unroll
            for (int j = 0; j < 4; ++j) z[tn][j] = __builtin_amdgcn_exp2f((acc[tm][tn][j] - off) * 1.44269504088896340736f);
            q[tn] = (z[tn][0] + z[tn][1]) + (z[tn][2] + z[tn][3]);
        }
        mxs[tm] = mx;
        sums[tm] = lx_over_row((q[0] + q[1]) + (q[2] + q[3]), [](float a, float b) { return a + b; });
        if constexpr (WANT_P) {
#pragma unroll
            for (int tn = 0; tn < 4; ++tn) {
                uint2 w;
                w.x = lx_pack_p(z[tn][0], z[tn][1]);
                w.y = lx_pack_p(z[tn][2], z[tn][3]);
                *reinterpret_cast<uint2*>(stg + lr * 64 + (((tn * 2 + (lg >> 1)) ^ (lr & 7)) << 3) + (lg & 1) * 4) = w;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = half * 8 + srow;
                const u32x4 o = *reinterpret_cast<const u32x4*>(stg + r * 64 + (((lane & 7) ^ srow) << 3));
                const int mr = m0 + tm * 16 + r;
                if (FULL || mr < p.M) __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(p.P + (size_t)mr * p.ldp + n0 + (lane & 7) * 8));
            }
        }
    }
    // lane group lg stores the statistics of the rows of tm = lg, lg + 4
#pragma unroll
    for (int h = 0; h < (FM + 3) / 4; ++h) {
        float mx = mxs[4 * h], sum = sums[4 * h], zsum = EXTRA ? zsums[4 * h] : 0.f;
#pragma unroll
        for (int k = 1; k < 4 && 4 * h + k < FM; ++k) {
            mx = lg == k ? mxs[4 * h + k] : mx;
            sum = lg == k ? sums[4 * h + k] : sum;
            if constexpr (EXTRA) zsum = lg == k ? zsums[4 * h + k] : zsum;
        }
        const int m = m0 + (4 * h + lg) * 16 + lr;
        if (4 * h + lg < FM && (FULL || m < p.M)) {
            const size_t at = (size_t)m * p.stat_cols + (n0 >> 6);
            p.stats[at] = make_float2(mx, sum);
            if (EXTRA && p.zsum != nullptr) p.zsum[at] = zsum;
        }
    }
}
template <int FM, bool EXTRA>
static __device__ __forceinline__ void lx_loss_epilogue(const LxGemmParams& p, f32x4 (&acc)[FM][4], int m0, int n0, bf16_t* stg) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int first = n0 + 4 * (lane >> 4), room = p.N - first;
    if constexpr (EXTRA) {
        if (p.bias != nullptr) {
#pragma unroll
            for (int tn = 0; tn < 4; ++tn) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = first + tn * 16 + j < p.N ? first + tn * 16 + j : p.N - 1;
                    const float u = p.bias_type == 1 ? bf2f(reinterpret_cast<const bf16_t*>(p.bias)[n]) : reinterpret_cast<const float*>(p.bias)[n];
#pragma unroll
                    for (int tm = 0; tm < FM; ++tm) acc[tm][tn][j] += u;
                }
            }
        }
    }
    if (n0 + 64 > p.N) {           // columns behind the vocabulary count as logits of -inf
#pragma unroll
        for (int tm = 0; tm < FM; ++tm)
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[tm][tn][j] = tn * 16 + j < room ? acc[tm][tn][j] : -INFINITY;
    }
    const bool full = m0 + FM * 16 <= p.M;
    if (p.P != nullptr) {
        if (full) lx_loss_rows<FM, EXTRA, true, true>(p, acc, m0, n0, stg);
        else lx_loss_rows<FM, EXTRA, true, false>(p, acc, m0, n0, stg);
    } else {
        if (full) lx_loss_rows<FM, EXTRA, false, true>(p, acc, m0, n0, stg);
        else lx_loss_rows<FM, EXTRA, false, false>(p, acc, m0, n0, stg);
    }
}

// range g of G of `total` steps: total / G each, the first total % G one more
static __host__ __device__ __forceinline__ void lx_range(int g, int total, int G, int& from, int& to) {
    const int q = total / G, r = total - q * G;
    from = g * q + (g < r ? g : r);
    to = from + q + (g < r ? 1 : 0);
}

#define LX_WAIT(n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n) : "memory")
#define LX_BARRIER()                       \
    __builtin_amdgcn_s_barrier();          \
    asm volatile("" ::: "memory")

// The logits: one 512-thread workgroup per compute unit works through 256 x 256 tiles, 8 waves (2 x 4) of 128 x 64 = 128 accumulator registers each,
// 64-deep steps.  Operands go from memory to LDS by DMA, two steps ahead across tile borders, into a double buffer; fragments are read one
// phase of 16 matrix instructions before their use.  An operand sits in LDS as [256][64], its 16-byte chunks XOR-swizzled by the row, and is
// read with ds_read_b128.  The matrix instruction's operands are swapped, so a lane holds four consecutive columns of one output row.
// Tiles are dealt by number (no counters: a captured graph may be replayed on any stream): workgroup g of G takes the tiles g, g + G, ...,
// in bands of 8 column tiles, which keeps what the 32 workgroups of an XCD read at a time to 4 row panels and 8 column panels.
// Two waves share a SIMD because the loss's epilogue is vector arithmetic (an exponential per logit), which one wave's stalls would leave
// uncovered: with four waves as in lx_grad_kernel 8192 x 100003 x 2048 takes 2820 instead of 2550 us, 2047 x 50021 x 1024 239 instead of 182.
// Matrix pipe 68 % busy at the first of these; a library product of the two operands alone takes 2501 us.
template <int EPI>
__global__ __launch_bounds__(512) void lx_logits_kernel(const LxGemmParams p) {
    extern __shared__ __attribute__((aligned(16))) bf16_t lsm[];   // [2 buffers][A tile | B tile], [8 waves][16][64] fp32

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int lr = lane & 15, lg = lane >> 4;
    const unsigned lds_base = __builtin_amdgcn_readfirstlane(lds_addr(lsm));
    const unsigned lds_stage = (unsigned)(wave * 4 * 1024);

    const int G = gridDim.x, tiles = p.tiles_m * p.tiles_n;
    const int items = __builtin_amdgcn_readfirstlane((int)blockIdx.x < tiles ? (tiles - 1 - (int)blockIdx.x) / G + 1 : 0);

    // ---- staging: where the next step's operands come from.  A piece is one instruction of one wave, 1 KB of LDS: 8 rows, LDS position lane % 8
    // receives chunk (lane % 8) ^ (row & 7).  A is staged in two halves, the rows that are the first 64 of a wave's 128 and the others.
    int sv = 0, sk = 0;
    const bf16_t* sA = p.A;
    const bf16_t* sB = p.B;
    unsigned voA[4], voB[4];
    auto locate = [&](int v, int& m0, int& n0) {
        const int tile = xcd_remap(blockIdx.x + v * G, tiles);
        const int full = p.tiles_m * 8;
        const int blk = tile / full;
        const int rem = tile - blk * full;
        const int c0 = blk * 8;
        const int width = p.tiles_n - c0 < 8 ? p.tiles_n - c0 : 8;
        const int tm = rem / width;
        // the divisions run on the vector unit: say that their results are the same in every lane
        m0 = __builtin_amdgcn_readfirstlane(tm * LX_TILE);
        n0 = __builtin_amdgcn_readfirstlane((c0 + rem - tm * width) * LX_TILE);
    };
    auto aim = [&](int v) {
        int m0, n0;
        locate(v, m0, n0);
        sk = 0;
        sA = p.A + (size_t)m0 * p.lda;
        sB = p.B + (size_t)n0 * p.ldb;
        // rows behind the edge of the output read the last valid ones: their results are not stored
        const int ma = p.M - 1 - m0, mb = p.N - 1 - n0;
        // the lane number passes through an empty asm, so that what is derived from it here is not kept in registers over the main loop
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int srow = ln >> 3, sch = (ln & 7) ^ srow;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = wave * 2 + (j & 1);
            const int ra = (b >> 3) * 128 + (j >> 1) * 64 + (b & 7) * 8 + srow, rb = (wave * 4 + j) * 8 + srow;
            voA[j] = (unsigned)(((ra < ma ? ra : ma) * p.lda + sch * 8) * 2);
            voB[j] = (unsigned)(((rb < mb ? rb : mb) * p.ldb + sch * 8) * 2);
        }
    };
    // what lies behind the contraction's end comes from the zero row (the lane number passes through an empty asm as in aim)
    auto stageA = [&](int par, int half) {
        const bf16_t* src = sA + (size_t)sk * LX_BK;
        const unsigned dst = lds_base + (unsigned)(par * 2 * LX_ELEMS * 2) + (wave >> 2) * 16384 + half * 8192 + (wave & 3) * 2048;
        if ((sk + 1) * LX_BK <= p.KA) {
            glds16(src, voA[2 * half], dst);
            glds16(src, voA[2 * half + 1], dst + 1024);
        } else {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const void* zrow = (const char*)lx_zero_row + (ln & 31) * 16;
            const int k = sk * LX_BK + ((ln & 7) ^ (ln >> 3)) * 8;
#pragma unroll
            for (int j = 0; j < 2; ++j) glds16_v(k < p.KA ? (const void*)((const char*)src + voA[2 * half + j]) : zrow, dst + j * 1024);
        }
    };
    auto stageB = [&](int par) {
        const bf16_t* src = sB + (size_t)sk * LX_BK;
        const unsigned dst = lds_base + (unsigned)((par * 2 + 1) * LX_ELEMS * 2) + lds_stage;
        if ((sk + 1) * LX_BK <= p.KA) {
#pragma unroll
            for (int j = 0; j < 4; ++j) glds16(src, voB[j], dst + j * 1024);
        } else {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const void* zrow = (const char*)lx_zero_row + (ln & 31) * 16;
            const int k = sk * LX_BK + ((ln & 7) ^ (ln >> 3)) * 8;
#pragma unroll
            for (int j = 0; j < 4; ++j) glds16_v(k < p.KA ? (const void*)((const char*)src + voB[j]) : zrow, dst + j * 1024);
        }
    };
    auto advance = [&]() {
        if (++sk == p.steps) {
            ++sv;
            if (sv < items) aim(sv);
        }
    };

    // ---- fragments
    int offA[2], offB[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int x = ((ks * 4 + lg) ^ (lr & 7)) << 3;
        offA[ks] = (wm * 128 + lr) * LX_BK + x;
        offB[ks] = (wn * 64 + lr) * LX_BK + x;
    }
    f32x4 acc[8][4];
    bf16x8 faE[4], faO[4], fbE[4], fbO[4];
    auto ldA = [&](bf16x8 (&f)[4], const bf16_t* cA, int ks, int h) {
#pragma unroll
        for (int t = 0; t < 4; ++t) f[t] = *reinterpret_cast<const bf16x8*>(cA + offA[ks] + (4 * h + t) * 16 * LX_BK);
    };
    auto ldB = [&](bf16x8 (&f)[4], const bf16_t* cB, int ks) {
#pragma unroll
        for (int t = 0; t < 4; ++t) f[t] = *reinterpret_cast<const bf16x8*>(cB + offB[ks] + t * 16 * LX_BK);
    };
    auto mma = [&](const bf16x8 (&fa)[4], const bf16x8 (&fb)[4], int h) {
#pragma unroll
        for (int tm = 0; tm < 4; ++tm)
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
                acc[4 * h + tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[tn], fa[tm], acc[4 * h + tm][tn], 0, 0, 0);
    };
    // interleave a phase's 16 matrix instructions with its LDS reads
#define LX_MIX(reads)                                                                 \
    _Pragma("unroll") for (int i = 0; i < (reads); ++i) {                             \
        __builtin_amdgcn_sched_group_barrier(0x008, 16 / (reads), 0);                 \
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                            \
    }                                                                                 \
    __builtin_amdgcn_sched_barrier(0)

    // The steps of all tiles of a workgroup form one stream, requested two steps ahead into the buffer of the current one.  A step is four
    // phases: (A half 0, k 0..31), (half 1, k 0..31), (half 0, k 32..63), (half 1, k 32..63), fragments read one phase ahead; behind the
    // third the whole buffer has been read and the barrier opens it: the requests for A of step s + 2 go out, a phase later those for B;
    // they have 0.75 to 1 step to arrive.  (Requesting B and half of A after the first phase, with a second barrier, costs a step 8 %.)
    // The output stores of a full tile (16 of a wave at least) between two steps may stay in flight over the first step's waits.
    if (blockIdx.x == 0 && tid == 0) *p.ticket = 0u;
    if (items == 0) return;
    aim(0);
    stageB(0); stageA(0, 0); stageA(0, 1);
    advance();
    if (sv < items) {
        stageB(1); stageA(1, 0); stageA(1, 1);
        advance();
        LX_WAIT(8);
    } else {
        LX_WAIT(0);
    }
    LX_BARRIER();
    ldB(fbE, lsm + LX_ELEMS, 0);
    ldA(faE, lsm, 0, 0);
    int par = 0;
    bool loose = false;         // at least 16 output stores of this wave are younger than its requests
    bool pend = false;          // A of a step is on its way into the other buffer, B is not yet requested

    for (int v = 0; v < items; ++v) {
        int m0, n0;
        locate(v, m0, n0);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int kt = 0; kt < p.steps; ++kt) {
            const bf16_t* cA = lsm + par * 2 * LX_ELEMS;
            const bf16_t* cB = cA + LX_ELEMS;
            const bf16_t* nA = lsm + (par ^ 1) * 2 * LX_ELEMS;
            const bf16_t* nB = nA + LX_ELEMS;
            if (pend) { stageB(par ^ 1); advance(); pend = false; }
            mma(faE, fbE, 0);
            ldA(faO, cA, 0, 1);
            LX_MIX(4);
            mma(faO, fbE, 1);
            ldB(fbO, cB, 1);
            ldA(faE, cA, 1, 0);
            LX_MIX(8);
            mma(faE, fbO, 0);
            ldA(faO, cA, 1, 1);
            LX_MIX(4);
            if (loose) LX_WAIT(16);
            else LX_WAIT(0);
            LX_BARRIER();
            if (sv < items) { stageA(par, 0); stageA(par, 1); pend = true; }
            mma(faO, fbO, 1);
            ldB(fbE, nB, 0);
            ldA(faE, nA, 0, 0);
            LX_MIX(8);
            loose = false;
            par ^= 1;
        }
        if (pend) { stageB(par ^ 1); advance(); pend = false; }      // before the stores: vmcnt counts in issue order
        lx_loss_epilogue<8, EPI == LX_XENT_BIAS>(p, acc, m0 + wm * 128, n0 + wn * 64, reinterpret_cast<bf16_t*>(lsm + 4 * LX_ELEMS) + wave * (16 * 64 * 2));
        loose = m0 + LX_TILE <= p.M && p.P != nullptr;       // every row is stored: 16 stores at least
    }
}

template <int I> struct lx_int { static constexpr int value = I; };
template <int FROM, int TO, class F>
static __device__ __forceinline__ void lx_static_for(F&& f) {
    if constexpr (FROM < TO) {
        f(lx_int<FROM>{});
        lx_static_for<FROM + 1, TO>(f);
    }
}
template <int OFF>
static __device__ __forceinline__ void lx_dma(const bf16_t* base, unsigned voff, unsigned lds_byte) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds_byte), "n"(OFF) : "memory", "m0", "scc");
}
static __device__ __forceinline__ void lx_mfma(f32x4& c, const bf16x8& a, const bf16x8& b) {
    asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
static __device__ __forceinline__ bf16x4 lx_lds_tr(unsigned at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) bf16x4*)(__UINTPTR_TYPE__)at);
}
static __device__ __forceinline__ bf16x8 lx_join(const bf16x4 a, const bf16x4 b) { return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}; }
static __device__ __forceinline__ bf16x8 lx_lds_row(unsigned at) {
    return *(const __attribute__((address_space(3))) bf16x8*)(__UINTPTR_TYPE__)at;
}
// to the other buffer, 64 KB on (the operands begin at LDS address 0, which the launch has no static LDS to move)
static __device__ __forceinline__ void lx_flip(unsigned& at) { asm volatile("v_xor_b32 %0, 0x10000, %0" : "+v"(at)); }
#define LX_PIN() __builtin_amdgcn_sched_barrier(0)
#define LX_LDS_DONE() __builtin_amdgcn_s_waitcnt(0xc07f)         // lgkmcnt(0) as the compiler knows it: it adds no waits of its own behind it

// The gradients, dx = dz W (NN) and dW = dz^T x (TN): persistent 256 x 256 tiles as above, but four waves (2 x 2) of 128 x 128, one on a SIMD with the
// whole register file: 256 accumulators, fragments of a k half in use and of the next one arriving.  What bounds the eight-wave form is LDS:
// its waves read 192 KB a step and the DMA writes 64 KB, together as many cycles at 128 bytes each as the matrix instructions take; four waves
// read 128 KB.  But one wave to a SIMD hides nothing: every other instruction has to be issued in the 12 cycles a matrix instruction leaves, so
// the order is written out instruction by instruction (the matrix instructions are inline assembly on accumulators that never move; a
// scheduling barrier stands behind each), with one LDS read or one request (three instructions) in a gap, requests 3 to 6 matrix
// instructions apart because each keeps the path to LDS busy for 16 cycles and a wave that runs into another's waits (issued in a burst,
// or at every third gap of half the step, they cost a step 1000 cycles of 2060), and the step's own bookkeeping - addresses, buffer
// change - in the same gaps.
// Power is the limit behind that: 32 x 32 x 16 instructions take the same cycles at a 10 % lower clock (2260 -> 2480 us), and every second row of the
// 8 x 8 runs backwards, so that an operand stays from row to row (0.4 %).
// Operands whose rows run along the output (x, W, and dz for dW) sit in LDS as [64][256] and are read with the transposing ds_read_b64_tr_b16:
// no transposed copy is made; dz for dx as [256][64] with ds_read_b128.
//   8192 x 100003 x 2048: dz W 2520 -> 2180 us, dz^T x 2500 -> 2330 us (matrix pipe 81 % and 79 % busy at 1.8 and 1.7 GHz; a library product of the same sizes and
//   the layout it likes best 2117 and 2299 us).  25088 x 8192 x 768: 320 -> 284 and 289 -> 277 us.
// Tiles are dealt by number as LxDeal says.
template <int LAY>
__global__ __launch_bounds__(256, 1) void lx_grad_kernel(const LxGemmParams p) {
    constexpr bool AT = LAY == LX_TN;               // A is stored with the contraction as its slow dimension (B always is)
    extern __shared__ __attribute__((aligned(16))) bf16_t lsm[];   // [2 buffers][A tile | B tile], [4 waves][16][64] fp32

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int lr = lane & 15, lg = lane >> 4;
    const int lq = lr >> 2, lp = lr & 3;
    const unsigned lds_base = __builtin_amdgcn_readfirstlane(lds_addr(lsm));

    const int G = gridDim.x;
    const int id = xcd_remap(blockIdx.x, G);        // a team's workgroups are neighbours on one XCD
    const int team = __builtin_amdgcn_readfirstlane(id / p.width);
    const int member = __builtin_amdgcn_readfirstlane(id - team * p.width);
    const int whole_items = __builtin_amdgcn_readfirstlane(team < p.whole ? (p.whole - 1 - team) / p.teams + 1 : 0);
    int parts = 0, r0 = 0, r1 = 0, rt = 0;
    if (team < p.ranges) {
        lx_range(team, p.rest * p.steps, p.ranges, r0, r1);
        r0 = __builtin_amdgcn_readfirstlane(r0);
        r1 = __builtin_amdgcn_readfirstlane(r1);
        rt = __builtin_amdgcn_readfirstlane(r0 / p.steps);        // row (of the rest) of the first part
        parts = r1 > (rt + 1) * p.steps ? 2 : 1;
    }
    const int items = whole_items + parts;

    int sv = 0, sk = 0, sk_end = 0;
    const bf16_t* sA = p.A;
    const bf16_t* sB = p.B;
    unsigned voA[8], voB[8];
    // item v: where its tile is, its steps k0 .. k1 - 1, and which part it is (-1: a whole tile)
    auto locate = [&](int v, int& m0, int& n0, int& k0, int& k1, int& part) {
        k0 = 0;
        k1 = p.steps;
        part = -1;
        int row = v * p.teams + team;
        if (v >= whole_items) {
            part = v - whole_items;
            row = p.whole + rt + part;
            if (part == 0) k0 = r0 - rt * p.steps;
            const int left = r1 - (rt + part) * p.steps;
            k1 = left < p.steps ? left : p.steps;
        }
        const int blk = row / p.tiles_m;
        const int tm = row - blk * p.tiles_m, tn = blk * p.width + member;
        m0 = __builtin_amdgcn_readfirstlane(tm * LX_TILE);
        n0 = __builtin_amdgcn_readfirstlane(tn * LX_TILE);
    };
    // ---- requests.  A step's operand is eight pieces of 1 KB per wave, each an instruction.  [256][64]: 8 rows each, LDS position lane % 8 receives
    // chunk (lane % 8) ^ (row & 7).  [64][256]: two rows each, pieces 0..3 of the contraction's first 32, position lane % 32 receives chunk
    // (lane % 32) ^ lx_swz(row).  What lies behind the contraction's end needs no zeros in B, because A has them: dz is zero from the vocabulary's end
    // to its row stride and, for dW, from the last row to a multiple of 64.  There B repeats its last row.
    auto aim_rows = [&](unsigned (&vo)[8], int ld, int most) {
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int srow = ln >> 3, sch = (ln & 7) ^ srow;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = (wave * 8 + j) * 8 + srow;
            vo[j] = (unsigned)(((r < most ? r : most) * ld + sch * 8) * 2);
        }
    };
    auto aim_cols = [&](unsigned (&vo)[8], int ld, int last, int most) {        // last: rows behind it re-read it; most: likewise columns
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int shalf = ln >> 5, spos = ln & 31;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = (j >> 2) * 32 + (wave * 4 + (j & 3)) * 2 + shalf;
            const int c = (spos ^ lx_swz(r)) * 8;
            vo[j] = (unsigned)(((r < last ? r : last) * ld + (c < most ? c : most)) * 2);
        }
    };
    int sm0 = 0, sn0 = 0;
    const long long dA = AT ? (long long)LX_BK * p.lda : LX_BK, dB = (long long)LX_BK * p.ldb;
    auto aim = [&](bool next) {
        if (next) {
            int part;
            locate(sv, sm0, sn0, sk, sk_end, part);
        }
        sA = p.A + (AT ? (size_t)sm0 : (size_t)sm0 * p.lda) + sk * dA;
        sB = p.B + sn0 + sk * dB;
        if (AT) aim_cols(voA, p.lda, LX_BK - 1, LX_TILE - 1);
        else aim_rows(voA, p.lda, p.M - 1 - sm0);
        aim_cols(voB, p.ldb, p.KB - 1 - sk * LX_BK, p.N - 8 - sn0);
    };
    const unsigned dmaA = lds_base + wave * (AT ? 4096u : 8192u), dmaB = lds_base + LX_ELEMS * 2 + wave * 4096u;
    auto stageA = [&](unsigned at, auto jt) __attribute__((always_inline)) {
        constexpr int j = decltype(jt)::value;
        lx_dma<AT ? (j >> 2) * 16384 + (j & 3) * 1024 : j * 1024>(sA, voA[j], dmaA + at);
    };
    auto stageB = [&](unsigned at, auto jt) __attribute__((always_inline)) {
        constexpr int j = decltype(jt)::value;
        lx_dma<(j >> 2) * 16384 + (j & 3) * 1024>(sB, voB[j], dmaB + at);
    };
    // A step has two phases, k 0..31 and k 32..63, and the fragments of a phase are read in the one before.  So a buffer's first half of a [64][256]
    // image is free from phase 0 of its step on, its second half and a [256][64] image from phase 1 on; there they are requested for the step after
    // next, the latter before the former, and have a step or more to arrive.  vmcnt counts in issue order: at the barrier before phase 0,
    // 16 requests are younger than the second halves it reads; before phase 1, WX are younger than what that one reads.
    constexpr int Q0 = AT ? 8 : 4, Q1 = 16 - Q0, WX = AT ? 16 : 8;
    auto request = [&](unsigned at, auto pt, auto qt) __attribute__((always_inline)) {
        constexpr int ph = decltype(pt)::value, q = decltype(qt)::value;
        if constexpr (ph == 0) {
            if constexpr (AT && q < 4) stageA(at, lx_int<q>{});
            else stageB(at, lx_int<AT ? q - 4 : q>{});
        } else if constexpr (AT) {
            if constexpr (q < 4) stageA(at, lx_int<q + 4>{});
            else stageB(at, lx_int<q>{});
        } else {
            if constexpr (q < 8) stageA(at, lx_int<q>{});
            else stageB(at, lx_int<q - 4>{});
        }
    };
    // sA and sB have been moved on by a step.  The last step of an item is aimed at anew (it may be a short one), the first one of the next item
    // too; behind the last step of all the requests repeat it.
    auto advance = [&]() {
        if (++sk + 1 < sk_end) return;
        bool next = false;
        if (sk == sk_end) {
            next = sv + 1 < items;
            sv += next ? 1 : 0;
            --sk;
        }
        aim(next);
    };

    // (read here, because a load that is in flight when the main loop begins would have to be waited for there)
    float sc = 1.f;
    if (p.scale != nullptr) sc = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(p.scale[0])));

    // ---- fragments: where they lie in the first buffer, in bytes; the second is 64 KB further
    unsigned atA[AT ? 8 : 2], atB[8];
    {
        const int rb = 8 * lg + lq, sw = lx_swz(rb);
#pragma unroll
        for (int t = 0; t < (AT ? 8 : 2); ++t)
            atA[t] = lds_base + (AT ? (unsigned)(rb * 512 + (lp & 1) * 8 + ((((wm * 16) | (lp >> 1)) ^ sw ^ (2 * t)) << 4))
                                    : (unsigned)((wm * 128 + lr) * 128 + (((t * 4 + lg) ^ (lr & 7)) << 4)));
#pragma unroll
        for (int t = 0; t < 8; ++t) atB[t] = lds_base + LX_ELEMS * 2 + (unsigned)(rb * 512 + (lp & 1) * 8 + ((((wn * 16) | (lp >> 1)) ^ sw ^ (2 * t)) << 4));
    }
    f32x4 acc[8][8];
    bf16x8 faE[8], fbE[8], faO[8], fbO[8];          // of the two k halves of a step
    auto ldA = [&](bf16x8& f, auto kt, auto tt) __attribute__((always_inline)) {
        constexpr int ks = decltype(kt)::value, t = decltype(tt)::value;
        if constexpr (AT) f = lx_join(lx_lds_tr(atA[t] + ks * 16384), lx_lds_tr(atA[t] + ks * 16384 + 2048));
        else f = lx_lds_row(atA[ks] + t * 2048);
    };
    auto ldB = [&](bf16x8& f, auto kt, auto tt) __attribute__((always_inline)) {
        constexpr int ks = decltype(kt)::value, t = decltype(tt)::value;
        f = lx_join(lx_lds_tr(atB[t] + ks * 16384), lx_lds_tr(atB[t] + ks * 16384 + 2048));
    };
    // A phase: the 64 matrix instructions of a k half, one by one; between them the reads of the next phase's fragments (B's
    // first, which its first eight instructions need), the requests, and in phase 0 behind the reads the step to the other buffer.
    auto phase = [&](const bf16x8 (&fa)[8], const bf16x8 (&fb)[8], bf16x8 (&ga)[8], bf16x8 (&gb)[8], unsigned at, auto pt) __attribute__((always_inline)) {
        constexpr int ph = decltype(pt)::value, Q = ph == 0 ? Q0 : Q1;
        bf16x4 lo;
        lx_static_for<0, 64>([&](auto gt) __attribute__((always_inline)) {
            constexpr int g = decltype(gt)::value, tm = g >> 3, tn = (tm & 1) ? 7 - (g & 7) : g & 7;
            lx_mfma(acc[tm][tn], fb[tn], fa[tm]);
            LX_PIN();
            // three gaps: half a [64][256] fragment each in the first two, a request in the third
            if constexpr (g % 3 < 2 && g < 48) {
                constexpr int i = g / 3;
                if constexpr (i < 8) {
                    if constexpr (g % 3 == 0) lo = lx_lds_tr(atB[i] + (1 - ph) * 16384);
                    else gb[i] = lx_join(lo, lx_lds_tr(atB[i] + (1 - ph) * 16384 + 2048));
                } else if constexpr (AT) {
                    if constexpr (g % 3 == 0) lo = lx_lds_tr(atA[i - 8] + (1 - ph) * 16384);
                    else ga[i - 8] = lx_join(lo, lx_lds_tr(atA[i - 8] + (1 - ph) * 16384 + 2048));
                } else if constexpr (g % 3 == 0) {
                    ldA(ga[i - 8], lx_int<1 - ph>{}, lx_int<i - 8>{});
                }
                LX_PIN();
            }
            if constexpr (g % 3 == 2) {
                // which of the phase's 4, 8 or 12 requests: in every fifth, every second or two of three of these gaps
                constexpr int h = g / 3;
                constexpr int q = Q == 4 ? (h % 5 == 0 && h < 20 ? h / 5 : -1) : Q == 8 ? (h % 2 == 0 && h < 16 ? h / 2 : -1) : (h % 3 < 2 && h < 18 ? h / 3 * 2 + h % 3 : -1);
                if constexpr (q >= 0) { request(at, pt, lx_int<q>{}); LX_PIN(); }
            }
            if constexpr (ph == 0 && g >= 48) {
                if constexpr (g - 48 < (AT ? 8 : 2)) lx_flip(atA[g - 48]);
                if constexpr (g >= 56) lx_flip(atB[g - 56]);
                LX_PIN();
            }
            if constexpr (ph == 1 && g == 62) { sA += dA; sB += dB; LX_PIN(); }
        });
    };
    if (items == 0) return;
    aim(true);
    lx_static_for<0, 2>([&](auto st) __attribute__((always_inline)) {
        constexpr unsigned at = decltype(st)::value * LX_ELEMS * 4u;
        lx_static_for<0, Q0>([&](auto q) __attribute__((always_inline)) { request(at, lx_int<0>{}, q); });
        lx_static_for<0, Q1>([&](auto q) __attribute__((always_inline)) { request(at, lx_int<1>{}, q); });
        sA += dA; sB += dB;
        advance();
    });
    LX_WAIT(16);
    LX_BARRIER();
    lx_static_for<0, 8>([&](auto t) __attribute__((always_inline)) { ldB(fbE[decltype(t)::value], lx_int<0>{}, t); });
    lx_static_for<0, 8>([&](auto t) __attribute__((always_inline)) { ldA(faE[decltype(t)::value], lx_int<0>{}, t); });
    unsigned at = 0;            // the current step's buffer
    bool loose = false;         // at least 32 output stores of this wave are younger than its requests
    for (int v = 0; v < items; ++v) {
        int m0, n0, k0, k1, part;
        locate(v, m0, n0, k0, k1, part);
        const int nk = k1 - k0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int kt = 0; kt < nk; ++kt) {
            if (loose) LX_WAIT(48);
            else LX_WAIT(16);
            LX_LDS_DONE();
            LX_BARRIER();
            LX_PIN();
            phase(faE, fbE, faO, fbO, at, lx_int<0>{});
            if (loose) LX_WAIT(WX + 32);
            else LX_WAIT(WX);
            LX_LDS_DONE();
            LX_BARRIER();
            LX_PIN();
            phase(faO, fbO, faE, fbE, at, lx_int<1>{});
            advance();
            loose = false;
            at ^= LX_ELEMS * 4u;
        }
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");          // the last matrix instructions' results
        LX_PIN();

        const int srow = lane >> 3;
        // accumulators -> rows of 64 columns through the wave's 4 KB of LDS, so that a store covers whole lines
        float* stg = reinterpret_cast<float*>(lsm + 4 * LX_ELEMS) + wave * (16 * 64);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const int tm = u >> 1, h = u & 1;
            const int n = n0 + wn * 128 + h * 64 + (lane & 7) * 8;
#pragma unroll
            for (int tn = 0; tn < 4; ++tn)
                *reinterpret_cast<f32x4*>(stg + lr * 64 + (((tn * 4 + lg) ^ (lr & 7)) << 2)) = acc[tm][4 * h + tn];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = half * 8 + srow;
                f32x4 lo = *reinterpret_cast<const f32x4*>(stg + r * 64 + (((2 * (lane & 7)) ^ srow) << 2));
                f32x4 hi = *reinterpret_cast<const f32x4*>(stg + r * 64 + (((2 * (lane & 7) + 1) ^ srow) << 2));
                const int m = m0 + wm * 128 + tm * 16 + r;
                if (m < p.M && n < p.N) {
                    if (part >= 0) {
                        float* q = p.slab + (size_t)((2 * team + part) * p.width + member) * 65536 + (m - m0) * 256 + (n - n0);
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
        loose = m0 + LX_TILE <= p.M && n0 + LX_TILE <= p.N;       // a full tile: 32 stores at least
    }
    LX_WAIT(0);         // nothing may arrive in LDS after the workgroup has ended
}

// ---------------------------------------------------------------------------------------------------- rows
struct LxRowParams {
    const bf16_t* x; long long ldx;
    const bf16_t* w; long long ldw;
    const void* bias; int bias_type;
    const long long* target; long long ignore_index;
    const float2* stats; const float* zsum; int stat_cols;
    unsigned* ticket; float* scale; float* loss; int mean;      // loss not null: the last row to finish adds the rows up (see lx_loss_kernel)
    bf16_t* P; long long ldp;          // P on entry (lx_pack_p), bf16 dz on exit; null: loss alone
    float* rows;
    bf16_t* xs;                        // [rows_n][D]: x, zero where a row is not counted; null: no dW
    float* delta;                      // what the target's dz lost to bf16, per row (0 where it is ignored); null: no db
    int V, D, rows_n, pad_rows;         // pad_rows rows of zeros behind the last (lx_grad_kernel reads steps of 64 of them)
    float smoothing;
    float a, u, hit;                   // dz = a p - u - hit [the target], see lx_factor
    double unit;                       // what dz is multiplied by
};

template <int WAVES>
static __device__ __forceinline__ float lx_block_max(float v, float* sh) {
    v = wave_max(v);
    if (WAVES == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v = fmaxf(v, sh[w]);
    return v;
}
template <int WAVES>
static __device__ __forceinline__ float lx_block_sum(float v, float* sh) {
    v = wave_sum(v);
    if (WAVES == 1) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += sh[w];
    return v;
}

// exp(m - mx) * 2^-s2 for a piece's maximum m <= the row's mx; infinite ones, and the lowest logits of a type, are equal to themselves
static __device__ __forceinline__ float lx_below(float m, float mx, float s2 = 0.f) {
    return __builtin_amdgcn_exp2f((m == mx ? 0.f : (m - mx) * 1.44269504088896340736f) - s2);
}
// 8 columns of P -> dz; f holds the 2^64 of lx_unpack_p
static __device__ __forceinline__ u32x4 lx_dz8(const u32x4 r, float f, float u, float hit, int n, int t, int V, bool valid) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = __builtin_fmaf(lx_unpack_p(r[k] & 0xffffu), f, -u);
        v[2 * k + 1] = __builtin_fmaf(lx_unpack_p(r[k] >> 16), f, -u);
    }
    if ((t & ~7) == n) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (n + k == t) v[k] -= hit;
    }
    if (!valid) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __builtin_nanf("");
    }
    if (n + 8 > V) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (n + k >= V) v[k] = 0.f;
    }
    return (u32x4){pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])};
}

// scale of the gradients and loss from the sum of the rows' losses and the count of the counted rows
static __device__ __forceinline__ void lx_finish(double s, long long count, int mean, double unit, float* scale, float* loss) {
    if (scale != nullptr) *scale = (float)(count == 0 ? 0.0 : mean ? unit / (double)count : unit);
    if (loss != nullptr) *loss = (float)(count == 0 ? 0.0 : mean ? s / (double)count : s);
}
// A row's loss is known: it is stored, and where p.loss is set the wave that is the last of all rows' first waves adds them up, lane by lane, then
// the lanes.  That saves a call of few rows a launch (see LX_FUSED_ROWS).
static __device__ __forceinline__ void lx_row_done(const LxRowParams& p, int row, int tid, float l) {
    if (tid >= 64) return;
    if (p.loss == nullptr) {
        if (tid == 0) p.rows[row] = l;
        return;
    }
    unsigned n = 0;
    if (tid == 0) {
        __hip_atomic_store(p.rows + row, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        n = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((int)__builtin_amdgcn_readfirstlane(n) != p.rows_n - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    double s = 0.0;
    int count = 0;
    for (int i = tid; i < p.rows_n; i += 64) {
        s += (double)__hip_atomic_load(p.rows + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        count += p.target[i] != p.ignore_index;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); count += __shfl_xor(count, o, 64); }
    if (tid == 0) lx_finish(s, count, p.mean, p.unit, p.scale, p.loss);
}

// WAVES waves per row: one workgroup, or for short rows one wave of a workgroup of four.  Bound by memory: 4 bytes per logit where the gradient
// is wanted, nothing to speak of where it is not.
#define LX_AHEAD 4          // chunks of 8 columns a thread has in flight
template <int WAVES, bool STREAM>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void lx_row_kernel(const LxRowParams p) {
    constexpr int NT = WAVES * 64;
    __shared__ float sh[WAVES];
    const int tid = WAVES == 1 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
    const int row = WAVES == 1 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
    if (row >= p.rows_n + p.pad_rows) return;
    const bool pad = row >= p.rows_n;
    const long long t64 = pad ? 0 : p.target[row];
    bf16_t* P = p.P != nullptr ? p.P + (size_t)row * p.ldp : nullptr;
    const int chunks = (int)(p.ldp / 8);
    if (pad || t64 == p.ignore_index) {
        if (P != nullptr)
            for (int c = tid; c < chunks; c += NT) __builtin_nontemporal_store((u32x4){0u, 0u, 0u, 0u}, reinterpret_cast<u32x4*>(P) + c);
        if (!pad) {
            if (p.xs != nullptr)
                for (int c = tid; c < p.D / 8; c += NT) reinterpret_cast<u32x4*>(p.xs + (size_t)row * p.D)[c] = (u32x4){0u, 0u, 0u, 0u};
            if (p.delta != nullptr && tid == 0) p.delta[row] = 0.f;
            lx_row_done(p, row, tid, 0.f);
        }
        return;
    }
    // a label outside [0, V) never becomes an address: the row's loss and gradient are NaN
    const bool valid = t64 >= 0 && t64 < (long long)p.V;
    const int t = valid ? (int)t64 : 0;
    const float2* st = p.stats + (size_t)row * p.stat_cols;
    const int entries = (p.V + LX_STAT - 1) / LX_STAT;          // what lies behind them up to stat_cols need not have been written
    // the target's logit
    const bf16_t* xr = p.x + (size_t)row * p.ldx;
    const bf16_t* wr = p.w + (size_t)t * p.ldw;
    float dot = 0.f;
    for (int c = tid; c < p.D / 8; c += NT) {
        float a[8], b[8];
        load8(xr + c * 8, a);
        load8(wr + c * 8, b);
        if (p.xs != nullptr) reinterpret_cast<u32x4*>(p.xs + (size_t)row * p.D)[c] = reinterpret_cast<const u32x4*>(xr)[c];
#pragma unroll
        for (int k = 0; k < 8; ++k) dot = __builtin_fmaf(a[k], b[k], dot);
    }
    float mx = -INFINITY;
#pragma unroll 4
    for (int c = tid; c < entries; c += NT) mx = fmaxf(mx, st[c].x);
    mx = lx_block_max<WAVES>(mx, sh);
    float s = 0.f, zs = 0.f;
#pragma unroll 4
    for (int c = tid; c < entries; c += NT) {
        const float2 v = st[c];
        s += v.y * lx_below(v.x, mx);           // an all -inf entry has s = 0, or NaN where a logit was NaN
        if (p.smoothing > 0.f) zs += p.zsum[(size_t)row * p.stat_cols + c];
    }
    s = lx_block_sum<WAVES>(s, sh);
    dot = lx_block_sum<WAVES>(dot, sh);
    if (p.smoothing > 0.f) zs = lx_block_sum<WAVES>(zs, sh);
    if (p.bias != nullptr) dot += p.bias_type == 1 ? bf2f(reinterpret_cast<const bf16_t*>(p.bias)[t]) : reinterpret_cast<const float*>(p.bias)[t];
    // lse - z as (max - z) + log s: lse as one number would be rounded to its own size, which is 30 times the loss of a certain row.  Neither loss
    // is negative; the target's logit, a sum of its own, may be an ulp above the maximum.
    const float s2 = log2f(s);
    auto above = [&](float z) { const float l = __builtin_fmaf(s2, 0.69314718055994530942f, mx - z); return l < 0.f ? 0.f : l; };
    float l = above(dot);
    if (p.smoothing > 0.f) l = (1.f - p.smoothing) * l + p.smoothing * above(zs / (float)p.V);
    lx_row_done(p, row, tid, valid ? l : __builtin_nanf(""));
    if (P == nullptr) return;
    const float u = p.u, hit = p.hit, a = p.a * 0x1p+64f;
    u32x4* q = reinterpret_cast<u32x4*>(P);
    for (int c0 = tid; c0 < chunks; c0 += LX_AHEAD * NT) {
        u32x4 r[LX_AHEAD];
        float m[LX_AHEAD];
#pragma unroll
        for (int j = 0; j < LX_AHEAD; ++j) {
            const int c = c0 + j * NT < chunks ? c0 + j * NT : c0;
            r[j] = STREAM ? __builtin_nontemporal_load(q + c) : q[c];
            m[j] = st[c >> 3].x;
        }
#pragma unroll
        for (int j = 0; j < LX_AHEAD; ++j) {
            const int c = c0 + j * NT;
            if (c < chunks) {
                const float f = lx_below(m[j], mx, s2) * a;
                const u32x4 o = lx_dz8(r[j], f, u, hit, c * 8, t, p.V, valid);
                if (p.delta != nullptr && c == (t >> 3)) {
                    const int shift = (t & 1) * 16;
                    unsigned in = 0, out = 0;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k == ((t & 7) >> 1)) { in = r[j][k]; out = o[k]; }
                    const float v = __builtin_fmaf(lx_unpack_p((in >> shift) & 0xffffu), f, -u) - hit;
                    p.delta[row] = valid ? v - bf2f((unsigned short)(out >> shift)) : 0.f;
                }
                if (STREAM) __builtin_nontemporal_store(o, q + c);
                else q[c] = o;
            }
        }
    }
}

// Count of the counted rows, the scale of the gradients (unit / count, or unit for a sum; 0 without a counted row) and the loss.  Workgroup b sums
// a stretch of the rows into part[b]; the last one to finish adds the parts up, one to a lane (the kernel that made the logits has zeroed the ticket).
#define LX_LOSS_WGS 64          // at most a wave's lanes
struct LxLossPart { double sum; long long count; };
__global__ __launch_bounds__(256) void lx_loss_kernel(const long long* __restrict__ target, long long ignore_index, const float* __restrict__ rows, int T, int per,
                                                      int mean, double unit, LxLossPart* part, unsigned* ticket, float* __restrict__ scale, float* __restrict__ loss) {
    __shared__ double sh[4];
    __shared__ int shc[4];
    const int i1 = (int)((blockIdx.x + 1ll) * per < T ? (blockIdx.x + 1ll) * per : T);
    double s = 0.0;
    int n = 0;
    for (int i0 = blockIdx.x * per + (int)threadIdx.x; i0 < i1; i0 += 8 * 256) {
        long long t[8];
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * 256 < i1 ? i0 + j * 256 : i0;
            t[j] = target[i];
            r[j] = rows != nullptr ? rows[i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j * 256 < i1) {
                n += t[j] != ignore_index;
                s += (double)r[j];
            }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); n += __shfl_xor(n, o, 64); }
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6] = s; shc[threadIdx.x >> 6] = n; }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    s = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    long long count = (long long)shc[0] + shc[1] + shc[2] + shc[3];
    if (gridDim.x > 1) {
        unsigned nth = 0;
        if (threadIdx.x == 0) {
            __hip_atomic_store(&part[blockIdx.x].sum, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(&part[blockIdx.x].count, count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            nth = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (__builtin_amdgcn_readfirstlane(nth) != gridDim.x - 1) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        const bool mine = threadIdx.x < gridDim.x;
        s = mine ? __hip_atomic_load(&part[threadIdx.x].sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
        count = mine ? __hip_atomic_load(&part[threadIdx.x].count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); count += __shfl_xor(count, o, 64); }
    }
    if (threadIdx.x == 0) lx_finish(s, count, mean, unit, scale, loss);
}

// The same products for outputs too small to fill the chip with 256 x 256 tiles, which also cost a call 8 to 10 us of pipeline fill and epilogue
// however short it is: one tile of (16 FM WM) x (64 WN) and one range of steps per 256-thread workgroup, several workgroups on a compute unit
// in place of a deep pipeline within one.  FM = 4, waves 2 x 2: 128 x 128 tiles, 64 KB of LDS; FM = 1, waves 4 x 1: 64 x 64, 32 KB.
// LX_OUT with p.splits > 1: the fp32 sums of range s go to slab[s][M][N].
template <int FM, int WM, int WN> struct LxSmall { static constexpr int lds = 2 * (FM * 16 * WM + 64 * WN) * LX_BK; };       // elements
template <int LAY, int EPI, int FM, int WM, int WN>
static __device__ __forceinline__ void lx_small_body(const LxGemmParams& p, bf16_t* sm, int block, int blocks) {
    constexpr bool AT = LAY == LX_TN, BT = LAY != LX_NT;
    constexpr int TM = FM * 16 * WM, TN = 64 * WN;              // the tile
    constexpr int PA = TM / 32, PB = TN / 32;                   // 1 KB pieces of an operand's step per wave
    constexpr int EA = TM * LX_BK, EB = TN * LX_BK;             // elements of a buffer
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int lr = lane & 15, lg = lane >> 4, lq = lr >> 2, lp = lr & 3;
    const unsigned lds_base = __builtin_amdgcn_readfirstlane(lds_addr(sm));

    const int id = xcd_remap(block, blocks);
    const int tiles = p.tiles_m * p.tiles_n;
    const int split = __builtin_amdgcn_readfirstlane(id / tiles);
    const int tile = id - split * tiles;
    const int tm_ = tile / p.tiles_n;
    const int m0 = __builtin_amdgcn_readfirstlane(tm_ * TM), n0 = __builtin_amdgcn_readfirstlane((tile - tm_ * p.tiles_n) * TN);
    int k0, k1;
    lx_range(split, p.steps, p.splits, k0, k1);
    k0 = __builtin_amdgcn_readfirstlane(k0);
    k1 = __builtin_amdgcn_readfirstlane(k1);

    // K-contiguous image [T][64]: a piece is 8 rows, position lane % 8 receives chunk (lane % 8) ^ (row & 7).  K-strided image [64][T]: a piece
    // is 512 / T rows; chunks are XOR-swizzled by the row so that the transposing read's 8 rows of a half wave meet different banks
    // (rows r and r + 4 have the same swizzle)
    auto swz = [](int r, int T) { return T == 128 ? lx_swz(r) : (((r >> 1) & 1) << 1) | (((r >> 3) & 1) << 2); };
    const bf16_t* gA = p.A + (AT ? (size_t)m0 : (size_t)m0 * p.lda);
    const bf16_t* gB = p.B + (BT ? (size_t)n0 : (size_t)n0 * p.ldb);
    unsigned voA[PA], voB[PB];
    int kA[PA], kB[PB];         // the lane's place in a step's contraction, per piece
#pragma unroll
    for (int j = 0; j < PA; ++j) {
        if (AT) {
            constexpr int CH = TM / 8;          // chunks of a row
            const int r = (wave * PA + j) * (64 / CH) + lane / CH;
            kA[j] = r;
            voA[j] = (unsigned)((r * p.lda + ((lane % CH) ^ swz(r, TM)) * 8) * 2);         // A's rows are padded to a multiple of 256
        } else {
            const int r = (wave * PA + j) * 8 + (lane >> 3), most = p.M - 1 - m0;
            kA[j] = ((lane & 7) ^ (r & 7)) * 8;
            voA[j] = (unsigned)(((r < most ? r : most) * p.lda + kA[j]) * 2);
        }
    }
#pragma unroll
    for (int j = 0; j < PB; ++j) {
        if (BT) {
            constexpr int CH = TN / 8;
            const int r = (wave * PB + j) * (64 / CH) + lane / CH, c = ((lane % CH) ^ swz(r, TN)) * 8;
            kB[j] = r;
            voB[j] = (unsigned)((r * p.ldb + (n0 + c < p.N ? c : p.N - 8 - n0)) * 2);
        } else {
            const int r = (wave * PB + j) * 8 + (lane >> 3), most = p.N - 1 - n0;
            kB[j] = ((lane & 7) ^ (r & 7)) * 8;
            voB[j] = (unsigned)(((r < most ? r : most) * p.ldb + kB[j]) * 2);
        }
    }
    const void* zrow = (const char*)lx_zero_row + (lane & 31) * 16;
    auto stage = [&](int k, int par) {
        const bf16_t* a = gA + (AT ? (size_t)k * LX_BK * p.lda : (size_t)k * LX_BK);
        const bf16_t* b = gB + (BT ? (size_t)k * LX_BK * p.ldb : (size_t)k * LX_BK);
        const unsigned dA = lds_base + (unsigned)(par * (EA + EB) * 2) + wave * PA * 1024, dB = lds_base + (unsigned)((par * (EA + EB) + EA) * 2) + wave * PB * 1024;
        if ((k + 1) * LX_BK <= p.KA) {
#pragma unroll
            for (int j = 0; j < PA; ++j) glds16(a, voA[j], dA + j * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < PA; ++j) glds16_v(k * LX_BK + kA[j] < p.KA ? (const void*)((const char*)a + voA[j]) : zrow, dA + j * 1024);
        }
        if ((k + 1) * LX_BK <= p.KB) {
#pragma unroll
            for (int j = 0; j < PB; ++j) glds16(b, voB[j], dB + j * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < PB; ++j) glds16_v(k * LX_BK + kB[j] < p.KB ? (const void*)((const char*)b + voB[j]) : zrow, dB + j * 1024);
        }
    };
    f32x4 acc[FM][4];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    stage(k0, 0);
    for (int k = k0; k < k1; ++k) {
        const int par = (k - k0) & 1;
        LX_WAIT(0);             // this step's operands have landed, the other buffer has been read
        LX_BARRIER();
        if (k + 1 < k1) stage(k + 1, par ^ 1);
        const bf16_t* cA = sm + par * (EA + EB);
        const bf16_t* cB = cA + EA;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8 fa[FM], fb[4];
            const int r = ks * 32 + 8 * lg + lq, ch = ks * 4 + lg;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (BT) {
                    const bf16_t* q = cB + r * TN + ((((wn * 64 + t * 16) >> 3) + (lp >> 1)) ^ swz(r, TN)) * 8 + (lp & 1) * 4;
                    fb[t] = lx_tr(q, q + 4 * TN);
                } else {
                    const int row = wn * 64 + t * 16 + lr;
                    fb[t] = *reinterpret_cast<const bf16x8*>(cB + row * LX_BK + ((ch ^ (row & 7)) << 3));
                }
            }
#pragma unroll
            for (int t = 0; t < FM; ++t) {
                if (AT) {
                    const bf16_t* q = cA + r * TM + ((((wm * FM * 16 + t * 16) >> 3) + (lp >> 1)) ^ swz(r, TM)) * 8 + (lp & 1) * 4;
                    fa[t] = lx_tr(q, q + 4 * TM);
                } else {
                    const int row = wm * FM * 16 + t * 16 + lr;
                    fa[t] = *reinterpret_cast<const bf16x8*>(cA + row * LX_BK + ((ch ^ (row & 7)) << 3));
                }
            }
#pragma unroll
            for (int tm = 0; tm < FM; ++tm)
#pragma unroll
                for (int tn = 0; tn < 4; ++tn)
                    acc[tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[tn], fa[tm], acc[tm][tn], 0, 0, 0);
        }
    }
    LX_WAIT(0);
    LX_BARRIER();           // every wave has read its operands: their LDS takes the epilogue's rows
    if constexpr (EPI == LX_OUT) {
        const float sc = p.scale != nullptr ? p.scale[0] : 1.0f;
        bf16_t* stg = sm + wave * (16 * 64);
        const int srow = lane >> 3;
#pragma unroll
        for (int tm = 0; tm < FM; ++tm) {
            const int m = m0 + (wm * FM + tm) * 16 + lr;
#pragma unroll
            for (int tn = 0; tn < 4; ++tn) {
                const int n = n0 + wn * 64 + tn * 16 + 4 * lg;
                const bool in = m < p.M && n < p.N;
                f32x4 v = acc[tm][tn];
                if (p.splits > 1) {
                    if (in) *reinterpret_cast<f32x4*>(p.slab + ((size_t)split * p.M + m) * p.N + n) = v;
                    continue;
                }
                v *= sc;
                if (p.add != nullptr && in) v += *reinterpret_cast<const f32x4*>(p.add + (size_t)m * p.N + n);
                if (p.out_f32) {
                    if (in) *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n) = v;
                } else {            // bf16: through the wave's 2 KB of LDS, so that a store covers whole lines
                    uint2 o;
                    o.x = pack2bf(v[0], v[1]);
                    o.y = pack2bf(v[2], v[3]);
                    *reinterpret_cast<uint2*>(stg + lr * 64 + (((tn * 2 + (lg >> 1)) ^ (lr & 7)) << 3) + (lg & 1) * 4) = o;
                }
            }
            if (p.splits == 1 && !p.out_f32) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = half * 8 + srow;
                    const u32x4 o = *reinterpret_cast<const u32x4*>(stg + r * 64 + (((lane & 7) ^ srow) << 3));
                    const int mr = m0 + (wm * FM + tm) * 16 + r, n = n0 + wn * 64 + (lane & 7) * 8;
                    if (mr < p.M && n < p.N) __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(reinterpret_cast<bf16_t*>(p.out) + (size_t)mr * p.ldo + n));
                }
            }
        }
    } else {
        lx_loss_epilogue<FM, true>(p, acc, m0 + wm * FM * 16, n0 + wn * 64, sm + wave * (16 * 64));
    }
}
template <int LAY, int EPI, int FM, int WM, int WN>
__global__ __launch_bounds__(256) void lx_small_kernel(const LxGemmParams p) {
    __shared__ __attribute__((aligned(1024))) bf16_t sm[LxSmall<FM, WM, WN>::lds];
    if (EPI != LX_OUT && blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0u;
    lx_small_body<LAY, EPI, FM, WM, WN>(p, sm, blockIdx.x, gridDim.x);
}
// Rows first, first + STEP, ... < end of dz, 8 columns, for db, with what the targets' dz lost to bf16: without that the target's own probability
// would be missing from every hit while it is small.  Eight rows are in flight; the targets, which are rare, are looked at behind them.
template <int STEP>
static __device__ __forceinline__ void lx_colsum_rows(float (&acc)[8], const bf16_t* dz, long long ldp, long long col, const long long* target, const float* delta,
                                                      int first, int end) {
    for (int r0 = first; r0 < end; r0 += 8 * STEP) {
        float v[8][8], d[8];
        int t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = r0 + j * STEP < end ? r0 + j * STEP : r0;
            load8(dz + (size_t)r * ldp + col, v[j]);
            const long long c = target[r] - col;
            t[j] = c >= 0 && c < 8 && r0 + j * STEP < end ? (int)c : 8;
            d[j] = delta[r];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = r0 + j * STEP < end;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += in ? v[j][k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (t[j] < 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] += t[j] == k ? d[j] : 0.f;
            }
    }
}
// db of up to 1024 rows: a workgroup sums 128 columns, 16 rows at a time
struct LxColsum { const bf16_t* dz; long long ldp; int T, V; const float* scale; void* db; int db_f32; const long long* target; const float* delta; };
static __device__ __forceinline__ void lx_colsum_few(const LxColsum& c, float (*sh)[128], int block) {
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
    const long long col = (long long)block * 128 + lane * 8;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    lx_colsum_rows<16>(acc, c.dz, c.ldp, col, c.target, c.delta, group, c.T);
#pragma unroll
    for (int k = 0; k < 8; ++k) sh[group][lane * 8 + k] = acc[k];
    __syncthreads();
    const int n = block * 128 + (int)threadIdx.x;
    if (threadIdx.x >= 128 || n >= c.V) return;
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < 16; ++g) s += sh[g][threadIdx.x];
    s *= c.scale[0];
    if (c.db_f32) reinterpret_cast<float*>(c.db)[n] = s;
    else reinterpret_cast<bf16_t*>(c.db)[n] = f2bf(s);
}
__global__ __launch_bounds__(256) void lx_colsum_few_kernel(const LxColsum c) {
    __shared__ float sh[16][128];
    lx_colsum_few(c, sh, blockIdx.x);
}
// dx, dW and db of few rows in one launch: they need dz alone.  The first bx workgroups are those of dx, the next bw those of dW.
template <int FM, int WM, int WN>
__global__ __launch_bounds__(256) void lx_small_grads_kernel(const LxGemmParams dx, const LxGemmParams dw, const LxColsum db, int bx, int bw) {
    __shared__ __attribute__((aligned(1024))) bf16_t sm[LxSmall<FM, WM, WN>::lds];
    const int block = blockIdx.x;
    if (block < bx) lx_small_body<LX_NN, LX_OUT, FM, WM, WN>(dx, sm, block, bx);
    else if (block < bx + bw) lx_small_body<LX_TN, LX_OUT, FM, WM, WN>(dw, sm, block - bx, bw);
    else lx_colsum_few(db, reinterpret_cast<float (*)[128]>(sm), block - bx - bw);
}

// out = scale * sum over the splits of slab[s] (+ add), fixed order; N % 4 == 0
__global__ __launch_bounds__(256) void lx_reduce_kernel(const LxGemmParams p) {
    const size_t total = (size_t)p.M * p.N / 4, stride = (size_t)p.M * p.N;
    const float sc = p.scale != nullptr ? p.scale[0] : 1.0f;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const float* q = p.slab + i * 4;
        f32x4 s = *reinterpret_cast<const f32x4*>(q);
#pragma unroll 4
        for (int k = 1; k < p.splits; ++k) s += *reinterpret_cast<const f32x4*>(q + k * stride);
        s *= sc;
        if (p.add != nullptr) s += *reinterpret_cast<const f32x4*>(p.add + i * 4);
        const size_t m = i * 4 / p.N, n = i * 4 - m * p.N;
        if (p.out_f32) {
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + m * p.ldo + n) = s;
        } else {
            uint2 o;
            o.x = pack2bf(s[0], s[1]);
            o.y = pack2bf(s[2], s[3]);
            *reinterpret_cast<uint2*>(reinterpret_cast<bf16_t*>(p.out) + m * p.ldo + n) = o;
        }
    }
}

// the tiles of the rest: out = scale * sum of their parts (+ add), in the order of the contraction; 8 rows of a tile per workgroup
__global__ __launch_bounds__(256) void lx_join_kernel(const LxGemmParams p) {
    const int r = (int)(blockIdx.x >> 5) / p.width, member = (int)(blockIdx.x >> 5) - r * p.width;
    const int blk = (p.whole + r) / p.tiles_m;
    const int m0 = (p.whole + r - blk * p.tiles_m) * LX_TILE, n0 = (blk * p.width + member) * LX_TILE;
    const int row = (int)(blockIdx.x & 31) * 8 + (int)(threadIdx.x >> 5), col = (int)(threadIdx.x & 31) * 8;
    const int m = m0 + row, n = n0 + col;
    if (m >= p.M || n >= p.N) return;
    // the ranges that meet this row's steps, from the one its first step lies in to the one of its last; the tile is the second part of
    // the first of them if that range began in the row before
    const int s0 = r * p.steps, total = p.rest * p.steps;
    const int q = total / p.ranges, more = total - q * p.ranges;
    auto owner = [&](int step) { return step < more * (q + 1) ? step / (q + 1) : more + (step - more * (q + 1)) / q; };
    const int first = owner(s0), last = owner(s0 + p.steps - 1);
    int from, to;
    lx_range(first, total, p.ranges, from, to);
    const float* at = p.slab + (size_t)member * 65536 + row * 256 + col;
    const size_t tile = (size_t)p.width * 65536;
    const float* w0 = at + (2 * first + (from < s0 ? 1 : 0)) * tile;
    f32x4 lo = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(w0)), hi = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(w0 + 4));
#pragma unroll 4
    for (int g = first + 1; g <= last; ++g) {
        const float* w = at + 2 * g * tile;
        lo += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(w));
        hi += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(w + 4));
    }
    const float sc = p.scale != nullptr ? p.scale[0] : 1.0f;
    lo *= sc;
    hi *= sc;
    if (p.add != nullptr) {
        const float* w = p.add + (size_t)m * p.N + n;
        lo += *reinterpret_cast<const f32x4*>(w);
        hi += *reinterpret_cast<const f32x4*>(w + 4);
    }
    if (p.out_f32) {
        float* w = reinterpret_cast<float*>(p.out) + (size_t)m * p.ldo + n;
        *reinterpret_cast<f32x4*>(w) = lo;
        *reinterpret_cast<f32x4*>(w + 4) = hi;
    } else {
        const u32x4 o = {pack2bf(lo[0], lo[1]), pack2bf(lo[2], lo[3]), pack2bf(hi[0], hi[1]), pack2bf(hi[2], hi[3])};
        *reinterpret_cast<u32x4*>(reinterpret_cast<bf16_t*>(p.out) + (size_t)m * p.ldo + n) = o;
    }
}

// db: column sums of dz.  A block sums 512 columns over a range of rows into partial[range][ldp]; the second kernel adds the ranges in order.
__global__ __launch_bounds__(256) void lx_colsum_kernel(const bf16_t* __restrict__ dz, long long ldp, int T, int rows_per_range, float* __restrict__ partial,
                                                        const long long* __restrict__ target, const float* __restrict__ delta) {
    __shared__ float sh[4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long col = (long long)blockIdx.x * 512 + lane * 8;
    const int r0 = blockIdx.y * rows_per_range, r1 = r0 + rows_per_range < T ? r0 + rows_per_range : T;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col < ldp) lx_colsum_rows<4>(acc, dz, ldp, col, target, delta, r0 + wave, r1);
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
#pragma unroll 16
    for (int r = 0; r < ranges; ++r) s += partial[(size_t)r * ldp + n];
    if (db == nullptr) { sum[n] = s; return; }
    s *= scale[0];
    if (db_f32) reinterpret_cast<float*>(db)[n] = s;
    else reinterpret_cast<bf16_t*>(db)[n] = f2bf(s);
}

// ---------------------------------------------------------------------------------------------------- host
// the rows' kernel adds the losses up itself for up to 512 rows, unless it rewrites more than 1 MB of P (each row's ticket waits for the
// stores before it to reach memory)
#define LX_FUSED_ROWS 512
#define LX_FUSED_BYTES ((size_t)1 << 20)
#define LX_CACHED ((size_t)640 << 20)

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
// ranges of rows that the column sums are cut into: more where there are few columns (25088 x 1000: 64 of them 23 + 4 us, 128 15 + 5)
static int lx_ranges(long long ldp) { return ldp <= 2048 ? 128 : 64; }
// dz / unit = a p - u - hit [the target].  Of the 128 bf16 numbers from 1 up, hit is the one for which u = hit e / (V (1 - e)) is nearest to a bf16 number
// too: half of all V within 1.4e-5, nine in ten within 5e-5 (1 - e and e/V themselves are off by up to 2^-8; 0.9 by 0.17 %, 0.1 / 21843 by 0.25 %).
// u stays inside the rounded factor: taken off the sums instead (as e/V times the sums of x and of W's rows), the factor would be rounded to
// 2^-8 of p also where p - e/V nearly cancels.
struct LxFactor { float a, u, hit; double unit; };
static LxFactor lx_factor(float smoothing, int V) {
    const double e = smoothing;
    if (e <= 0.0) return {1.f, 0.f, 1.f, 1.0};
    if (e >= 1.0) return {(float)V, 1.f, 0.f, 1.0 / V};
    const double r = e / (V * (1.0 - e));
    int exponent, best = 128;
    const double f = frexp(r, &exponent);
    double least = 1.0;
    for (int m = 128; m < 256; ++m) {
        const double t = f * m < 128.0 ? 2.0 * f * m : f * m, off = fabs(rint(t) - t) / t;
        if (off < least) { least = off; best = m; }
    }
    const double hit = best / 128.0, unit = (1.0 - e) / hit;
    return {(float)(1.0 / unit), (float)(r * hit), (float)hit, unit};
}
static size_t lx_up(size_t n) { return (n + 255) & ~(size_t)255; }

// How the tiles of dx and dW are dealt.  `width` column tiles side by side form a row, worked on by a team of as many workgroups in step, so
// that what they share of the other operand is fetched once; there are tiles_m * tiles_n / width rows.  Of `teams` teams, team t takes the
// whole rows t, t + teams, ... below `whole`; the `rest` rows behind them are one sequence of rest * steps steps, cut into `ranges`
// equal ranges (at most two parts of rows each) whose fp32 sums go to slab[2 range + part][width][256][256] and are joined in order.
// The small kernel (kind LX_SMALL64, LX_SMALL128): `splits` ranges of steps per tile, slab[splits][M][N].
enum { LX_BIG = 0, LX_SMALL128 = 1, LX_SMALL64 = 2 };
struct LxDeal { int kind, width, teams, whole, rest, ranges, splits; size_t slab; double us; };
// how the rows are cut and where everything lies in the workspace
struct LxPlan {
    long long ldp, stat_cols;
    int block, blocks;              // rows per block, blocks
    LxDeal dx[2], dw[2];            // of a block, of the last one
    size_t scale, stats, zsum, P, xs, acc, slab, colpart, colsum, delta, total;
};
// The kernel and its cut that a model of the time finds fastest, in microseconds on 256 compute units, from 28 shapes between 1 x 1000 x 192 and
// 512 x 100003 x 1024 measured with each of the three kernels (time of x W^T / dz W / dz^T x in us, large : 128 : 64):
//   1 x 1000 x 192       10 23 12 : 7 8 7 : 4 7 4             512 x 8192 x 768     22 33 22 : 15 21 14 : 19 19 16
//   1024 x 1024 x 1024   30 31 33 : 16 17 16 : 11 12 10       8192 x 8192 x 768    89 119 120 : 157 114 99 : 244 154 156
//   512 x 21843 x 768    25 43 37 : 31 36 34 : 47 33 36       512 x 100003 x 1024  117 118 142 : 158 156 189 : 245 262 260
// It is off by up to 18 %; where that makes it take the slower one (512 x 100003 x 1024: 308 us for both gradients, the large kernel 260), another
// term for the memory cost as much elsewhere (512 x 50000 x 2048: 247, 264).
// Large: whole rows alone take ceil(rows / teams) rounds; cutting what does not fill a round into ranges fills it at the price of parts written
// and read, 0.13 us for one of 256 x 256 (512 KB at 4 TB/s).
#define LX_US_STEP 1.25
#define LX_US_PART 0.13
static LxDeal lx_deal_big(int M, int N, int steps, int cus, bool loss) {
    LxDeal d = {};
    d.kind = LX_BIG;
    d.splits = 1;
    const int tiles_m = (M + LX_TILE - 1) / LX_TILE, tiles_n = (N + LX_TILE - 1) / LX_TILE;
    if (loss) {             // the logits: whole tiles, dealt one by one
        const long long tiles = (long long)tiles_m * tiles_n;
        d.teams = tiles < cus ? (int)tiles : cus;
        d.us = 4.0 + (double)((tiles + cus - 1) / cus) * (steps * LX_US_STEP + 7.5);
        return d;
    }
    const double tile = 6.0;
    for (d.width = tiles_n < 8 ? tiles_n : 8; tiles_n % d.width; --d.width) {}
    const int rows = tiles_m * (tiles_n / d.width);
    const int most = cus / d.width > 0 ? cus / d.width : 1;
    const int rounds = rows / most, rest = rows - rounds * most;
    d.teams = rows < most ? rows : most;
    d.whole = rows;
    d.us = 4.0 + (rounds + (rest > 0)) * (steps * LX_US_STEP + tile);
    if (rest == 0 || (long long)rest * steps > 0x7fffffff) return d;
    const double part = LX_US_PART * (M < LX_TILE ? M : LX_TILE) / LX_TILE * d.width;
    for (int k = 1; k <= 16; ++k) {
        const int ranges = most * k / 16;
        if (ranges <= rest || (long long)rest * steps / ranges < 2) continue;
        const double us = 8.0 + rounds * (steps * LX_US_STEP + tile) + (double)rest * steps / ranges * LX_US_STEP + 2 * tile + part * (ranges + rest);
        if (us < 0.98 * d.us) { d.us = us; d.teams = rounds > 0 ? most : ranges; d.whole = rounds * most; d.rest = rest; d.ranges = ranges; }
    }
    d.slab = (size_t)2 * d.ranges * d.width * 65536;
    return d;
}
// Small: a step of a workgroup alone on its compute unit takes `alone`, workgroups that share one get a step in `shared` each in turn.
static LxDeal lx_deal_small(int M, int N, int steps, int cus, bool loss, int kind) {
    const bool s64 = kind == LX_SMALL64;
    const int tile = s64 ? 64 : 128;
    const double alone = s64 ? 0.30 : 0.62, shared = s64 ? 0.31 : loss ? 0.52 : 0.45, base = s64 ? 3.2 : 4.0, last = loss ? (s64 ? 0.6 : 2.5) : (s64 ? 0.3 : 0.8);
    const long long tiles = (long long)((M + tile - 1) / tile) * ((N + tile - 1) / tile);
    LxDeal best = {};
    best.us = 1e30;
    for (int splits = 1; splits <= (loss ? 1 : 256); splits += splits < 8 ? 1 : splits / 4) {
        if (splits > 1 && steps / splits < 4) break;
        const long long wgs = tiles * splits, per = (wgs + cus - 1) / cus;
        if (wgs > 0x7fffffff) break;
        double us = base + ((steps + splits - 1) / splits) * (per > 1 ? shared * per : alone) + last * per;
        if (splits > 1) us += 3.0 + 2e-6 * splits * M * N;          // the sums written and read at 4 TB/s, and another launch
        if (us >= best.us) continue;
        best.us = us; best.kind = kind; best.splits = splits;
        best.slab = splits > 1 ? (size_t)splits * M * N : 0;
    }
    return best;
}
static LxDeal lx_deal(int M, int N, int steps, int cus, bool loss) {
    LxDeal d = lx_deal_big(M, N, steps, cus, loss);
    for (int kind : {LX_SMALL128, LX_SMALL64}) {
        const LxDeal e = lx_deal_small(M, N, steps, cus, loss, kind);
        if (e.us < d.us) d = e;
    }
    return d;
}
// The logits of M rows and N classes.  Tiles of 256 x 256 that do not fill a last round of the chip are better given to the small kernel, in tiles it
// deals over all compute units: `rows` rows or `cols` classes from the front are the large kernel's (one of them is all), the others the small one's
// (2047 x 50021 x 1024, 6.1 rounds: 181 -> 171 us; 1024 x 50000 x 768: 90 -> 82; 3000 x 21843 x 768: 113 -> 103).  A row's sums are the same either way.
struct LxLogits { LxDeal front, rest; int rows, cols; };
static LxLogits lx_deal_logits(int M, int N, int steps, int cus) {
    LxLogits q = {lx_deal(M, N, steps, cus, true), {}, M, N};
    if (q.front.kind != LX_BIG) return q;
    const int tiles_m = (M + LX_TILE - 1) / LX_TILE, tiles_n = (N + LX_TILE - 1) / LX_TILE;
    const long long whole = (long long)tiles_m * tiles_n / cus * cus;
    double best = 0.98 * q.front.us;
    for (int by_rows = 0; by_rows < 2; ++by_rows) {
        const int front = (int)(whole / (by_rows ? tiles_n : tiles_m)) * LX_TILE;
        if (front <= 0 || front >= (by_rows ? M : N)) continue;
        const int rows = by_rows ? front : M, cols = by_rows ? N : front;
        const LxDeal f = lx_deal_big(rows, cols, steps, cus, true);
        for (int kind : {LX_SMALL128, LX_SMALL64}) {
            const LxDeal r = lx_deal_small(by_rows ? M - front : M, by_rows ? N : N - front, steps, cus, true, kind);
            if (f.us + r.us < best) { best = f.us + r.us; q = {f, r, rows, cols}; }
        }
    }
    return q;
}
// dx and dW of the same small kind share a launch: about 5 us less for the two, and each fills what the other leaves
static bool lx_one_launch(const LxDeal& dx, const LxDeal& dw) { return dx.kind == dw.kind && dx.kind != LX_BIG; }
static void lx_deal_grads(int n, int V, int D, int cus, LxDeal& dx, LxDeal& dw) {
    const int sx = (V + LX_BK - 1) / LX_BK, sw = (n + LX_BK - 1) / LX_BK;
    dx = lx_deal(n, D, sx, cus, false);
    dw = lx_deal(V, D, sw, cus, false);
    if (lx_one_launch(dx, dw)) return;
    for (int kind : {LX_SMALL128, LX_SMALL64}) {
        const LxDeal x = lx_deal_small(n, D, sx, cus, false, kind), w = lx_deal_small(V, D, sw, cus, false, kind);
        if (x.us + w.us < dx.us + dw.us + 5.0) { dx = x; dw = w; return; }
    }
}
static LxPlan lx_plan(long long T, int V, int D, int grad, int smoothing, int dw_f32, int bias, size_t block_bytes) {
    LxPlan q = {};
    q.ldp = ((long long)V + LX_TILE - 1) / LX_TILE * LX_TILE;
    q.stat_cols = q.ldp / LX_STAT;
    const size_t row = (grad ? (size_t)q.ldp * 2 : 0) + (size_t)q.stat_cols * (smoothing ? 12 : 8);
    long long rows = (long long)(block_bytes / row) / LX_TILE * LX_TILE;
    if (rows < LX_TILE) rows = LX_TILE;
    if (rows > (1 << 21)) rows = 1 << 21;
    if (rows > T) rows = T;
    q.blocks = (int)((T + rows - 1) / rows);
    // equal blocks: the last one is not a remnant
    rows = (T + q.blocks - 1) / q.blocks;
    if (q.blocks > 1) rows = (rows + LX_TILE - 1) / LX_TILE * LX_TILE;
    q.block = (int)rows;
    q.blocks = (int)((T + rows - 1) / rows);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += lx_up(n); return here; };
    q.scale = take(16 + LX_LOSS_WGS * sizeof(LxLossPart));          // scale, ticket, the loss's parts
    q.stats = take((size_t)rows * q.stat_cols * sizeof(float2));
    q.zsum = smoothing ? take((size_t)rows * q.stat_cols * sizeof(float)) : 0;
    if (grad) {
        q.P = take((size_t)((rows + LX_BK - 1) / LX_BK * LX_BK) * q.ldp * 2);
        q.xs = take((size_t)rows * D * 2);
        if (q.blocks > 1 && !dw_f32) q.acc = take((size_t)V * D * sizeof(float));
        const int cus = lx_cus();
        size_t slab = 0;            // dx and dW use it one after the other
        for (int last = q.blocks > 1 ? 0 : 1; last < 2; ++last) {          // [1]: the last block, which may be the only one
            const int n = last ? (int)(T - (long long)(q.blocks - 1) * rows) : (int)rows;
            lx_deal_grads(n, V, D, cus, q.dx[last], q.dw[last]);
            const size_t need = q.dx[last].slab + (lx_one_launch(q.dx[last], q.dw[last]) ? q.dw[last].slab : 0);
            if (need > slab) slab = need;
            if (q.dw[last].slab > slab) slab = q.dw[last].slab;
        }
        if (slab > 0) q.slab = take(slab * sizeof(float));
        if (bias) {
            q.colpart = take((size_t)lx_ranges(q.ldp) * q.ldp * sizeof(float));
            q.colsum = take((size_t)V * sizeof(float));
            q.delta = take((size_t)rows * sizeof(float));
        }
    }
    q.total = at;
    return q;
}

static void lx_tiles(LxGemmParams& p, const LxDeal& d) {
    const int tile = d.kind == LX_SMALL64 ? 64 : d.kind == LX_SMALL128 ? 128 : LX_TILE;
    p.tiles_m = (p.M + tile - 1) / tile;
    p.tiles_n = (p.N + tile - 1) / tile;
    p.splits = d.splits;
}
static int lx_reduce(const LxGemmParams& p, hipStream_t s, const char* what) {
    const long long quads = (long long)p.M * p.N / 4;
    lx_reduce_kernel<<<(int)((quads + 255) / 256 < 4096 ? (quads + 255) / 256 : 4096), 256, 0, s>>>(p);
    return vitk_check_launch(what);
}
template <int LAY, int EPI>
static int lx_launch(LxGemmParams& p, const LxDeal& d, hipStream_t s, const char* what) {
    lx_tiles(p, d);
    if (d.kind != LX_BIG) {
        constexpr int E = EPI == LX_OUT ? LX_OUT : LX_XENT_BIAS;
        const int grid = p.tiles_m * p.tiles_n * d.splits;
        if (d.kind == LX_SMALL64) lx_small_kernel<LAY, E, 1, 4, 1><<<grid, 256, 0, s>>>(p);
        else lx_small_kernel<LAY, E, 4, 2, 2><<<grid, 256, 0, s>>>(p);
        if (int rc = vitk_check_launch(what)) return rc;
        return d.splits > 1 ? lx_reduce(p, s, what) : VITK_OK;
    }
    static VitkLdsOnce once = {};
    if constexpr (EPI == LX_OUT) {
        if (int rc = vitk_lds_once(once, (const void*)lx_grad_kernel<LAY>, LX_GRAD_LDS, what)) return rc;
        p.width = d.width; p.teams = d.teams; p.whole = d.whole; p.rest = d.rest; p.ranges = d.ranges;
        lx_grad_kernel<LAY><<<d.teams * d.width, 256, LX_GRAD_LDS, s>>>(p);
        if (int rc = vitk_check_launch(what)) return rc;
        if (p.rest > 0) lx_join_kernel<<<p.rest * p.width * 32, 256, 0, s>>>(p);
    } else {
        if (int rc = vitk_lds_once(once, (const void*)lx_logits_kernel<EPI>, LX_LDS, what)) return rc;
        lx_logits_kernel<EPI><<<d.teams, 512, LX_LDS, s>>>(p);
    }
    return vitk_check_launch(what);
}

extern "C" {

size_t vitk_linear_xent_workspace(int64_t T, int V, int D, int want_grad, int smoothing, int dw_f32, int bias, size_t block_bytes) {
    if (T <= 0 || T > (1 << 30) || V <= 0 || V > (1 << 22) || D <= 0 || D > (1 << 20)) return 0;
    return lx_plan(T, V, D, want_grad, smoothing, dw_f32, bias, block_bytes).total;
}

int vitk_linear_xent(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, int bias_type, const int64_t* target, int64_t T, int V, int D,
                     float smoothing, int64_t ignore_index, int mean, float* loss, float* rows, void* dx, int64_t lddx, void* dw, int64_t lddw, int dw_f32,
                     void* db, int db_f32, void* workspace, size_t workspace_bytes, size_t block_bytes, void* stream) {
    VITK_REQUIRE(T > 0 && T <= (1 << 30) && V > 0 && V <= (1 << 22) && D > 0 && D <= (1 << 20), "linear_xent: bad shape T=%lld V=%d D=%d", (long long)T, V, D);
    VITK_REQUIRE(x && w && target && loss && rows && workspace, "linear_xent: null pointer");
    VITK_REQUIRE(D % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && ldx >= D && ldw >= D && ldx < (1 << 22) && ldw < (1 << 22),
                 "linear_xent: D and the row strides must be multiples of 8, strides from D to 2^22 (D=%d ldx=%lld ldw=%lld)", D, (long long)ldx, (long long)ldw);
    VITK_REQUIRE(vitk_aligned(x, 16) && vitk_aligned(w, 16) && vitk_aligned(workspace, 256) && vitk_aligned(target, 8), "linear_xent: rows must be 16-byte aligned");
    VITK_REQUIRE(smoothing >= 0.f && smoothing <= 1.f, "linear_xent: smoothing %g outside [0, 1]", (double)smoothing);
    VITK_REQUIRE(!bias || bias_type == 0 || bias_type == 1, "linear_xent: bias types are 0 (fp32) and 1 (bf16)");
    const bool grad = dx || dw || db;
    VITK_REQUIRE((!dx || (lddx % 8 == 0 && lddx >= D && vitk_aligned(dx, 16))) && (!dw || (lddw % 8 == 0 && lddw >= D && vitk_aligned(dw, 16))),
                 "linear_xent: gradient rows must be 16-byte aligned with strides that are multiples of 8 (lddx=%lld lddw=%lld)", (long long)lddx, (long long)lddw);
    VITK_REQUIRE(!db || bias, "linear_xent: db needs a bias");
    const LxPlan q = lx_plan(T, V, D, grad, smoothing > 0.f, dw_f32, db != nullptr, block_bytes);
    VITK_REQUIRE(!dw || !dw_f32 || q.blocks == 1 || lddw == D, "linear_xent: an fp32 dw over several blocks of rows must be contiguous");
    if (workspace_bytes < q.total) {
        vitk_set_error("linear_xent: workspace %zu < %zu", workspace_bytes, q.total);
        return VITK_ENOSPC;
    }
    hipStream_t s = (hipStream_t)stream;
    const int cus = lx_cus();
    const LxFactor factor = grad ? lx_factor(smoothing, V) : LxFactor{};
    char* ws = (char*)workspace;
    float* scale = (float*)(ws + q.scale);
    unsigned* ticket = (unsigned*)(ws + q.scale + 8);
    const long long* tg = (const long long*)target;
    if (q.blocks > 1 && grad) {
        lx_loss_kernel<<<1, 256, 0, s>>>(tg, ignore_index, nullptr, (int)T, (int)T, mean, factor.unit, nullptr, nullptr, scale, nullptr);
        if (int rc = vitk_check_launch("linear_xent_count")) return rc;
    }
    for (int b = 0; b < q.blocks; ++b) {
        const long long r0 = (long long)b * q.block;
        const int n = (int)(T - r0 < q.block ? T - r0 : q.block);
        const bool last = b == q.blocks - 1;
        LxGemmParams g = {};
        g.A = (const bf16_t*)x + r0 * ldx; g.lda = (int)ldx; g.B = (const bf16_t*)w; g.ldb = (int)ldw;
        g.M = n; g.N = V; g.KA = g.KB = D; g.steps = (D + LX_BK - 1) / LX_BK;
        g.bias = bias; g.bias_type = bias_type;
        g.stats = (float2*)(ws + q.stats); g.stat_cols = (int)q.stat_cols; g.zsum = smoothing > 0.f ? (float*)(ws + q.zsum) : nullptr;
        g.P = grad ? (unsigned short*)(ws + q.P) : nullptr; g.ldp = q.ldp; g.ticket = ticket;
        const LxLogits deal = lx_deal_logits(n, V, g.steps, cus);
        auto logits = [&](LxGemmParams q, const LxDeal& how) {
            return q.bias || q.zsum ? lx_launch<LX_NT, LX_XENT_BIAS>(q, how, s, "linear_xent_logits") : lx_launch<LX_NT, LX_XENT>(q, how, s, "linear_xent_logits");
        };
        LxGemmParams front = g, rest = g;
        front.M = deal.rows; front.N = deal.cols;
        if (int rc = logits(front, deal.front)) return rc;
        if (deal.rows < n || deal.cols < V) {
            const int r1 = deal.rows < n ? deal.rows : 0, c1 = deal.cols < V ? deal.cols : 0;          // multiples of 256
            rest.M = n - r1; rest.N = V - c1;
            rest.A = g.A + r1 * ldx; rest.B = g.B + c1 * ldw;
            if (bias) rest.bias = (const char*)bias + (size_t)c1 * (bias_type == 1 ? 2 : 4);
            const size_t entry = (size_t)r1 * g.stat_cols + c1 / LX_STAT;
            rest.stats = g.stats + entry;
            if (g.zsum) rest.zsum = g.zsum + entry;
            if (g.P) rest.P = g.P + r1 * g.ldp + c1;
            if (int rc = logits(rest, deal.rest)) return rc;
        }
        LxRowParams r = {};
        r.x = g.A; r.ldx = ldx; r.w = g.B; r.ldw = ldw; r.bias = bias; r.bias_type = bias_type; r.target = tg + r0; r.ignore_index = ignore_index;
        r.stats = g.stats; r.zsum = g.zsum; r.stat_cols = g.stat_cols;
        const bool fused = q.blocks == 1 && T <= LX_FUSED_ROWS && (!grad || (size_t)T * q.ldp * 2 <= LX_FUSED_BYTES);
        r.ticket = ticket; r.scale = scale; r.loss = fused ? loss : nullptr; r.mean = mean;
        r.P = (bf16_t*)g.P; r.ldp = q.ldp; r.rows = rows + r0; r.V = V; r.D = D; r.rows_n = n; r.smoothing = smoothing;
        r.a = factor.a; r.u = factor.u; r.hit = factor.hit; r.unit = factor.unit;
        r.pad_rows = dw && q.dw[last].kind == LX_BIG ? (LX_BK - n % LX_BK) % LX_BK : 0;
        r.xs = dw ? (bf16_t*)(ws + q.xs) : nullptr;
        r.delta = db ? (float*)(ws + q.delta) : nullptr;
        const int row_wgs = n + r.pad_rows;
        // long rows get more waves.  By the vocabulary alone, so that a row's sums do not depend on how many rows there are or what is wanted.
        // STREAM: past the caches, where the block is larger than they are.
        const bool stream = grad && (size_t)n * q.ldp * 2 > LX_CACHED;
        if (q.ldp >= 65536) {
            if (stream) lx_row_kernel<16, true><<<row_wgs, 1024, 0, s>>>(r);
            else lx_row_kernel<16, false><<<row_wgs, 1024, 0, s>>>(r);
        } else if (q.ldp >= 16384) {
            if (stream) lx_row_kernel<8, true><<<row_wgs, 512, 0, s>>>(r);
            else lx_row_kernel<8, false><<<row_wgs, 512, 0, s>>>(r);
        } else if (q.ldp >= 4096) {
            if (stream) lx_row_kernel<4, true><<<row_wgs, 256, 0, s>>>(r);
            else lx_row_kernel<4, false><<<row_wgs, 256, 0, s>>>(r);
        } else {
            if (stream) lx_row_kernel<1, true><<<(row_wgs + 3) / 4, 256, 0, s>>>(r);
            else lx_row_kernel<1, false><<<(row_wgs + 3) / 4, 256, 0, s>>>(r);
        }
        if (int rc = vitk_check_launch("linear_xent_rows")) return rc;
        if (last && !fused) {
            int per = (int)((T + LX_LOSS_WGS - 1) / LX_LOSS_WGS);
            if (per < 1024) per = 1024;
            lx_loss_kernel<<<(int)((T + per - 1) / per), 256, 0, s>>>(tg, ignore_index, rows, (int)T, per, mean, factor.unit, (LxLossPart*)(ws + q.scale + 16), ticket,
                                                                      q.blocks > 1 ? nullptr : scale, loss);
            if (int rc = vitk_check_launch("linear_xent_loss")) return rc;
        }
        if (!grad) continue;
        const bf16_t* dz = (const bf16_t*)(ws + q.P);
        // dx = dz W: dz is zero behind the vocabulary up to its row stride
        LxGemmParams d = {};
        d.A = dz; d.lda = (int)q.ldp; d.B = (const bf16_t*)w; d.ldb = (int)ldw; d.M = n; d.N = D; d.KA = (int)q.ldp; d.KB = V; d.steps = (V + LX_BK - 1) / LX_BK;
        d.scale = scale; d.out = (bf16_t*)dx + r0 * lddx; d.ldo = lddx; d.slab = (float*)(ws + q.slab);
        // dW = dz^T x, summed over the blocks in fp32
        LxGemmParams e = {};
        e.A = dz; e.lda = (int)q.ldp; e.B = r.xs; e.ldb = D; e.M = V; e.N = D; e.KA = e.KB = n; e.steps = (n + LX_BK - 1) / LX_BK;
        e.scale = scale; e.slab = d.slab;
        float* acc = dw_f32 ? (float*)dw : (float*)(ws + q.acc);
        e.add = b > 0 ? acc : nullptr;
        if (last) { e.out = dw; e.ldo = lddw; e.out_f32 = dw_f32; }
        else { e.out = acc; e.ldo = D; e.out_f32 = 1; }
        const LxColsum c = {dz, q.ldp, n, V, scale, db, db_f32, r.target, r.delta};
        const bool few = db != nullptr && q.blocks == 1 && n <= 1024;
        const LxDeal& dd = q.dx[last];
        const LxDeal& de = q.dw[last];
        const bool together = dx && dw && lx_one_launch(dd, de);
        if (together) {
            lx_tiles(d, dd);
            lx_tiles(e, de);
            e.slab = d.slab + dd.slab;
            const int bx = d.tiles_m * d.tiles_n * dd.splits, bw = e.tiles_m * e.tiles_n * de.splits;
            const int bc = few ? (int)(q.ldp / 128) : 0;
            if (dd.kind == LX_SMALL64) lx_small_grads_kernel<1, 4, 1><<<bx + bw + bc, 256, 0, s>>>(d, e, c, bx, bw);
            else lx_small_grads_kernel<4, 2, 2><<<bx + bw + bc, 256, 0, s>>>(d, e, c, bx, bw);
            if (int rc = vitk_check_launch("linear_xent_grads")) return rc;
            if (dd.splits > 1)
                if (int rc = lx_reduce(d, s, "linear_xent_dx_sum")) return rc;
            if (de.splits > 1)
                if (int rc = lx_reduce(e, s, "linear_xent_dw_sum")) return rc;
        } else {
            if (dx)
                if (int rc = lx_launch<LX_NN, LX_OUT>(d, dd, s, "linear_xent_dx")) return rc;
            if (dw)
                if (int rc = lx_launch<LX_TN, LX_OUT>(e, de, s, "linear_xent_dw")) return rc;
        }
        if (few) {
            if (!together) lx_colsum_few_kernel<<<(unsigned)(q.ldp / 128), 256, 0, s>>>(c);
            if (int rc = vitk_check_launch("linear_xent_db")) return rc;
        } else if (db != nullptr) {
            float* part = (float*)(ws + q.colpart);
            int per = (n + lx_ranges(q.ldp) - 1) / lx_ranges(q.ldp);
            if (per < 32) per = 32;
            const int ranges = (n + per - 1) / per;
            lx_colsum_kernel<<<dim3((unsigned)((q.ldp + 511) / 512), ranges), 256, 0, s>>>(dz, q.ldp, n, per, part, r.target, r.delta);
            lx_colsum_final_kernel<<<(V + 255) / 256, 256, 0, s>>>(part, q.ldp, ranges, V, scale, (float*)(ws + q.colsum), b == 0, last ? db : nullptr, db_f32);
            if (int rc = vitk_check_launch("linear_xent_db")) return rc;
        }
    }
    return VITK_OK;
}

}  // extern "C"
