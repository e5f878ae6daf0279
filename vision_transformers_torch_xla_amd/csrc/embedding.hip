// Lookup of token embeddings with scaling, out[t] = scale * table[ids[t]], and the gradient of the table,
// dtable[v] (+)= scale * sum over {t : ids[t] = v} of dout[t].  Both are HBM-bound.
//
// The gradient is summed without atomics: the tokens are sorted by id (stable, so the order inside a row is the order of the tokens),
// the sorted list is cut into pieces of equal length whatever the ids are, and a workgroup adds up the runs of equal ids inside its
// piece in fp32.  A run that ends inside its piece is final; the parts of a run that crosses pieces go to fp32 partial rows that a
// second kernel joins in order.  So one id that is half of all tokens costs what any other mix costs, and the result does not depend
// on the schedule.
// Ids outside [0, V) never become an address: the lookup gives a row of NaN for them, the gradient leaves them out.
#include "common.h"

struct EmbFwdParams {
    const void* ids; const void* table; void* out;
    long long T, V, ldt, ldo;
    int chunks;             // 8-element chunks per row
    int rows_per_block;
    float scale;
};

template <typename T8> struct Emb8;
template <> struct Emb8<bf16_t> {
    static __device__ __forceinline__ void load(const bf16_t* p, float (&v)[8]) { load8(p, v); }
    static __device__ __forceinline__ void store(bf16_t* p, const float (&v)[8]) { store8(p, v); }
};
template <> struct Emb8<float> {
    static __device__ __forceinline__ void load(const float* p, float (&v)[8]) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};

template <typename I>
static __device__ __forceinline__ long long emb_id(const void* ids, long long t) { return (long long)reinterpret_cast<const I*>(ids)[t]; }

// A block takes rows_per_block rows, flattened into 8-element chunks; a thread has up to four chunks in flight.  Bound by memory: 65536 rows of 1024
// bf16 values out of 50021 take 48 us with cold caches (237 MB at 4.9 TB/s), 31 us where the table is still in them.
template <typename I, typename TI, typename TO>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const EmbFwdParams p) {
    const long long row0 = (long long)blockIdx.x * p.rows_per_block;
    const long long left = p.T - row0;
    const unsigned rows = left < p.rows_per_block ? (unsigned)left : (unsigned)p.rows_per_block;
    const unsigned total = rows * (unsigned)p.chunks;
    const TI* table = reinterpret_cast<const TI*>(p.table);
    TO* out = reinterpret_cast<TO*>(p.out);
    for (unsigned base = threadIdx.x; base < total; base += 1024) {
        float v[4][8];
        unsigned row[4], col[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned c = base + j * 256;
            row[j] = c / (unsigned)p.chunks;
            col[j] = (c - row[j] * (unsigned)p.chunks) * 8u;
            if (c < total) {
                const long long id = emb_id<I>(p.ids, row0 + row[j]);
                if (id >= 0 && id < p.V) {
                    Emb8<TI>::load(table + id * p.ldt + col[j], v[j]);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[j][k] = __builtin_nanf("");
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (base + j * 256 < total) {
#pragma unroll
                for (int k = 0; k < 8; ++k) v[j][k] *= p.scale;
                Emb8<TO>::store(out + (row0 + row[j]) * p.ldo + col[j], v[j]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------- sorting
// Stable radix sort of (key, position) by key, 9 bits a pass.  Key V is the sentinel of tokens without a gradient (padding, an id out
// of range); it sorts behind every row.
#define SORT_BINS 512
#define SORT_BITS 9
#define SORT_THREADS 1024
#define SORT_WAVES (SORT_THREADS / 64)
#define SORT_ITEMS 2            // 2048 tokens a workgroup (100352 tokens: the four launches take 21 us; with 4096 25; 256 threads of 8 28, of 16 39)

template <typename I>
static __device__ __forceinline__ unsigned emb_key(const void* ids, long long t, long long V, long long padding) {
    const long long id = emb_id<I>(ids, t);
    return id >= 0 && id < V && id != padding ? (unsigned)id : (unsigned)V;
}
// lanes of the wave with the same digit: their mask
static __device__ __forceinline__ unsigned long long sort_peers(unsigned digit) {
    unsigned long long m = ~0ull;
#pragma unroll
    for (int b = 0; b < SORT_BITS; ++b) {
        const unsigned long long bal = __ballot((digit >> b) & 1u);
        m &= (digit >> b) & 1u ? bal : ~bal;
    }
    return m;
}
// inclusive sum over the wave
static __device__ __forceinline__ unsigned wave_scan(unsigned v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
// rank of the thread's items among the block's: items j = 0.. of wave w are tokens w * 64 * SORT_ITEMS + j * 64 + lane, so the order of
// (wave, item, lane) is the order of the input.  hist[wave][bin] holds the wave's first rank per bin and is moved on.
static __device__ __forceinline__ unsigned sort_rank(unsigned* hist_wave, unsigned digit) {
    const int lane = threadIdx.x & 63;
    const unsigned long long m = sort_peers(digit);
    const unsigned before = (unsigned)__popcll(m & ((1ull << lane) - 1ull));
    const unsigned base = hist_wave[digit];         // the wave's LDS operations run in order: all lanes read before the first of a bin writes
    asm volatile("" ::: "memory");
    if (before == 0) hist_wave[digit] = base + (unsigned)__popcll(m);
    asm volatile("" ::: "memory");
    return base + before;
}

// Grouping in one launch, for up to 28672 tokens of a vocabulary up to 2^18.  Workgroup g of 256 owns the ids that are g modulo 256.  It
// reads ALL ids (out of the L2 cache), counts how many belong to the workgroups before it - which is where its part of the sorted list
// begins, so the workgroups need nothing from each other - and keeps its own tokens in a list in LDS, one in 256 of a text's.  Wave w has
// a contiguous stretch of the tokens, so its list is in their order; a token's place is the wave's first one for its id plus the number of
// equal ids before it in the wave.  A wave with more own tokens than its list holds reads its stretch again instead.  Tokens without a
// gradient come last.  The workgroups behind the 256 zero the gradient meanwhile.  16384 tokens and 77 MB of zeros take 19 us together
// (a radix sort in one workgroup 46 us).  A whole gradient with it and with the four launches below, 8192 x 768: 1024 tokens 18 and 26 us, 16384 29 and
// 33, 32768 39 and 37, 49152 50 and 42.
#define GROUP_MAX 28672
#define GROUP_WG 256
#define GROUP_WAVES 16
#define GROUP_LIST 192          // list entries of a wave
#define GROUP_AHEAD 8           // strips of 64 ids in flight
static size_t emb_group_lds(long long V) {
    return (size_t)GROUP_WAVES * GROUP_LIST * sizeof(uint2) + (size_t)GROUP_WAVES * ((V + GROUP_WG - 1) / GROUP_WG) * sizeof(unsigned) + 2 * GROUP_WAVES * sizeof(unsigned);
}
template <typename I>
__global__ __launch_bounds__(1024) void emb_group_kernel(const void* ids, int T, long long V, long long padding, uint2* sorted, uint4* zero, long long zero16) {
    extern __shared__ uint2 group_sh[];         // [16][GROUP_LIST] own tokens, [16][rows] counts, [2][16] sums
    if (blockIdx.x >= GROUP_WG) {
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        const long long step = (long long)(gridDim.x - GROUP_WG) * 1024;
        for (long long i = (long long)(blockIdx.x - GROUP_WG) * 1024 + threadIdx.x; i < zero16; i += step) zero[i] = z;
        return;
    }
    const unsigned own = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned long long lower = (1ull << lane) - 1ull;
    const int rows = (int)((V + GROUP_WG - 1) / GROUP_WG);
    uint2* list = group_sh + wave * GROUP_LIST;
    unsigned* hist = reinterpret_cast<unsigned*>(group_sh + GROUP_WAVES * GROUP_LIST);
    unsigned* sums = hist + GROUP_WAVES * rows;
    unsigned* mine = hist + wave * rows;
    for (int i = threadIdx.x; i < GROUP_WAVES * rows; i += 1024) hist[i] = 0;
    __syncthreads();
    const int strips = (T + 63) / 64, per = (strips + GROUP_WAVES - 1) / GROUP_WAVES;
    const int s0 = wave * per, s1 = s0 + per < strips ? s0 + per : strips;
    unsigned before = 0, valid = 0;         // of the lane's tokens: those of workgroups before this one, those with a gradient
    int listed = 0;                         // the wave's own tokens
    for (int s = s0; s < s1; s += GROUP_AHEAD) {
        unsigned key[GROUP_AHEAD];
#pragma unroll
        for (int j = 0; j < GROUP_AHEAD; ++j) {
            const int t = (s + j) * 64 + lane;
            key[j] = s + j < s1 && t < T ? emb_key<I>(ids, t, V, padding) : (unsigned)V;
        }
#pragma unroll
        for (int j = 0; j < GROUP_AHEAD; ++j) {
            const unsigned g = key[j] & (GROUP_WG - 1);
            const bool ok = key[j] < (unsigned)V, hit = ok && g == own;
            valid += ok ? 1u : 0u;
            before += ok && g < own ? 1u : 0u;
            const unsigned long long m = __ballot(hit);
            if (m != 0) {
                if (hit) {
                    atomicAdd(&mine[key[j] / GROUP_WG], 1u);
                    const int at = listed + __popcll(m & lower);
                    if (at < GROUP_LIST) list[at] = make_uint2(key[j], (unsigned)((s + j) * 64 + lane));
                }
                listed += __popcll(m);
            }
        }
    }
    before = wave_scan(before);
    valid = wave_scan(valid);
    if (lane == 63) { sums[wave] = before; sums[GROUP_WAVES + wave] = valid; }
    __syncthreads();
    unsigned at = 0, total_valid = 0;
#pragma unroll
    for (int w = 0; w < GROUP_WAVES; ++w) { at += sums[w]; total_valid += sums[GROUP_WAVES + w]; }
    __syncthreads();
    // first places: ids in order, within an id the waves in order; `rows` is at most 1024
    {
        const int r = (int)threadIdx.x;
        unsigned count = 0;
        if (r < rows)
            for (int w = 0; w < GROUP_WAVES; ++w) { const unsigned c = hist[w * rows + r]; hist[w * rows + r] = count; count += c; }
        const unsigned incl = wave_scan(count);
        if (lane == 63) sums[wave] = incl;
        __syncthreads();
        unsigned base = at + incl - count;
        for (int w = 0; w < wave; ++w) base += sums[w];
        if (r < rows)
            for (int w = 0; w < GROUP_WAVES; ++w) hist[w * rows + r] += base;
        __syncthreads();
    }
    // the wave's own tokens of one group of 64 are put down; one round for each different id among them
    auto place = [&](unsigned key, unsigned t, bool hit) {
        unsigned long long left = __ballot(hit);
        while (left != 0) {
            const unsigned k = (unsigned)__builtin_amdgcn_readlane((int)key, (int)__builtin_ctzll(left));
            const unsigned long long same = __ballot(hit && key == k);
            if (hit && key == k) {
                const unsigned first = mine[k / GROUP_WG];
                asm volatile("" ::: "memory");
                const unsigned n = (unsigned)__popcll(same & lower);
                sorted[first + n] = make_uint2(key, t);
                if (n == 0) mine[k / GROUP_WG] = first + (unsigned)__popcll(same);
                asm volatile("" ::: "memory");
            }
            left &= ~same;
        }
    };
    if (listed <= GROUP_LIST) {
        for (int i = 0; i < listed; i += 64) {
            const uint2 e = i + lane < listed ? list[i + lane] : make_uint2(0u, 0u);
            place(e.x, e.y, i + lane < listed);
        }
    } else {
        for (int s = s0; s < s1; ++s) {
            const int t = s * 64 + lane;
            const unsigned key = t < T ? emb_key<I>(ids, t, V, padding) : (unsigned)V;
            place(key, (unsigned)t, key < (unsigned)V && (key & (GROUP_WG - 1)) == own);
        }
    }
    for (unsigned i = total_valid + own * 1024u + threadIdx.x; i < (unsigned)T; i += GROUP_WG * 1024u) sorted[i] = make_uint2((unsigned)V, 0u);
}

// Several workgroups: per pass a histogram launch (counts[block][bin]) and a launch that turns the counts into ranks and scatters.  For that a
// workgroup adds up the counts of all others; from SORT_DIRECT workgroups on, a launch in between turns the counts of SORT_GROUP workgroups
// into sums over those before and a total per group, so that only the totals are added up.
#define SORT_BLOCK (SORT_THREADS * SORT_ITEMS)       // tokens per workgroup
#define SORT_DIRECT 128
#define SORT_GROUP 32

template <typename I, bool FIRST>
static __device__ __forceinline__ uint2 sort_item(const void* ids, const uint2* in, long long t, long long T, long long V, long long padding) {
    if (t >= T) return make_uint2(0xffffffffu, 0u);
    if (FIRST) return make_uint2(emb_key<I>(ids, t, V, padding), (unsigned)t);
    return in[t];
}

template <typename I, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void emb_hist_kernel(const void* ids, const uint2* in, long long T, long long V, long long padding, int shift,
                                                       unsigned* counts, int blocks, uint4* zero, long long zero16) {
    __shared__ unsigned hist[SORT_BINS];
    if ((int)blockIdx.x >= blocks) {        // the blocks behind the sort's zero the gradient (first pass only)
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        const long long step = (long long)(gridDim.x - blocks) * SORT_THREADS;
        for (long long i = (long long)(blockIdx.x - blocks) * SORT_THREADS + threadIdx.x; i < zero16; i += step) zero[i] = z;
        return;
    }
    if (threadIdx.x < SORT_BINS) hist[threadIdx.x] = 0;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * SORT_BLOCK;
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const long long t = t0 + j * SORT_THREADS + threadIdx.x;
        const uint2 it = sort_item<I, FIRST>(ids, in, t, T, V, padding);
        if (t < T) atomicAdd(&hist[(it.x >> shift) & (SORT_BINS - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < SORT_BINS) counts[(size_t)blockIdx.x * SORT_BINS + threadIdx.x] = hist[threadIdx.x];
}

__global__ __launch_bounds__(SORT_BINS) void emb_scan_kernel(unsigned* counts, int blocks, unsigned* totals) {
    const int b0 = blockIdx.x * SORT_GROUP, n = blocks - b0 < SORT_GROUP ? blocks - b0 : SORT_GROUP;
    unsigned* q = counts + (size_t)b0 * SORT_BINS + threadIdx.x;
    unsigned c[SORT_GROUP], sum = 0;
#pragma unroll
    for (int b = 0; b < SORT_GROUP; ++b) c[b] = b < n ? q[b * SORT_BINS] : 0u;
#pragma unroll
    for (int b = 0; b < SORT_GROUP; ++b) {
        if (b < n) q[b * SORT_BINS] = sum;
        sum += c[b];
    }
    totals[(size_t)blockIdx.x * SORT_BINS + threadIdx.x] = sum;
}

// totals: the counts themselves and entries = blocks, or the groups' totals
template <typename I, bool FIRST>
__global__ __launch_bounds__(SORT_THREADS) void emb_scatter_kernel(const void* ids, const uint2* in, long long T, long long V, long long padding, int shift,
                                                          const unsigned* __restrict__ counts, const unsigned* __restrict__ totals, int entries, uint2* out) {
    __shared__ unsigned hist[SORT_WAVES * SORT_BINS];
    __shared__ unsigned sums[SORT_WAVES];
    __shared__ unsigned odd[2][SORT_BINS];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    unsigned* mine = hist + wave * SORT_BINS;
    for (int i = threadIdx.x; i < SORT_WAVES * SORT_BINS; i += SORT_THREADS) hist[i] = 0;
    __syncthreads();
    uint2 item[SORT_ITEMS];
    const long long t0 = (long long)blockIdx.x * SORT_BLOCK + wave * (64 * SORT_ITEMS);
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const long long t = t0 + j * 64 + lane;
        item[j] = sort_item<I, FIRST>(ids, in, t, T, V, padding);
        if (t < T) atomicAdd(&mine[(item[j].x >> shift) & (SORT_BINS - 1)], 1u);
    }
    // threads i and 512 + i add up the even and the odd entries of bin i: its total and the share of the blocks before this one
    const int bin = (int)threadIdx.x & (SORT_BINS - 1);
    const int own = totals == counts ? (int)blockIdx.x : (int)blockIdx.x / SORT_GROUP;
    unsigned tot = 0, pre = 0;
#pragma unroll 8
    for (int b = threadIdx.x / SORT_BINS; b < entries; b += SORT_THREADS / SORT_BINS) {
        const unsigned c = totals[(size_t)b * SORT_BINS + bin];
        pre += b < own ? c : 0u;
        tot += c;
    }
    if (threadIdx.x >= SORT_BINS) { odd[0][bin] = tot; odd[1][bin] = pre; }
    __syncthreads();
    unsigned incl = 0;
    if (threadIdx.x < SORT_BINS) {
        tot += odd[0][bin];
        pre += odd[1][bin] + (totals != counts ? counts[(size_t)blockIdx.x * SORT_BINS + bin] : 0u);
        incl = wave_scan(tot);
        if (lane == 63) sums[wave] = incl;
    }
    __syncthreads();
    if (threadIdx.x < SORT_BINS) {
        unsigned r = incl - tot + pre;
        for (int w = 0; w < wave; ++w) r += sums[w];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            const unsigned c = hist[w * SORT_BINS + bin];
            hist[w * SORT_BINS + bin] = r;
            r += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const long long t = t0 + j * 64 + lane;
        // tokens behind the last one take ranks of bin 511 behind every real one of this block, which is the last block; they are not stored
        const unsigned r = sort_rank(mine, (item[j].x >> shift) & (SORT_BINS - 1));
        if (t < T) out[r] = item[j];
    }
}

// ---------------------------------------------------------------------------------------------------- sums
struct EmbBwdParams {
    const uint2* sorted; const void* dout; void* out; float* partial;       // partial: [pieces][2][D]: the piece's head run, its tail run
    long long T, V, ldd, ldo;
    int D, piece, pieces, accumulate;
    float scale;
};

template <typename TO>
static __device__ __forceinline__ void emb_put(const EmbBwdParams& p, unsigned key, int col, float (&acc)[8]) {
    TO* q = reinterpret_cast<TO*>(p.out) + (long long)key * p.ldo + col;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] *= p.scale;
    if (p.accumulate) {
        float o[8];
        Emb8<TO>::load(q, o);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] += o[k];
    }
    Emb8<TO>::store(q, acc);
}

// A row of blockDim.x threads per piece of the sorted list and slice of 8 * blockDim.x columns; narrow tables have several pieces to a wave.
// The rows of a piece are independent loads: EMB_AHEAD of them are in flight while the sums are formed in order.  100352 rows of 768 bf16 values take
// 29 us (154 MB read at 5.3 TB/s), 16384 rows 9 us out of the caches.
#define EMB_AHEAD 8
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void embedding_bwd_kernel(const EmbBwdParams p) {
    const int col = ((int)blockIdx.y * (int)blockDim.x + (int)threadIdx.x) * 8;
    const long long piece = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    if (col >= p.D || piece >= p.pieces) return;
    const long long i0 = piece * p.piece;
    const long long i1 = i0 + p.piece < p.T ? i0 + p.piece : p.T;
    const TI* dout = reinterpret_cast<const TI*>(p.dout);
    float* part = p.partial + (size_t)piece * 2 * p.D + col;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    unsigned key = p.sorted[i0].x;
    if ((long long)key >= p.V) return;
    bool head = i0 > 0 && p.sorted[i0 - 1].x == key;        // the run began in an earlier piece
    for (long long i = i0; i < i1; i += EMB_AHEAD) {
        float v[EMB_AHEAD][8];
        uint2 it[EMB_AHEAD];
#pragma unroll
        for (int j = 0; j < EMB_AHEAD; ++j) {
            const long long at = i + j < i1 ? i + j : i1 - 1;
            it[j] = p.sorted[at];
        }
#pragma unroll
        for (int j = 0; j < EMB_AHEAD; ++j) Emb8<TI>::load(dout + (long long)it[j].y * p.ldd + col, v[j]);
#pragma unroll
        for (int j = 0; j < EMB_AHEAD; ++j) {
            if (i + j >= i1) break;
            if (it[j].x != key) {
                if ((long long)key < p.V) {
                    if (head) Emb8<float>::store(part, acc);
                    else emb_put<TO>(p, key, col, acc);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] = 0.f;
                key = it[j].x;
                head = false;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += v[j][k];
        }
        if ((long long)key >= p.V) break;       // only tokens without a gradient follow
    }
    if ((long long)key >= p.V) return;
    const bool goes_on = i1 < p.T && p.sorted[i1].x == key;
    if (head) Emb8<float>::store(part, acc);
    else if (goes_on) Emb8<float>::store(part + p.D, acc);
    else emb_put<TO>(p, key, col, acc);
}

// Runs that cross pieces: the threads of the piece a run begins in (as its tail) add the head sums of the pieces that follow; of a table that
// takes a wave or more per piece (GROUPS = 4) a quarter of them each of four groups of threads, then the four in order.
template <typename TO, int GROUPS>
__global__ __launch_bounds__(1024) void embedding_join_kernel(const EmbBwdParams p) {
    __shared__ float quarter[GROUPS > 1 ? GROUPS - 1 : 1][256][8];
    const int col = ((int)blockIdx.y * (int)blockDim.x + (int)threadIdx.x) * 8;
    const int group = GROUPS > 1 ? (int)threadIdx.y : 0;
    const long long piece = GROUPS > 1 ? (long long)blockIdx.x : (long long)blockIdx.x * blockDim.y + threadIdx.y;
    if (piece + 1 >= p.pieces) return;
    const long long i1 = (piece + 1) * p.piece;
    const unsigned key = p.sorted[i1 - 1].x;
    if ((long long)key >= p.V || p.sorted[i1].x != key) return;       // nothing crosses this border
    const long long i0 = i1 - p.piece;
    if (p.sorted[i0].x == key && i0 > 0 && p.sorted[i0 - 1].x == key) return;       // the run began earlier
    // how many pieces the run enters (equal ids are neighbours: first piece whose first id is another one)
    long long lo = piece + 1, hi = p.pieces;
    while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if (p.sorted[mid * p.piece].x == key) lo = mid + 1; else hi = mid;
    }
    const long long c0 = piece + 1, n = lo - c0;
    const long long from = c0 + n * group / GROUPS, to = c0 + n * (group + 1) / GROUPS;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col < p.D) {
        if (group == 0) Emb8<float>::load(p.partial + ((size_t)piece * 2 + 1) * p.D + col, acc);
        const float* q = p.partial + col;
        constexpr int JOIN_AHEAD = GROUPS > 1 ? 4 : 8;        // partial rows in flight (8 in each of four groups: 9.4 instead of 6.3 us where most runs end at once)
        for (long long c = from; c < to; c += JOIN_AHEAD) {
            float v[JOIN_AHEAD][8];
#pragma unroll
            for (int j = 0; j < JOIN_AHEAD; ++j)
                if (j == 0 || c + j < to) Emb8<float>::load(q + (size_t)(c + j) * 2 * p.D, v[j]);
#pragma unroll
            for (int j = 0; j < JOIN_AHEAD; ++j)
                if (c + j < to) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[k] += v[j][k];
                }
        }
    }
    if constexpr (GROUPS > 1) {
        if (group > 0) Emb8<float>::store(quarter[group - 1][threadIdx.x], acc);
        __syncthreads();
        if (group > 0 || col >= p.D) return;
#pragma unroll
        for (int g = 0; g < GROUPS - 1; ++g)
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += quarter[g][threadIdx.x][k];
    }
    if (col < p.D) emb_put<TO>(p, key, col, acc);
}

// Few tokens: everything in one launch, without a list.  The last workgroups zero the rows that no token has; each of the others is one token
// and a slice of the columns, and if its token is the first with its id it collects the tokens that have the same one, in order, and
// adds them up: up to eight by one group of threads, more by 256 / lanes groups, a stretch each, whose sums are joined in order.
// A call takes 9 us instead of 16 (512 tokens, 1000 x 768), with 50021 x 768 to zero 16 instead of 21; the worst mix, one id alone before so large a
// table, 28 instead of 22.  Most workgroups end at once, but 4096 of them take as long to start as the other form needs.
#define FEW_MAX 1024
#define FEW_WGS 2048            // tokens times slices
#define FEW_AHEAD 16
#define FEW_ROWS 2048           // rows of the gradient a workgroup zeroes at a time, at most
template <typename I, typename TI, typename TO>
__global__ __launch_bounds__(256) void embedding_bwd_few_kernel(const EmbBwdParams p, const void* ids, long long padding, int zero_wgs, int zero_rows, int slices, int lanes) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, T = (int)p.T;
    unsigned key[FEW_MAX / 256];
#pragma unroll
    for (int r = 0; r < FEW_MAX / 256; ++r) key[r] = r * 256 + tid < T ? emb_key<I>(ids, r * 256 + tid, p.V, padding) : (unsigned)p.V;
    const int block = (int)blockIdx.x - T * slices;
    if (block >= 0) {
        __shared__ unsigned taken[FEW_ROWS / 32];
        const unsigned row16 = (unsigned)(p.D * sizeof(TO) / 16);
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        for (long long r0 = (long long)block * zero_rows; r0 < p.V; r0 += (long long)zero_wgs * zero_rows) {
            const int rows = p.V - r0 < zero_rows ? (int)(p.V - r0) : zero_rows;
            if (tid < FEW_ROWS / 32) taken[tid] = 0u;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < FEW_MAX / 256; ++r) {
                const long long at = (long long)key[r] - r0;
                if (key[r] < (unsigned)p.V && at >= 0 && at < rows) atomicOr(&taken[at >> 5], 1u << (at & 31));
            }
            __syncthreads();
            uint4* q = reinterpret_cast<uint4*>(reinterpret_cast<TO*>(p.out) + r0 * p.D);
            for (unsigned i = tid; i < rows * row16; i += 256) {
                const unsigned r = i / row16;
                if (((taken[r >> 5] >> (r & 31)) & 1u) == 0u) q[i] = z;
            }
            __syncthreads();
        }
        return;
    }
    __shared__ unsigned short list[FEW_MAX];
    __shared__ int counts[FEW_MAX / 64];
    __shared__ float sums[256][8];
    const int t = (int)blockIdx.x / slices, slice = (int)blockIdx.x - t * slices;
    const unsigned mine = emb_key<I>(ids, t, p.V, padding);
    if (mine == (unsigned)p.V) return;
    unsigned long long same[FEW_MAX / 256];
#pragma unroll
    for (int r = 0; r < FEW_MAX / 256; ++r) {
        same[r] = __ballot(key[r] == mine);
        if (lane == 0) counts[r * 4 + wave] = __popcll(same[r]);
    }
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < FEW_MAX / 64; ++w) {
        if ((w & 3) == wave && key[w >> 2] == mine) list[n + __popcll(same[w >> 2] & ((1ull << lane) - 1ull))] = (unsigned short)((w >> 2) * 256 + tid);
        n += counts[w];
    }
    __syncthreads();
    if (list[0] != t) return;
    const int groups = n > 8 ? 256 / lanes : 1, g = tid / lanes, col = (slice * lanes + tid - g * lanes) * 8;
    const int from = g < groups ? n * g / groups : 0, to = g < groups ? n * (g + 1) / groups : 0;
    const TI* dout = reinterpret_cast<const TI*>(p.dout) + col;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (col < p.D) {
        for (int i = from; i < to; i += FEW_AHEAD) {
            float v[FEW_AHEAD][8];
#pragma unroll
            for (int j = 0; j < FEW_AHEAD; ++j)
                if (i + j < to) Emb8<TI>::load(dout + (long long)list[i + j] * p.ldd, v[j]);
#pragma unroll
            for (int j = 0; j < FEW_AHEAD; ++j)
                if (i + j < to) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[k] += v[j][k];
                }
        }
    }
    if (groups > 1) {
        if (g > 0) Emb8<float>::store(sums[tid], acc);
        __syncthreads();
        if (g == 0)
            for (int o = 1; o < groups; ++o)
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] += sums[o * lanes + tid][k];
    }
    if (g == 0 && col < p.D) emb_put<TO>(p, mine, col, acc);
}

// threads per piece: the columns in eights, a power of two below a wave and whole waves above
static int emb_lanes(int D) {
    const int n = D / 8;
    if (n >= 256) return 256;
    if (n > 32) return (n + 63) / 64 * 64;
    int w = 1;
    while (w < n) w *= 2;
    return w;
}
// tokens per piece: about 1024 workgroups where there are enough tokens, 16 to 512 tokens each (2048 of 8 and more: the sums take as long, the
// joining of their parts 7.4 and 10.9 instead of 6.1 and 6.6 us for 16384 and 100352 tokens of 768 columns)
static int emb_piece(long long T, int D) {
    const int lanes = emb_lanes(D), side = lanes < 64 ? 256 / lanes : 1;
    const long long wgs = side > 1 ? 512 * side : 1024;
    long long c = (T + wgs - 1) / wgs;
    c = (c + 7) / 8 * 8;
    return (int)(c < 16 ? 16 : c > 512 ? 512 : c);
}
static int emb_passes(long long V) {
    int bits = 0;
    while (bits < 32 && (V >> bits) != 0) ++bits;        // keys 0 .. V
    return (bits + SORT_BITS - 1) / SORT_BITS;
}
static bool emb_one(long long T, long long V) { return T <= GROUP_MAX && V <= (1 << 18); }
static int emb_few_lanes(int D) { return D > 256 ? 32 : emb_lanes(D); }
static int emb_few_slices(int D) { return (D / 8 + emb_few_lanes(D) - 1) / emb_few_lanes(D); }
static bool emb_few(long long T, int D) { return T <= FEW_MAX && T * emb_few_slices(D) <= FEW_WGS; }
static long long emb_sort_blocks(long long T) { return (T + SORT_BLOCK - 1) / SORT_BLOCK; }
static long long emb_sort_groups(long long T) { return emb_sort_blocks(T) > SORT_DIRECT ? (emb_sort_blocks(T) + SORT_GROUP - 1) / SORT_GROUP : 0; }
static size_t emb_up(size_t n) { return (n + 255) & ~(size_t)255; }

extern "C" {

int vitk_embedding_fwd(const void* ids, int ids_are_64, const void* table, int table_type, int64_t ldt, void* out, int out_type, int64_t ldo,
                       int64_t T, int64_t V, int D, float scale, void* stream) {
    VITK_REQUIRE(T >= 0 && V > 0 && D > 0, "embedding_fwd: bad shape T=%lld V=%lld D=%d", (long long)T, (long long)V, D);
    VITK_REQUIRE((table_type == 0 || table_type == 1) && (out_type == 0 || out_type == 1), "embedding_fwd: types are 0 (fp32) and 1 (bf16)");
    if (T == 0) return VITK_OK;
    VITK_REQUIRE(ids && table && out, "embedding_fwd: null pointer");
    VITK_REQUIRE(D % 8 == 0 && ldt % 8 == 0 && ldo % 8 == 0 && ldt >= D && ldo >= D, "embedding_fwd: D and the row strides must be multiples of 8, strides >= D (D=%d ldt=%lld ldo=%lld)",
                 D, (long long)ldt, (long long)ldo);
    VITK_REQUIRE(vitk_aligned(table, 16) && vitk_aligned(out, 16) && vitk_aligned(ids, ids_are_64 ? 8 : 4), "embedding_fwd: rows must be 16-byte aligned");
    EmbFwdParams p;
    p.ids = ids; p.table = table; p.out = out; p.T = T; p.V = V; p.ldt = ldt; p.ldo = ldo; p.scale = scale;
    p.chunks = D / 8;
    p.rows_per_block = p.chunks >= 1024 ? 1 : 1024 / p.chunks;
    const long long blocks = (T + p.rows_per_block - 1) / p.rows_per_block;
    VITK_REQUIRE(blocks < 0x7fffffff, "embedding_fwd: too many tokens (%lld)", (long long)T);
    hipStream_t s = (hipStream_t)stream;
#define EMB_FWD(I, TI, TO) embedding_fwd_kernel<I, TI, TO><<<(int)blocks, 256, 0, s>>>(p)
    switch ((ids_are_64 ? 4 : 0) | (table_type << 1) | out_type) {
        case 0: EMB_FWD(int32_t, float, float); break;
        case 1: EMB_FWD(int32_t, float, bf16_t); break;
        case 2: EMB_FWD(int32_t, bf16_t, float); break;
        case 3: EMB_FWD(int32_t, bf16_t, bf16_t); break;
        case 4: EMB_FWD(int64_t, float, float); break;
        case 5: EMB_FWD(int64_t, float, bf16_t); break;
        case 6: EMB_FWD(int64_t, bf16_t, float); break;
        default: EMB_FWD(int64_t, bf16_t, bf16_t); break;
    }
#undef EMB_FWD
    return vitk_check_launch("embedding_fwd");
}

size_t vitk_embedding_bwd_workspace(int64_t T, int64_t V, int D) {
    if (T <= 0 || V <= 0 || D <= 0 || emb_few(T, D)) return 0;
    const long long pieces = (T + emb_piece(T, D) - 1) / emb_piece(T, D);
    size_t n = emb_up((size_t)T * sizeof(uint2)) + emb_up((size_t)pieces * 2 * D * sizeof(float));
    if (!emb_one(T, V)) n += emb_up((size_t)T * sizeof(uint2)) + emb_up((size_t)(emb_sort_blocks(T) + emb_sort_groups(T)) * SORT_BINS * sizeof(unsigned));
    return n;
}

int vitk_embedding_bwd(const void* dout, int dout_type, int64_t ldd, const void* ids, int ids_are_64, void* dtable, int dtable_type, int64_t ldo,
                       int64_t T, int64_t V, int D, float scale, int64_t padding_idx, int accumulate, void* workspace, size_t workspace_bytes,
                       void* stream) {
    VITK_REQUIRE(T >= 0 && V > 0 && D > 0, "embedding_bwd: bad shape T=%lld V=%lld D=%d", (long long)T, (long long)V, D);
    VITK_REQUIRE((dout_type == 0 || dout_type == 1) && (dtable_type == 0 || dtable_type == 1), "embedding_bwd: types are 0 (fp32) and 1 (bf16)");
    VITK_REQUIRE(T < 0x7fffffffll && V < 0x7fffffffll && D <= (1 << 23), "embedding_bwd: T and V must be below 2^31, D at most 2^23");
    VITK_REQUIRE(dtable && (workspace || emb_few(T, D)) && (T == 0 || (dout && ids)), "embedding_bwd: null pointer");
    VITK_REQUIRE(D % 8 == 0 && ldd % 8 == 0 && ldo % 8 == 0 && ldd >= D && ldo >= D, "embedding_bwd: D and the row strides must be multiples of 8, strides >= D (D=%d ldd=%lld ldo=%lld)",
                 D, (long long)ldd, (long long)ldo);
    VITK_REQUIRE(vitk_aligned(dtable, 16) && vitk_aligned(workspace, 16) && (T == 0 || (vitk_aligned(dout, 16) && vitk_aligned(ids, ids_are_64 ? 8 : 4))),
                 "embedding_bwd: rows must be 16-byte aligned");
    VITK_REQUIRE(accumulate || ldo == D, "embedding_bwd: without accumulate the gradient must be contiguous (ldo == D)");
    if (workspace_bytes < vitk_embedding_bwd_workspace(T, V, D)) {
        vitk_set_error("embedding_bwd: workspace %zu < %zu", workspace_bytes, vitk_embedding_bwd_workspace(T, V, D));
        return VITK_ENOSPC;
    }
    if (T == 0 && accumulate) return VITK_OK;
    hipStream_t s = (hipStream_t)stream;
    EmbBwdParams p = {};
    p.dout = dout; p.out = dtable; p.T = T; p.V = V; p.ldd = ldd; p.ldo = ldo; p.D = D; p.accumulate = accumulate; p.scale = scale;
    const int types = (dout_type << 1) | dtable_type;
    if (emb_few(T, D)) {
        const int lanes = emb_few_lanes(D), few_slices = emb_few_slices(D);
        const long long bytes = (long long)D * (dtable_type == 0 ? 4 : 2);
        const int zero_rows = (int)(bytes >= 65536 ? 1 : 65536 / bytes < FEW_ROWS ? 65536 / bytes : FEW_ROWS);
        const int zero_wgs = accumulate ? 0 : (int)((V + zero_rows - 1) / zero_rows < 1024 ? (V + zero_rows - 1) / zero_rows : 1024);
#define EMB_FEW(TI, TO)                                                                                                                                    \
    if (ids_are_64) embedding_bwd_few_kernel<int64_t, TI, TO><<<zero_wgs + (int)T * few_slices, 256, 0, s>>>(p, ids, padding_idx, zero_wgs, zero_rows, few_slices, lanes); \
    else embedding_bwd_few_kernel<int32_t, TI, TO><<<zero_wgs + (int)T * few_slices, 256, 0, s>>>(p, ids, padding_idx, zero_wgs, zero_rows, few_slices, lanes)
        switch (types) {
            case 0: EMB_FEW(float, float); break;
            case 1: EMB_FEW(float, bf16_t); break;
            case 2: EMB_FEW(bf16_t, float); break;
            default: EMB_FEW(bf16_t, bf16_t); break;
        }
#undef EMB_FEW
        return vitk_check_launch("embedding_bwd_few");
    }
    const long long zero16 = accumulate ? 0 : (long long)V * D * (dtable_type == 0 ? 4 : 2) / 16;
    const int zero_blocks = (int)(zero16 / 4096 < 1024 ? (zero16 + 4095) / 4096 : 1024);
    const int passes = emb_passes(V);
    char* ws = (char*)workspace;
    uint2* sorted = (uint2*)ws;
    ws += emb_up((size_t)T * sizeof(uint2));
    p.sorted = sorted;
    p.piece = emb_piece(T, D);
    p.pieces = (int)((T + p.piece - 1) / p.piece);
    p.partial = (float*)ws;
    ws += emb_up((size_t)p.pieces * 2 * D * sizeof(float));
    if (emb_one(T, V)) {
        const int grid = GROUP_WG + zero_blocks;
        const size_t lds = emb_group_lds(V);
        static VitkLdsOnce once64 = {}, once32 = {};        // the largest is allowed once; a launch asks for what its vocabulary needs
        if (int rc = ids_are_64 ? vitk_lds_once(once64, (const void*)emb_group_kernel<int64_t>, emb_group_lds(1 << 18), "embedding_bwd")
                                : vitk_lds_once(once32, (const void*)emb_group_kernel<int32_t>, emb_group_lds(1 << 18), "embedding_bwd"))
            return rc;
        if (ids_are_64) emb_group_kernel<int64_t><<<grid, 1024, lds, s>>>(ids, (int)T, V, padding_idx, sorted, (uint4*)dtable, zero16);
        else emb_group_kernel<int32_t><<<grid, 1024, lds, s>>>(ids, (int)T, V, padding_idx, sorted, (uint4*)dtable, zero16);
        if (int rc = vitk_check_launch("embedding_bwd_sort")) return rc;
    } else {
        uint2* other = (uint2*)ws;
        ws += emb_up((size_t)T * sizeof(uint2));
        unsigned* counts = (unsigned*)ws;
        const int blocks = (int)emb_sort_blocks(T), groups = (int)emb_sort_groups(T), entries = groups > 0 ? groups : blocks;
        unsigned* totals = groups > 0 ? counts + (size_t)blocks * SORT_BINS : counts;
        // the last pass has to write `sorted`
        uint2* to = passes & 1 ? sorted : other;
        uint2* from = nullptr;
        for (int pass = 0; pass < passes; ++pass) {
            const int shift = pass * SORT_BITS, extra = pass == 0 ? zero_blocks : 0;
#define EMB_PASS(I, F)                                                                                                                       \
    emb_hist_kernel<I, F><<<blocks + extra, SORT_THREADS, 0, s>>>(ids, from, T, V, padding_idx, shift, counts, blocks, (uint4*)dtable, zero16);      \
    if (groups > 0) emb_scan_kernel<<<groups, SORT_BINS, 0, s>>>(counts, blocks, totals);                                                    \
    emb_scatter_kernel<I, F><<<blocks, SORT_THREADS, 0, s>>>(ids, from, T, V, padding_idx, shift, counts, totals, entries, to)
            if (pass > 0) { EMB_PASS(int64_t, false); }
            else if (ids_are_64) { EMB_PASS(int64_t, true); }
            else { EMB_PASS(int32_t, true); }
#undef EMB_PASS
            if (int rc = vitk_check_launch("embedding_bwd_sort")) return rc;
            from = to;
            to = to == sorted ? other : sorted;
        }
    }
    const int lanes = emb_lanes(D), side = lanes < 64 ? 256 / lanes : 1, slices = (D / 8 + lanes - 1) / lanes;
    const dim3 block(lanes, side), grid((p.pieces + side - 1) / side, slices);
#define EMB_BWD(TI, TO)                                                                                                            \
    embedding_bwd_kernel<TI, TO><<<grid, block, 0, s>>>(p);                                                                        \
    if (p.pieces > 1 && side > 1) embedding_join_kernel<TO, 1><<<grid, block, 0, s>>>(p);                                          \
    else if (p.pieces > 1) embedding_join_kernel<TO, 4><<<dim3(p.pieces - 1, slices), dim3(lanes, 4), 0, s>>>(p)
    switch (types) {
        case 0: EMB_BWD(float, float); break;
        case 1: EMB_BWD(float, bf16_t); break;
        case 2: EMB_BWD(bf16_t, float); break;
        default: EMB_BWD(bf16_t, bf16_t); break;
    }
#undef EMB_BWD
    return vitk_check_launch("embedding_bwd");
}

}  // extern "C"
