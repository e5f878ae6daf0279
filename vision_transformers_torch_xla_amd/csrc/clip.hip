// Global L2 norm of many gradient tensors of mixed types, and clipping by it: N = sqrt(sum g^2), c = min(1, max_norm / (N + 1e-6)),
// out = c * g.  HBM-bound: every gradient is read once for the norm and, where anything is scaled or copied, once more and written.
//
// The tensor list travels in the kernel arguments (no device table, so nothing is uploaded, kept between calls or tied to an address,
// and a captured graph holds its own copy): up to MT_MAX tensors per launch, cut into chunks of MT_CHUNK elements that the blocks of
// the launch walk in a fixed order.  Two stages: partial sums of squares (one double per block), then every block of the second stage
// adds all partials up in the same order - the same bits in every block, on every run - and scales its chunks.  No atomics.
// Squares are formed and summed in double: the square of any finite fp32 / bf16 / fp16 value is representable, so the norm neither
// overflows nor vanishes where sums in float would, at the same speed (the loads are what the kernel waits for).
#include "common.h"

#define MT_MAX 180             // what 4 KB of arguments hold (128 with an 8-byte count each: 152 tensors took 14 us more in two launches a stage)
#define MT_CHUNK 8192          // elements per chunk: 32 per thread
#define MT_BLOCKS 2048         // blocks of a launch at most: 8 per compute unit

enum { MT_F32 = 0, MT_BF16 = 1, MT_F16 = 2 };

struct MtList {
    const void* src[MT_MAX];
    void* dst[MT_MAX];
    unsigned first[MT_MAX + 1];             // first chunk of each tensor; first[count] = chunks of this launch
    unsigned short tail_type[MT_MAX];       // elements of the last chunk less one, type from bit 13 on
    int count;
};
static_assert(MT_CHUNK <= 1 << 13 && sizeof(MtList) <= 4000, "kernel arguments are limited to 4 KB");

static __device__ __forceinline__ int mt_find(const MtList& l, unsigned chunk) {
    int lo = 0, hi = l.count - 1;           // largest t with first[t] <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

static __device__ __forceinline__ float mt_half(unsigned short u) { return (float)__builtin_bit_cast(_Float16, u); }
static __device__ __forceinline__ unsigned short mt_to_half(float f) { return __builtin_bit_cast(unsigned short, (_Float16)f); }
static __device__ __forceinline__ float mt_load(const void* p, int type, size_t i) {
    if (type == MT_F32) return reinterpret_cast<const float*>(p)[i];
    const unsigned short u = reinterpret_cast<const unsigned short*>(p)[i];
    return type == MT_BF16 ? bf2f(u) : mt_half(u);
}
static __device__ __forceinline__ void mt_store(void* p, int type, size_t i, float v) {
    if (type == MT_F32) reinterpret_cast<float*>(p)[i] = v;
    else reinterpret_cast<unsigned short*>(p)[i] = type == MT_BF16 ? f2bf(v) : mt_to_half(v);
}
static __device__ __forceinline__ double mt_block_sum(double v, double* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    const double s = sh[0] + sh[1] + sh[2] + sh[3];
    __syncthreads();
    return s;
}

// four (fp32) or eight (16-bit) consecutive values from a 16-byte aligned address
static __device__ __forceinline__ int mt_unpack(const uint4 r, int type, float (&v)[8]) {
    if (type == MT_F32) {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
        return 4;
    }
    const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (type == MT_BF16) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        else { v[2 * i] = mt_half((unsigned short)w[i]); v[2 * i + 1] = mt_half((unsigned short)(w[i] >> 16)); }
    }
    return 8;
}
static __device__ __forceinline__ uint4 mt_pack(const float (&v)[8], int type) {
    uint4 r;
    if (type == MT_F32) { r.x = __float_as_uint(v[0]); r.y = __float_as_uint(v[1]); r.z = __float_as_uint(v[2]); r.w = __float_as_uint(v[3]); return r; }
    if (type == MT_BF16) return pack8_bf16(v);
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (unsigned)mt_to_half(v[2 * i]) | ((unsigned)mt_to_half(v[2 * i + 1]) << 16);
    r.x = w[0]; r.y = w[1]; r.z = w[2]; r.w = w[3];
    return r;
}

template <int TYPE>
static __device__ __forceinline__ double mt_chunk_sumsq(const void* src, size_t at, int n) {
    constexpr int W = TYPE == MT_F32 ? 4 : 8, SIZE = TYPE == MT_F32 ? 4 : 2;
    const char* base = reinterpret_cast<const char*>(src) + at * SIZE;
    double s = 0.0;
    if ((reinterpret_cast<size_t>(base) & 15) != 0) {        // a view that starts between 16-byte lines
        for (int i = threadIdx.x; i < n; i += 256) { const double v = mt_load(base, TYPE, i); s += v * v; }
        return s;
    }
    const uint4* p = reinterpret_cast<const uint4*>(base);
    if (n == MT_CHUNK) {
        constexpr int R = MT_CHUNK / (256 * W);
        uint4 r[R];
#pragma unroll
        for (int j = 0; j < R; ++j) r[j] = p[j * 256 + threadIdx.x];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float v[8];
            mt_unpack(r[j], TYPE, v);
#pragma unroll
            for (int k = 0; k < W; ++k) s += (double)v[k] * (double)v[k];
        }
        return s;
    }
    const int full = n / W;
    for (int i = threadIdx.x; i < full; i += 256) {
        float v[8];
        mt_unpack(p[i], TYPE, v);
#pragma unroll
        for (int k = 0; k < W; ++k) s += (double)v[k] * (double)v[k];
    }
    for (int i = full * W + threadIdx.x; i < n; i += 256) { const double v = mt_load(base, TYPE, i); s += v * v; }
    return s;
}

__global__ __launch_bounds__(256) void mt_sumsq_kernel(const MtList l, double* __restrict__ partial) {
    __shared__ double sh[4];
    double s = 0.0;
    const unsigned chunks = l.first[l.count];
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = mt_find(l, c);
        const int type = (int)(l.tail_type[t] >> 13);
        const size_t at = (size_t)(c - l.first[t]) * MT_CHUNK;
        const int m = c + 1 == l.first[t + 1] ? (int)(l.tail_type[t] & 8191) + 1 : MT_CHUNK;
        if (type == MT_F32) s += mt_chunk_sumsq<MT_F32>(l.src[t], at, m);
        else if (type == MT_BF16) s += mt_chunk_sumsq<MT_BF16>(l.src[t], at, m);
        else s += mt_chunk_sumsq<MT_F16>(l.src[t], at, m);
    }
    s = mt_block_sum(s, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

typedef __attribute__((ext_vector_type(4))) unsigned mt_u32x4;
template <int TYPE>
static __device__ __forceinline__ void mt_chunk_scale(const void* src, void* dst, size_t at, int n, float coef, bool stream) {
    constexpr int W = TYPE == MT_F32 ? 4 : 8, SIZE = TYPE == MT_F32 ? 4 : 2;
    const char* a = reinterpret_cast<const char*>(src) + at * SIZE;
    char* b = reinterpret_cast<char*>(dst) + at * SIZE;
    if (((reinterpret_cast<size_t>(a) | reinterpret_cast<size_t>(b)) & 15) != 0) {
        for (int i = threadIdx.x; i < n; i += 256) mt_store(b, TYPE, i, mt_load(a, TYPE, i) * coef);
        return;
    }
    const uint4* p = reinterpret_cast<const uint4*>(a);
    uint4* q = reinterpret_cast<uint4*>(b);
    if (n == MT_CHUNK) {
        constexpr int R = MT_CHUNK / (256 * W);
        uint4 r[R];
#pragma unroll
        for (int j = 0; j < R; ++j) r[j] = p[j * 256 + threadIdx.x];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float v[8];
            mt_unpack(r[j], TYPE, v);
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] *= coef;
            // into other tensors: past the caches, which keep the gradients that are still to be read (152 tensors of 22 M values 57.8 -> 48.8 us,
            // 400 of 600 M 1002 -> 968 us)
            const uint4 w = mt_pack(v, TYPE);
            if (stream) __builtin_nontemporal_store((mt_u32x4){w.x, w.y, w.z, w.w}, reinterpret_cast<mt_u32x4*>(q) + j * 256 + threadIdx.x);
            else q[j * 256 + threadIdx.x] = w;
        }
        return;
    }
    const int full = n / W;
    for (int i = threadIdx.x; i < full; i += 256) {
        float v[8];
        mt_unpack(p[i], TYPE, v);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] *= coef;
        q[i] = mt_pack(v, TYPE);
    }
    for (int i = full * W + threadIdx.x; i < n; i += 256) mt_store(b, TYPE, i, mt_load(a, TYPE, i) * coef);
}

// the total of the partial sums, in the same order in every block
static __device__ __forceinline__ float mt_norm(const double* partial, int nparts, double* sh) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += partial[i];
    return (float)sqrt(mt_block_sum(s, sh));
}

__global__ __launch_bounds__(256) void mt_scale_kernel(const MtList l, const double* __restrict__ partial, int nparts, float max_norm,
                                                       float* __restrict__ norm_out, int in_place) {
    __shared__ double sh[4];
    const float norm = mt_norm(partial, nparts, sh);
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float coef = max_norm / (norm + 1e-6f);
    if (coef > 1.0f) coef = 1.0f;                   // NaN stays NaN, an infinite norm gives 0 (and NaN where the gradient is infinite)
    if (in_place && coef == 1.0f) return;
    const unsigned chunks = l.first[l.count];
    for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = mt_find(l, c);
        const int type = (int)(l.tail_type[t] >> 13);
        const size_t at = (size_t)(c - l.first[t]) * MT_CHUNK;
        const int m = c + 1 == l.first[t + 1] ? (int)(l.tail_type[t] & 8191) + 1 : MT_CHUNK;
        if (type == MT_F32) mt_chunk_scale<MT_F32>(l.src[t], l.dst[t], at, m, coef, !in_place);
        else if (type == MT_BF16) mt_chunk_scale<MT_BF16>(l.src[t], l.dst[t], at, m, coef, !in_place);
        else mt_chunk_scale<MT_F16>(l.src[t], l.dst[t], at, m, coef, !in_place);
    }
}

__global__ __launch_bounds__(256) void mt_norm_kernel(const double* __restrict__ partial, int nparts, float* __restrict__ norm_out) {
    __shared__ double sh[4];
    const float norm = mt_norm(partial, nparts, sh);
    if (threadIdx.x == 0) *norm_out = norm;
}

// the launch that starts at tensor `from`: fills l, returns the tensor after its last one; empty tensors take no chunk
static int mt_fill(MtList& l, const void* const* src, void* const* dst, const int64_t* numel, const int* type, int count, int from) {
    l.count = 0;
    unsigned long long chunks = 0;
    int t = from;
    for (; t < count && l.count < MT_MAX; ++t) {
        if (numel[t] == 0) continue;
        const unsigned long long c = ((unsigned long long)numel[t] + MT_CHUNK - 1) / MT_CHUNK;
        if (chunks + c > 0xf0000000ull) break;
        l.src[l.count] = src[t];
        l.dst[l.count] = dst ? dst[t] : nullptr;
        l.tail_type[l.count] = (unsigned short)(((unsigned long long)(numel[t] - 1) % MT_CHUNK) | ((unsigned)type[t] << 13));
        l.first[l.count] = (unsigned)chunks;
        chunks += c;
        ++l.count;
    }
    l.first[l.count] = (unsigned)chunks;
    return t;
}
static int mt_grid(const MtList& l) {
    const unsigned chunks = l.first[l.count];
    return chunks < MT_BLOCKS ? (int)chunks : MT_BLOCKS;
}

extern "C" {

size_t vitk_clip_grads_workspace(int count) {
    if (count <= 0) return 0;
    return (size_t)((count + MT_MAX - 1) / MT_MAX + 1) * MT_BLOCKS * sizeof(double);
}

int vitk_clip_grads(const void* const* src, void* const* dst, const int64_t* numel, const int* type, int count, float max_norm,
                    float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    VITK_REQUIRE(count >= 0 && norm && workspace && vitk_aligned(workspace, 8), "clip_grads: null pointer or negative count");
    VITK_REQUIRE(count == 0 || (src && numel && type), "clip_grads: null tensor table");
    VITK_REQUIRE(!dst || max_norm >= 0.f, "clip_grads: max_norm must not be negative (and not NaN)");
    for (int t = 0; t < count; ++t) {
        VITK_REQUIRE(type[t] >= MT_F32 && type[t] <= MT_F16, "clip_grads: tensor %d: type %d (0 fp32, 1 bf16, 2 fp16)", t, type[t]);
        VITK_REQUIRE(numel[t] >= 0 && numel[t] < (1ll << 44), "clip_grads: tensor %d has %lld elements", t, (long long)numel[t]);
        const size_t size = type[t] == MT_F32 ? 4 : 2;
        VITK_REQUIRE(numel[t] == 0 || (src[t] && vitk_aligned(src[t], size) && (!dst || (dst[t] && vitk_aligned(dst[t], size)))),
                     "clip_grads: tensor %d: null or misaligned pointer", t);
    }
    if (workspace_bytes < vitk_clip_grads_workspace(count > 0 ? count : 1)) {
        vitk_set_error("clip_grads: workspace %zu < %zu", workspace_bytes, vitk_clip_grads_workspace(count > 0 ? count : 1));
        return VITK_ENOSPC;
    }
    hipStream_t s = (hipStream_t)stream;
    double* partial = (double*)workspace;
    const int room = (int)(workspace_bytes / sizeof(double) < 0x7fffffff ? workspace_bytes / sizeof(double) : 0x7fffffff);
    MtList l;
    int nparts = 0;
    for (int from = 0; from < count;) {
        from = mt_fill(l, src, dst, numel, type, count, from);
        if (l.count == 0) break;
        const int grid = mt_grid(l);
        VITK_REQUIRE(nparts + grid <= room, "clip_grads: the tensors are too large for %d partial sums", room);
        mt_sumsq_kernel<<<grid, 256, 0, s>>>(l, partial + nparts);
        if (int rc = vitk_check_launch("clip_grads_sumsq")) return rc;
        nparts += grid;
    }
    if (dst == nullptr || nparts == 0) {
        mt_norm_kernel<<<1, 256, 0, s>>>(partial, nparts, norm);
        return vitk_check_launch("clip_grads_norm");
    }
    float* out = norm;
    for (int from = 0; from < count;) {
        from = mt_fill(l, src, dst, numel, type, count, from);
        if (l.count == 0) break;
        int in_place = 1;
        for (int t = 0; t < l.count; ++t) in_place &= l.src[t] == l.dst[t];
        mt_scale_kernel<<<mt_grid(l), 256, 0, s>>>(l, partial, nparts, max_norm, out, in_place);
        if (int rc = vitk_check_launch("clip_grads_scale")) return rc;
        out = nullptr;
    }
    return VITK_OK;
}

}  // extern "C"
