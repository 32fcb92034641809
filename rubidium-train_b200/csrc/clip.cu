// clip.cu — the global gradient norm over many tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2) / scale,   out = g min(1, max_norm / norm)
//
// Memory bound: the gradients are read for the norm, and where clipping bites (or out is not g) read again
// and written.  Two launches, ordered by programmatic dependent launch: every block of the first leaves the
// FP64 sum of its chunks, every block of the second adds those sums in the same order and scales its chunks.
// 163 M FP32 gradients (652 MB), out of place: 323 us, of which 303 are its bytes at the rate of a copy; 48 tensors
// of 48 KB: 5.2 us.
// The tensors' addresses travel as kernel parameters, so the call copies nothing to the device and can be
// captured into a graph.
//
// A tensor is cut into chunks of 16 KB whose borders lie on 16-byte boundaries of g: whatever g's alignment, all
// its vectors but the first and the last are whole.  The blocks take the chunks in turn, so that they stream through
// the same stretch of memory together (each its own run of neighbours: 338 us against 323); a block searches the
// table for its first chunk's tensor and walks on from there.  The second kernel goes backwards.
#include <algorithm>
#include <cfloat>
#include <new>
#include <vector>

#include "common.cuh"

namespace rbk {
namespace clip {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 16 << 10;
constexpr int kVec = kChunkBytes / 16 / kThreads;        // 16-byte vectors of a chunk per thread
constexpr int kPerSm = 6;                                // blocks
constexpr int kMaxBlocks = RBK_CLIP_WS_BYTES / 8;        // FP64 sums, of all launches of a call

struct Tensor {
    const char* g;
    char* out;
    long long n;
    int first;                                           // its first chunk
    int half;
};
// As many tensors as a launch's parameters hold: 900 is 28.8 KB of the 32764 bytes.
template <int CAP>
struct Table {
    Tensor t[CAP];
    int count, chunks;
};

// The tensor of chunk c: the last one whose first chunk is <= c.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& tab, int c) {
    int lo = 0, hi = tab.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.t[mid].first <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Sum of squares of one 16-byte vector.  FP32 squares go to FP64 one by one: a square may be beyond FP32's
// range.  FP16 squares are exact in FP32 (22 bits) and eight of them stay far below its largest value.
__device__ __forceinline__ double squares(const uint4& v, int half) {
    if (half) {
        float f[8];
        h8_to_f(v, f);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(f[i], f[i], s);
        return s;
    }
    const double a = __uint_as_float(v.x), b = __uint_as_float(v.y), c = __uint_as_float(v.z), d = __uint_as_float(v.w);
    return fma(a, a, b * b) + fma(c, c, d * d);
}

// One chunk of a tensor as this thread's kVec vectors, kThreads apart: `e` is the element at which its first one
// starts (negative where the aligned span begins before g).
struct Chunk {
    long long e;
    bool whole;                                          // every vector of the chunk, of all threads
};
__device__ __forceinline__ Chunk chunk_of(const Tensor& t, int c) {
    const int ve = t.half ? 8 : 4, skip = (int)(reinterpret_cast<uintptr_t>(t.g) & 15u) / (t.half ? 2 : 4);
    const long long e0 = (long long)(c - t.first) * (kChunkBytes / 16) * ve - skip;
    return {e0 + (long long)threadIdx.x * ve, e0 >= 0 && e0 + (kChunkBytes / 16) * ve <= t.n};
}
__device__ __forceinline__ void load_chunk(uint4* v, const Tensor& t, const Chunk& k) {
    const int ve = t.half ? 8 : 4;
    if (k.whole) {
        const uint4* p = reinterpret_cast<const uint4*>(t.g + k.e * (t.half ? 2 : 4));
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = p[i * kThreads];
        return;
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {                     // the ends of a tensor, element by element: zeros outside
        const long long e = k.e + (long long)i * kThreads * ve;
        uint32_t w[4] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j >= ve || e + j < 0 || e + j >= t.n) continue;
            if (t.half) w[j / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(t.g)[e + j] << (16 * (j & 1));
            else w[j & 3] = reinterpret_cast<const uint32_t*>(t.g)[e + j];
        }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The block's sum of v in thread 0, warps in order.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double sw[kThreads / 32];
    v = warp_sum_d(v);
    if ((threadIdx.x & 31) == 0) sw[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    if (threadIdx.x == 0)
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) s += sw[w];
    return s;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table<CAP> tab, double* part) {
    grid_dependency_sync();
    double acc = 0.0;
    int c = blockIdx.x;
    for (int k = tensor_of(tab, c); c < tab.chunks; c += gridDim.x) {
        while (k + 1 < tab.count && tab.t[k + 1].first <= c) ++k;
        const Tensor& t = tab.t[k];
        uint4 v[kVec];
        load_chunk(v, t, chunk_of(t, c));
        if (t.half) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc += squares(v[i], 1);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc += squares(v[i], 0);
        }
    }
    acc = block_sum(acc);
    if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// v * coef, or with TINY v * 2^-126 * coef: a factor below FP32's normal range as two in it.  What the first product
// rounds, below 2^-126, ends below 2^-126 of that; a half is nothing there.
template <bool TINY>
__device__ __forceinline__ uint4 scaled(uint4 v, int half, float coef) {
    if (half) {
        float f[8];
        h8_to_f(v, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= TINY ? 0.0f : coef;
        return f_to_h8(f);
    }
    if (TINY) {
        v.x = __float_as_uint(__uint_as_float(v.x) * FLT_MIN);
        v.y = __float_as_uint(__uint_as_float(v.y) * FLT_MIN);
        v.z = __float_as_uint(__uint_as_float(v.z) * FLT_MIN);
        v.w = __float_as_uint(__uint_as_float(v.w) * FLT_MIN);
    }
    v.x = __float_as_uint(__uint_as_float(v.x) * coef);
    v.y = __float_as_uint(__uint_as_float(v.y) * coef);
    v.z = __float_as_uint(__uint_as_float(v.z) * coef);
    v.w = __float_as_uint(__uint_as_float(v.w) * coef);
    return v;
}
// Elements [a, b) of a vector to dst.
__device__ __forceinline__ void store_part(char* dst, const uint4& v, int half, int a, int b) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (j < a || j >= b) continue;
        if (half) reinterpret_cast<unsigned short*>(dst)[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
        else if (j < 4) reinterpret_cast<uint32_t*>(dst)[j] = w[j];
    }
}
// The 16 bytes that start s bytes (a multiple of 2, the same in all threads) into v followed by next.
__device__ __forceinline__ uint4 funnel(const uint4& v, const uint4& next, int s) {
    uint32_t a[8] = {v.x, v.y, v.z, v.w, next.x, next.y, next.z, next.w};
    if (s & 4)
#pragma unroll
        for (int k = 0; k < 7; ++k) a[k] = a[k + 1];
    if (s & 8)
#pragma unroll
        for (int k = 0; k < 6; ++k) a[k] = a[k + 2];
    if (s & 2)
#pragma unroll
        for (int k = 0; k < 5; ++k) a[k] = __funnelshift_r(a[k], a[k + 1], 16);
    return make_uint4(a[0], a[1], a[2], a[3]);
}
// A chunk to out, scaled.  out's alignment is its own: where its 16-byte vectors lie s bytes off g's, each is put
// together from two neighbouring vectors of g, the second from the next lane (lane 31 reads it again).
template <bool TINY>
__device__ __forceinline__ void store_chunk(const Tensor& t, const Chunk& k, const uint4* v, float coef) {
    const int ve = t.half ? 8 : 4, es = t.half ? 2 : 4;
    char* o = t.out + k.e * es;
    if (!k.whole) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {                 // the ends of a tensor
            const long long e = k.e + (long long)i * kThreads * ve;
            if (e + ve > 0 && e < t.n)
                store_part(o + (long long)i * kThreads * 16, v[i], t.half, (int)max(0LL, -e), (int)min((long long)ve, t.n - e));
        }
        return;
    }
    const int s = (int)(-reinterpret_cast<uintptr_t>(o) & 15u);
    if (s == 0) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) reinterpret_cast<uint4*>(o)[i * kThreads] = v[i];
        return;
    }
    if (threadIdx.x == 0) store_part(o, v[0], t.half, 0, s / es);
    const uint4* g = reinterpret_cast<const uint4*>(t.g + k.e * es);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        uint4 next;
        next.x = __shfl_down_sync(0xffffffffu, v[i].x, 1);
        next.y = __shfl_down_sync(0xffffffffu, v[i].y, 1);
        next.z = __shfl_down_sync(0xffffffffu, v[i].z, 1);
        next.w = __shfl_down_sync(0xffffffffu, v[i].w, 1);
        if (i == kVec - 1 && threadIdx.x == kThreads - 1) {
            store_part(o + (long long)i * kThreads * 16, v[i], t.half, s / es, ve);
            continue;
        }
        if ((threadIdx.x & 31) == 31) next = scaled<TINY>(g[i * kThreads + 1], t.half, coef);
        *reinterpret_cast<uint4*>(o + s + (long long)i * kThreads * 16) = funnel(v[i], next, s);
    }
}

// The chunks of a block, backwards.
template <int CAP, bool TINY>
__device__ __forceinline__ void scale_chunks(const Table<CAP>& tab, float coef) {
    int c = tab.chunks - 1 - (int)blockIdx.x;
    for (int k = c >= 0 ? tensor_of(tab, c) : 0; c >= 0; c -= gridDim.x) {
        while (tab.t[k].first > c) --k;
        const Tensor& t = tab.t[k];
        if (!t.out || (t.out == t.g && coef == 1.0f && !TINY)) continue;
        const Chunk ch = chunk_of(t, c);
        uint4 v[kVec];
        load_chunk(v, t, ch);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = scaled<TINY>(v[i], t.half, coef);
        store_chunk<TINY>(t, ch, v, coef);
    }
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kPerSm) scale_kernel(const __grid_constant__ Table<CAP> tab, const double* part,
                                                         int parts, float max_norm, const rbk_scaler* scaler,
                                                         float* norm_out) {
    __shared__ float coef_s;
    __shared__ int tiny_s;
    grid_dependency_sync();
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
    s = block_sum(s);
    if (threadIdx.x == 0) {
        const double norm = sqrt(s) / (scaler ? (double)scaler->scale : 1.0);
        // 1 too for a NaN (no comparison holds) and an infinite norm
        const bool bites = max_norm > 0.0f && norm > (double)max_norm && norm <= 1.7976931348623157e308;
        const double f = bites ? (double)max_norm / norm : 1.0;
        tiny_s = f < (double)FLT_MIN;
        coef_s = (float)(tiny_s ? f / (double)FLT_MIN : f);
        if (norm_out && blockIdx.x == 0) *norm_out = (float)norm;
    }
    __syncthreads();
    if (tiny_s) scale_chunks<CAP, true>(tab, coef_s);
    else scale_chunks<CAP, false>(tab, coef_s);
}

// Written ranges overlap nothing but the gradient they replace.
static bool disjoint(const rbk_grad* t, int count) {
    struct Range {
        uintptr_t a, b;
        bool written;
    };
    std::vector<Range> r;
    r.reserve(2 * (size_t)count);
    for (int i = 0; i < count; ++i) {
        const uintptr_t bytes = (uintptr_t)t[i].n * (t[i].half ? 2 : 4), g = (uintptr_t)t[i].g, o = (uintptr_t)t[i].out;
        if (!bytes) continue;
        r.push_back({g, g + bytes, o == g});
        if (o && o != g) r.push_back({o, o + bytes, true});
    }
    const auto by_start = [](const Range& x, const Range& y) { return x.a < y.a; };
    if (!std::is_sorted(r.begin(), r.end(), by_start)) std::sort(r.begin(), r.end(), by_start);
    uintptr_t end = 0, end_written = 0;                  // of the ranges before
    for (const Range& x : r) {
        if (x.a < (x.written ? end : end_written)) return false;
        end = std::max(end, x.b);
        if (x.written) end_written = std::max(end_written, x.b);
    }
    return true;
}

static int check(const rbk_grad* t, int count, float max_norm, const float* norm, const void* ws) {
    const char* who = "rbk_clip_grad_norm";
    RBK_REQUIRE(count >= 0, "%s: negative count", who);
    RBK_REQUIRE(t || !count, "%s: tensors is NULL", who);
    RBK_REQUIRE(norm, "%s: norm is NULL", who);
    RBK_REQUIRE(max_norm == max_norm, "%s: max_norm is NaN", who);
    RBK_REQUIRE(aligned16(ws), "%s: ws must be 16-byte aligned", who);
    long long chunks = 0;
    for (int i = 0; i < count; ++i) {
        RBK_REQUIRE(t[i].n >= 0, "%s: tensor %d has a negative size", who, i);
        RBK_REQUIRE(t[i].half == 0 || t[i].half == 1, "%s: tensor %d: half must be 0 or 1", who, i);
        RBK_REQUIRE(t[i].g || !t[i].n, "%s: tensor %d is NULL", who, i);
        const uintptr_t es = t[i].half ? 2 : 4;
        RBK_REQUIRE((uintptr_t)t[i].g % es == 0 && (uintptr_t)t[i].out % es == 0,
                    "%s: tensor %d is not aligned to its type", who, i);
        RBK_REQUIRE(t[i].n < (1LL << 40), "%s: tensor %d is too large", who, i);
        chunks += t[i].n * (long long)es / kChunkBytes + 2;
        RBK_REQUIRE(chunks < (1LL << 30), "%s: the tensors are too large", who);   // a block's next chunk fits an int
    }
    try {
        RBK_REQUIRE(disjoint(t, count), "%s: a written range overlaps another tensor", who);
    } catch (const std::bad_alloc&) {
        set_error("%s: out of host memory", who);
        return RBK_ERR_NOMEM;
    }
    return RBK_OK;
}

// The next tensors that fit one launch, from *at on.
template <int CAP>
static void fill(Table<CAP>& tab, const rbk_grad* t, int count, int* at) {
    tab.count = tab.chunks = 0;
    for (; *at < count && tab.count < CAP; ++*at) {
        const rbk_grad& s = t[*at];
        if (!s.n) continue;
        const int es = s.half ? 2 : 4;
        Tensor& d = tab.t[tab.count++];
        d.g = (const char*)s.g;
        d.out = (char*)s.out;
        d.n = s.n;
        d.half = (int)s.half;
        d.first = tab.chunks;
        const long long bytes = (long long)((uintptr_t)s.g & 15u) + s.n * es;
        tab.chunks += (int)((bytes + kChunkBytes - 1) / kChunkBytes);
    }
}

template <int CAP>
static int run(rbk_ctx* ctx, const rbk_grad* t, int count, float max_norm, const rbk_scaler* scaler, float* norm,
               double* part, cudaStream_t st) {
    static_assert(sizeof(Table<CAP>) <= 32000, "kernel parameters");
    Table<CAP> tab;
    // each launch of the first kernel has its own stretch of the sums
    const int launches = std::max(1, (count + CAP - 1) / CAP);
    const int per = std::max(1, std::min(kPerSm * ctx->num_sms, kMaxBlocks / launches));
    RBK_REQUIRE(launches * per <= kMaxBlocks, "rbk_clip_grad_norm: more than %d tensors", kMaxBlocks * CAP);
    int parts = 0;
    for (int at = 0; at < count;) {
        fill(tab, t, count, &at);
        if (!tab.chunks) continue;
        const int grid = std::min(per, tab.chunks);
        RBK_CUDA(launch_pdl(squares_kernel<CAP>, dim3(grid), dim3(kThreads), 0, st, tab, part + parts));
        RBK_LAUNCHED("squares_kernel");
        parts += grid;
    }
    int at = 0;
    do {
        fill(tab, t, count, &at);
        const int grid = std::max(1, std::min(kPerSm * ctx->num_sms, tab.chunks));
        RBK_CUDA(launch_pdl(scale_kernel<CAP>, dim3(grid), dim3(kThreads), 0, st, tab, (const double*)part, parts,
                            max_norm, scaler, norm));
        RBK_LAUNCHED("scale_kernel");
    } while (at < count);
    return RBK_OK;
}

}  // namespace clip
}  // namespace rbk

using namespace rbk;

extern "C" int rbk_clip_grad_norm(rbk_ctx* ctx, const rbk_grad* tensors, int count, float max_norm,
                                  const rbk_scaler* scaler, float* norm, void* ws, void* stream) {
    RBK_TRY(clip::check(tensors, count, max_norm, norm, ws));
    RBK_TRY(check_device(ctx, "rbk_clip_grad_norm"));
    if (!ws) RBK_TRY(ctx_scratch(ctx, RBK_CLIP_WS_BYTES, &ws));
    double bytes = 0.0;
    for (int i = 0; i < count; ++i) bytes += (tensors[i].out ? 3.0 : 1.0) * tensors[i].n * (tensors[i].half ? 2 : 4);
    ProfScope prof(ctx, as_stream(stream), kCatOther, bytes);
    // a table of the size that is needed: the parameters are copied with each launch
    if (count <= 120) return clip::run<120>(ctx, tensors, count, max_norm, scaler, norm, (double*)ws, as_stream(stream));
    return clip::run<900>(ctx, tensors, count, max_norm, scaler, norm, (double*)ws, as_stream(stream));
}
