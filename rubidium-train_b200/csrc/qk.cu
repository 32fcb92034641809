// qk.cu — per-head RMS normalisation of queries and keys and the rotary position
// embedding in one pass over the heads, and its backward.
//
//   xhat = x rstd, rstd = 1 / sqrt(mean x^2 + eps);  z = gain xhat;  y = R z
//   R rotates pair i of a head by t_i = p f_i:  (a, b) -> (a cos - b sin, a sin + b cos)
// Backward, with d = R^T dy (the rotation by -t) and w = gain d:
//   dgain = sum over all rows of d xhat,   dx = rstd (w - xhat mean(w xhat))
// Both sums of a row, of x^2 and of w x, are over the head as it was read, so the
// backward needs no statistics from the forward.
//
// Memory bound: 4 bytes per element forward, 6 backward, each touched once.  16384 tokens, 16 + 16 heads of
// 128: forward 45.7 us = 5880 GB/s, backward 65.4 us = 6160 GB/s (0.91 and 0.95 of a copy's rate); 16384
// tokens, 12 + 12 heads of 64: backward 27.5 us = 5490 GB/s; 32 tokens forward: 2.8 us, a launch.  These are replays
// from a graph; a stream of calls, whose clock is lower, takes 50.6, 73.7 and 31.4 us (0.82, 0.85 and 0.75 of a copy's
// rate): three in five issue slots are taken.  Few heads and odd widths are bound by their instructions: 65740 tokens,
// 3 + 3 heads of 80, backward 54 us = 3500 GB/s, and its 128 registers spill 16 bytes (the backwards of 3, 5, 6, 10 and
// 16 lanes all spill, 4 to 48 bytes, of 2, 4 and 8 lanes some, 4 to 12).
// Layout: a head is split over G lanes (dh / 16, or the next of 8, 10 and 16), a lane holding two
// 16-byte chunks of it, chosen so that both members of every rotated pair are in the
// same lane: no exchange is needed for the rotation.  A warp, or each half of one (T = 2,
// where fewer lanes then idle: 12 heads of 64 are 3 full steps of 4 for two tokens and not one
// full and one half step of 8), works on the heads of one token, so a token's angles are
// computed once for all of its heads, each by one of the lanes that need it (they get it by
// shuffle).  Each lane copies its vectors of the
// warp's next steps, across tokens too, into slots of its own in shared memory with cp.async
// and waits for its own copies only: no barrier, and no registers for what is in flight (with
// the next step's vectors in registers the same forward took 55.6 us, the backward 93.2).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "index.cuh"
#include "tc.cuh"

namespace rbk {
namespace qk {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxDh = 256;
constexpr int kMaxParts = 32;                // warps that share a token's heads
constexpr int kMaxRows = 1024;               // partial rows of the gain gradients (RBK_QK_BWD_WS_BYTES)

struct Heads {                               // strides in 16-byte vectors
    uint4* p;
    int sb, ss, sh;
};
struct Side {                                // the queries or the keys
    int H;
    int parts, heads_per_part;               // a warp takes heads_per_part heads of one token at a time
    Heads x, o, dy;
    const half* gain;
};
struct Params {
    Side side[2];
    int tokens, S, dh, rot, interleaved;
    uint32_t s_mul, s_shift;                 // token / S = (umulhi(token, s_mul) + token) >> s_shift
    int blocks0;                             // blocks [0, blocks0) work on side 0, the others on side 1
    float eps, inv_dh;
    const int* pos;
    int pos0;
    float* part;                             // [gridDim.x][dh] partial gain gradients (backward)
    unsigned long long freq[kMaxDh / 2];     // fractions of a turn per position, 2^-64; zero where nothing rotates
};

// cos and sin of position p's angle for a frequency of `freq` 2^-64 turns per position.  The product wraps
// modulo 2^64 = modulo a turn, exactly; its top 32 bits, rounded, are the angle to 2^-32 turns.  Split into the
// nearest quarter turn and a rest of at most an eighth, x = 2 pi rest <= pi / 4, whose sine and cosine are Taylor
// sums (the first terms left out: x^11 / 11! < 2^-28, x^10 / 10! < 2^-25).
__device__ __forceinline__ void turn(int p, unsigned long long freq, float& c, float& s) {
    const unsigned long long t = (unsigned long long)(long long)p * freq + 0x80000000ull;
    const uint32_t u = (uint32_t)(t >> 32), q = (u + 0x20000000u) >> 30;
    const float x = (float)(int)(u - (q << 30)) * 1.4629180792671596e-9f;   // 2 pi 2^-32
    const float z = x * x;
    const float sx = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), x);
    const float cx = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 40320.0f, -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
    const float a = q & 1 ? sx : cx, b = q & 1 ? cx : sx;
    c = __uint_as_float(__float_as_uint(a) ^ ((q + 1) << 30 & 0x80000000u));   // minus in quarters 1 and 2
    s = __uint_as_float(__float_as_uint(b) ^ (q << 30 & 0x80000000u));         // minus in quarters 2 and 3
}
__device__ __forceinline__ float rsqrt_fast(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a lane holds of a head: chunks (8 channels, one vector each) a and b, each neighbours of the next lane's.
struct Lane {
    int a, b;
    bool has_a, has_b, rot_a, rot_b;
    int fa, fb;                              // the frequencies of its first and its last four pairs start here
};
__device__ __forceinline__ Lane lane_of(const Params& p, int j) {
    Lane l;
    const int chunks = p.dh >> 3, rs = p.rot >> 4;
    if (p.interleaved) {                     // pairs within a chunk
        l.a = j;
        l.b = j + ((chunks + 1) >> 1);
        l.has_a = l.a < (chunks + 1) >> 1;
        l.rot_a = l.a < (p.rot >> 3);
        l.rot_b = l.b < (p.rot >> 3);
        l.fa = 4 * l.a;
        l.fb = 4 * l.b;
    } else {                                 // rs chunks and their partners, then those that do not turn
        const int half = (chunks - 2 * rs + 1) >> 1, t = j - rs;
        l.a = j < rs ? j : 2 * rs + t;
        l.b = j < rs ? j + rs : 2 * rs + half + t;
        l.has_a = j < rs || t < half;
        l.rot_a = l.rot_b = j < rs;
        l.fa = 8 * j;
        l.fb = 8 * j + 4;
    }
    l.has_b = l.has_a && l.b < chunks;
    return l;
}

using tc::lo2;
using tc::hi2;
using tc::pk2;
using tc::padd2;
using tc::psub2;
using tc::pmul2;
using tc::pfma2;

// What a lane holds of a head: packed pairs of neighbouring channels, 0..3 of chunk a, 4..7 of chunk b.
struct Row {
    uint64_t v[8];
};

// The rotation, or with T its transpose, of a lane's channels by cs = cosines and sn = sines: packed like the
// channels when pairs are half a rotation apart, (pair 2i, pair 2i + 1) when they are neighbours.
template <bool INTER, bool T>
__device__ __forceinline__ void rotate(const Lane& l, Row& r, const uint64_t* cs, const uint64_t* sn) {
    if constexpr (INTER) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < 4 ? !l.rot_a : !l.rot_b) continue;
            const float x = lo2(r.v[i]), y = hi2(r.v[i]);
            const float c = i & 1 ? hi2(cs[i / 2]) : lo2(cs[i / 2]), s = i & 1 ? hi2(sn[i / 2]) : lo2(sn[i / 2]);
            r.v[i] = T ? pk2(fmaf(y, s, x * c), fmaf(-x, s, y * c)) : pk2(fmaf(-y, s, x * c), fmaf(x, s, y * c));
        }
    } else if (l.rot_a) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t a = r.v[i], b = r.v[4 + i];
            if (T) {
                r.v[i] = pfma2(b, sn[i], pmul2(a, cs[i]));
                r.v[4 + i] = psub2(pmul2(b, cs[i]), pmul2(a, sn[i]));
            } else {
                r.v[i] = psub2(pmul2(a, cs[i]), pmul2(b, sn[i]));
                r.v[4 + i] = pfma2(a, sn[i], pmul2(b, cs[i]));
            }
        }
    }
}

__device__ __forceinline__ uint4 load8(const uint4* p, bool on) { return on ? *p : make_uint4(0, 0, 0, 0); }
// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const uint4* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}
// The sum over the G lanes of this lane's group.  G a power of two: a butterfly.  Else running sums over the next
// 2, 4, .. lanes of the group, in a circle, put together to G: each lane adds in an order of its own.
template <int G>
__device__ __forceinline__ float group_sum(float v, int j) {
    if constexpr ((G & (G - 1)) == 0) {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    } else {
        const int lane = threadIdx.x & 31;
        auto ahead = [&](float x, int o) { return __shfl_sync(0xffffffffu, x, j + o < G ? lane + o : lane + o - G); };
        float sum = 0.0f;
        int done = 0;                                               // lanes in sum
#pragma unroll
        for (int n = 1; n <= G; n <<= 1) {                          // v: the next n lanes
            if (G & n) {
                sum = done ? sum + ahead(v, done) : v;
                done += n;
            }
            if (2 * n <= G) v += ahead(v, n);
        }
        return sum;
    }
}

// Blocks of an SM, steps in flight and a step's bytes of a warp.  16 warps at 128 registers with 5 steps under way
// (backward: 2 of twice the bytes); heads of 128, forward, one token a warp: 24 warps at 78 registers with 3 under
// way, which is 45.8 us against 50.6 for 16384 tokens of 16 + 16 heads.  The other forwards are bound by their
// instructions and lose at 80 registers: one head of 256 on each side 80 us against 41, 12 + 4 heads of 200 56
// against 38, 12 + 12 of 64 alike.
constexpr int per_sm(int lanes, int T, bool bwd) { return !bwd && lanes == 8 && T == 1 ? 3 : 2; }
template <int G, int T, bool BWD>
struct Flight {
    static constexpr int PER_SM = per_sm(G, T, BWD);
    static constexpr int DEPTH = BWD ? 3 : PER_SM == 3 ? 4 : 6;
    static constexpr int STEP = 32 * 16 * (BWD ? 4 : 2);
    static constexpr int SMEM = kWarps * DEPTH * STEP;
};
static_assert(kWarps * 32 * 16 * 4 <= Flight<1, 1, true>::SMEM, "the gain gradients' sums, at most 16 per lane, reuse it");

template <int G, int T, bool INTER, bool BWD>
__global__ void __launch_bounds__(kThreads, per_sm(G, T, BWD)) qk_kernel(const __grid_constant__ Params p) {
    constexpr int HPS = 32 / T / G;                                 // heads of a token per step
    constexpr int ANG = (8 + HPS - 1) / HPS;                        // angles that a lane computes of its slot's 8
    constexpr bool POW2 = (G & (G - 1)) == 0;                       // else some lanes are in no group
    constexpr int DEPTH = Flight<G, T, BWD>::DEPTH, STEP = Flight<G, T, BWD>::STEP;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int which = (int)blockIdx.x >= p.blocks0;
    const Side& sd = p.side[which];
    const int w = (which ? blockIdx.x - p.blocks0 : blockIdx.x) * kWarps + warp;
    const int stride = T * max(1, (int)(which ? gridDim.x - p.blocks0 : p.blocks0) * kWarps / sd.parts);   // tokens of a round
    const int g = lane % (32 / T) / G, j = lane % (32 / T) % G, sub = lane / (32 / T);
    const Lane l = lane_of(p, j);
    const uint32_t slot = tc::su32(smem) + warp * (DEPTH * STEP) + lane * 16;
    unsigned long long freq[ANG];
#pragma unroll
    for (int i = 0; i < ANG; ++i) {
        const int k = min(g * ANG + i, 7);
        freq[i] = p.freq[min(k < 4 ? l.fa + k : l.fb + k - 4, kMaxDh / 2 - 1)];
    }
    grid_dependency_sync();

    Row gain;
    {
        const uint4 one = make_uint4(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u);
        const uint4* gp = reinterpret_cast<const uint4*>(sd.gain);
        tc::h8_to_p(gp ? load8(gp + l.a, l.has_a) : one, gain.v);
        tc::h8_to_p(gp ? load8(gp + l.b, l.has_b) : one, gain.v + 4);
    }
    Row acc = {};                                                   // gain gradient

    const int part = w % sd.parts, h0 = part * sd.heads_per_part + g;
    const int h1 = min(sd.H, (part + 1) * sd.heads_per_part) + g;   // a lane's heads: h0, h0 + HPS .. below h1
    const int ab = l.b - l.a;
    // the warp's token, or its first one: lanes with sub = 1 work on the next, if there is one
    int token = T * (w / sd.parts) < stride ? T * (w / sd.parts) : p.tokens, h = h0;
    auto next = [&](int tk) { return p.tokens - tk > stride ? tk + stride : p.tokens; };
    auto row_of = [&](int tk) { return (int)((__umulhi((uint32_t)tk, p.s_mul) + (uint32_t)tk) >> p.s_shift); };
    auto at = [&](const Heads& t, int tk) {                         // this lane's chunk a of head h0
        tk = token_at(tk, sub, p.tokens);
        const int bi = row_of(tk), si = tk - bi * p.S;
        return t.p + ((long long)bi * t.sb + (long long)si * t.ss + (long long)h0 * t.sh + l.a);
    };
    auto pos_of = [&](int tk) {
        tk = token_at(tk, sub, p.tokens);
        return p.pos ? p.pos[tk] : p.pos0 + (tk - row_of(tk) * p.S);
    };
    // whether this lane has head hd of token tk (+ sub)
    auto has = [&](int tk, int hd) { return hd < sd.H && (T == 1 || tk + sub < p.tokens) && (POW2 || g < HPS); };

    // The copies run DEPTH - 1 steps ahead of the work: token ft, head fh.
    int ft = token, fh = h0, fs = 0;
    const uint4 *xp = nullptr, *ep = nullptr;
    auto fetch = [&] {
        if (ft < p.tokens) {
            if (fh == h0) {
                xp = at(sd.x, ft);
                if (BWD) ep = at(sd.dy, ft);
            }
            const uint32_t d = slot + fs * STEP;
            const bool on = has(ft, fh);
            copy16(d, xp, on && l.has_a);
            copy16(d + 512, xp + ab, on && l.has_b);
            xp += HPS * (long long)sd.x.sh;
            if (BWD) {
                copy16(d + 1024, ep, on && l.has_a);
                copy16(d + 1536, ep + ab, on && l.has_b);
                ep += HPS * (long long)sd.dy.sh;
            }
            fh += HPS;
            if (fh >= h1) {                                         // the same in all lanes
                ft = next(ft);
                fh = h0;
            }
        }
        fs = fs + 1 == DEPTH ? 0 : fs + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) fetch();
    uint4* op = nullptr;
    int cur = 0, pos = token < p.tokens ? pos_of(token) : 0;
    uint64_t cs[4], sn[4];
    while (token < p.tokens) {
        if (h == h0) {                                              // a new token: its angles
            op = at(sd.o, token);
            float c[ANG], s[ANG];
#pragma unroll
            for (int i = 0; i < ANG; ++i) turn(pos, freq[i], c[i], s[i]);
            pos = pos_of(next(token));
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int s0 = sub * (32 / T) + i / ANG * G + j, s1 = sub * (32 / T) + (i + 1) / ANG * G + j;
                cs[i / 2] = pk2(__shfl_sync(0xffffffffu, c[i % ANG], s0), __shfl_sync(0xffffffffu, c[(i + 1) % ANG], s1));
                sn[i / 2] = pk2(__shfl_sync(0xffffffffu, s[i % ANG], s0), __shfl_sync(0xffffffffu, s[(i + 1) % ANG], s1));
            }
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
        const uint32_t d = slot + cur * STEP;
        cur = cur + 1 == DEPTH ? 0 : cur + 1;
        Row x, e;
        tc::h8_to_p(lds16(d), x.v);
        tc::h8_to_p(lds16(d + 512), x.v + 4);
        if (BWD) {
            tc::h8_to_p(lds16(d + 1024), e.v);
            tc::h8_to_p(lds16(d + 1536), e.v + 4);
        }
        fetch();                                                    // into the slot of the step before

        uint64_t ss = 0;                                            // two zeros
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = pfma2(x.v[i], x.v[i], ss);
        if constexpr (!BWD) {
            const float rstd = rsqrt_fast(group_sum<G>(lo2(ss) + hi2(ss), j) * p.inv_dh + p.eps);
            const uint64_t r2 = pk2(rstd, rstd);
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = pmul2(pmul2(x.v[i], r2), gain.v[i]);
            rotate<INTER, false>(l, x, cs, sn);
        } else {
            rotate<INTER, true>(l, e, cs, sn);
            // d in e: m = d x gives both sums, sum of w x = m gain and the gain gradient's d xhat = m rstd
            Row m;
            uint64_t wx = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m.v[i] = pmul2(e.v[i], x.v[i]);
                wx = pfma2(m.v[i], gain.v[i], wx);
                e.v[i] = pmul2(e.v[i], gain.v[i]);                   // w
            }
            const float rstd = rsqrt_fast(group_sum<G>(lo2(ss) + hi2(ss), j) * p.inv_dh + p.eps);
            // dx = rstd w - x rstd^2 mean(w xhat)
            const float t = -group_sum<G>(lo2(wx) + hi2(wx), j) * p.inv_dh * rstd * rstd * rstd;
            const uint64_t r2 = pk2(rstd, rstd), t2 = pk2(t, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc.v[i] = pfma2(m.v[i], r2, acc.v[i]);
                x.v[i] = pfma2(x.v[i], t2, pmul2(e.v[i], r2));
            }
        }
        const bool on = has(token, h);
        if (on && l.has_a) op[0] = tc::p_to_h8(x.v);
        if (on && l.has_b) op[ab] = tc::p_to_h8(x.v + 4);
        op += HPS * (long long)sd.o.sh;
        h += HPS;
        if (h >= h1) {                                              // the same in all lanes
            token = next(token);
            h = h0;
        }
    }
    if constexpr (BWD) {
        // lanes of the same slot, then the warps, in a fixed order
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                                            // the slots are free
        constexpr int ROWS = POW2 ? 1 : T * HPS;                    // of sums that a warp leaves
        auto acc_s = reinterpret_cast<float(*)[16 * G]>(smem);      // [kWarps * ROWS]
        const int row = POW2 ? warp : warp * ROWS + sub * HPS + g;
        const bool keeps = POW2 ? lane < G : g < HPS;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = lo2(acc.v[i]), b = hi2(acc.v[i]);
            if constexpr (POW2) {
#pragma unroll
                for (int o = G; o < 32; o <<= 1) {
                    a += __shfl_xor_sync(0xffffffffu, a, o);
                    b += __shfl_xor_sync(0xffffffffu, b, o);
                }
            }
            const int c = i < 4 ? 8 * l.a + 2 * i : 8 * l.b + 2 * (i - 4);
            if (keeps && (i < 4 ? l.has_a : l.has_b)) {
                acc_s[row][c] = a;
                acc_s[row][c + 1] = b;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.dh; c += kThreads) {
            float v = 0.0f;
#pragma unroll 8
            for (int w = 0; w < kWarps * ROWS; ++w) v += acc_s[w][c];
            p.part[(size_t)blockIdx.x * p.dh + c] = v;
        }
    }
}

// dgain[c] (+)= sum over the side's partial rows: a block takes 32 channels, its warps every eighth row, and the
// warps' sums are added in order.  Latency bound (up to 296 rows of 1 KB): about 3 us behind the main kernel.
__global__ void __launch_bounds__(kThreads) qk_gain_kernel(float* dgq, float* dgk, const float* part, int dh, int rows0,
                                                           int rows, int accumulate) {
    __shared__ float s[kWarps][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ch = blockIdx.x * 32 + lane;
    const int which = blockIdx.y;
    float* out = which ? dgk : dgq;
    grid_dependency_sync();
    float v = 0.0f;
    if (ch < dh) {
        const int end = which ? rows : rows0;
#pragma unroll 8
        for (int r = (which ? rows0 : 0) + warp; r < end; r += kWarps) v += part[(size_t)r * dh + ch];
    }
    s[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && ch < dh && out) {
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += s[w][lane];
        out[ch] = accumulate ? out[ch] + v : v;
    }
}

template <int G, int T, bool INTER, bool BWD>
cudaError_t launch_one(const Params& p, int grid, cudaStream_t st) {
    return launch_pdl(qk_kernel<G, T, INTER, BWD>, dim3(grid), dim3(kThreads), Flight<G, T, BWD>::SMEM, st, p);
}
template <int T, bool INTER, bool BWD>
int launch(const Params& p, int lanes, int grid, cudaStream_t st) {
    switch (lanes) {
        case 1: RBK_CUDA((launch_one<1, T, INTER, BWD>(p, grid, st))); break;
        case 2: RBK_CUDA((launch_one<2, T, INTER, BWD>(p, grid, st))); break;
        case 3: RBK_CUDA((launch_one<3, T, INTER, BWD>(p, grid, st))); break;
        case 4: RBK_CUDA((launch_one<4, T, INTER, BWD>(p, grid, st))); break;
        case 5: RBK_CUDA((launch_one<5, T, INTER, BWD>(p, grid, st))); break;
        case 6: RBK_CUDA((launch_one<6, T, INTER, BWD>(p, grid, st))); break;
        case 8: RBK_CUDA((launch_one<8, T, INTER, BWD>(p, grid, st))); break;
        case 10: RBK_CUDA((launch_one<10, T, INTER, BWD>(p, grid, st))); break;
        default: RBK_CUDA((launch_one<16, T, INTER, BWD>(p, grid, st))); break;
    }
    RBK_LAUNCHED("qk_kernel");
    return RBK_OK;
}

static int check_heads(const char* who, const char* what, const rbk_heads& t, const rbk_qk_args* a, int H, bool out) {
    RBK_REQUIRE(t.p, "%s: %s is NULL", who, what);
    RBK_REQUIRE(aligned16(t.p), "%s: %s must be 16-byte aligned", who, what);
    RBK_REQUIRE(t.sb % 8 == 0 && t.ss % 8 == 0 && t.sh % 8 == 0, "%s: strides of %s must be multiples of 8 elements",
                who, what);
    const int64_t most = 8LL * 0x7fffffff;                           // strides are 32-bit counts of vectors
    for (const int64_t s : {t.sb, t.ss, t.sh})
        RBK_REQUIRE(s >= -most && s <= most, "%s: strides of %s must be below 2^34 elements", who, what);
    RBK_REQUIRE(!out || ((t.sb || a->B <= 1) && (t.ss || a->S <= 1) && (t.sh || H <= 1)),
                "%s: %s is written and must not repeat elements (zero stride)", who, what);
    return RBK_OK;
}

static Heads heads(const rbk_heads& t) { return {(uint4*)t.p, (int)(t.sb / 8), (int)(t.ss / 8), (int)(t.sh / 8)}; }

template <bool BWD>
int entry(rbk_ctx* ctx, const rbk_qk_args* a, void* stream) {
    const char* who = BWD ? "rbk_qk_norm_rope_bwd" : "rbk_qk_norm_rope_fwd";
    RBK_REQUIRE(a, "%s: args is NULL", who);
    RBK_REQUIRE(a->B >= 0 && a->S >= 0 && a->Hq >= 0 && a->Hk >= 0, "%s: negative size", who);
    RBK_REQUIRE(a->Hq <= (1 << 20) && a->Hk <= (1 << 20), "%s: more than 2^20 heads", who);
    RBK_REQUIRE((long long)a->B * a->S <= 0x7fffffffLL, "%s: more than 2^31 - 1 tokens", who);
    RBK_REQUIRE(a->dh >= 8 && a->dh <= kMaxDh && a->dh % 8 == 0, "%s: dh must be a multiple of 8 in [8, %d], got %d",
                who, kMaxDh, a->dh);
    RBK_REQUIRE(a->rot >= 0 && a->rot <= a->dh && a->rot % (a->interleaved ? 8 : 16) == 0,
                "%s: rot must be a multiple of %d in [0, dh], got %d", who, a->interleaved ? 8 : 16, a->rot);
    RBK_REQUIRE(a->eps >= FLT_MIN && std::isfinite(a->eps), "%s: eps must be positive and normal", who);
    RBK_REQUIRE(a->inv_freq || a->rot == 0 || (a->theta > 0.0 && std::isfinite(a->theta)),
                "%s: theta must be positive", who);
    RBK_REQUIRE(a->positions || a->pos0 <= 0x7fffffffLL - std::max(a->S - 1, 0), "%s: positions beyond 2^31 - 1", who);
    RBK_REQUIRE((!a->gq || aligned16(a->gq)) && (!a->gk || aligned16(a->gk)), "%s: gains must be 16-byte aligned", who);
    const int H[2] = {a->Hq, a->Hk};
    const rbk_heads* x[2] = {&a->q, &a->k};
    const rbk_heads* o[2] = {&a->oq, &a->ok};
    const rbk_heads* dy[2] = {&a->dyq, &a->dyk};
    const int tokens = a->B * a->S;
    for (int i = 0; i < 2; ++i) {
        if (!H[i] || !tokens) continue;
        RBK_TRY(check_heads(who, i ? "k" : "q", *x[i], a, H[i], false));
        RBK_TRY(check_heads(who, i ? "ok" : "oq", *o[i], a, H[i], true));
        if (BWD) RBK_TRY(check_heads(who, i ? "dyk" : "dyq", *dy[i], a, H[i], false));
    }
    RBK_REQUIRE(!BWD || aligned16(a->ws), "%s: ws must be 16-byte aligned", who);
    if (a->inv_freq)
        for (int i = 0; i < a->rot / 2; ++i)
            RBK_REQUIRE(std::isfinite(a->inv_freq[i]), "%s: inv_freq[%d] is not finite", who, i);
    RBK_TRY(check_device(ctx, who));

    Params p;
    p.tokens = tokens;
    p.S = a->S;
    p.s_shift = 0;
    while (a->S > 0 && (1u << p.s_shift) < (uint32_t)a->S) ++p.s_shift;
    p.s_mul = a->S > 0 ? (uint32_t)((((1ull << p.s_shift) - (uint32_t)a->S) << 32) / (uint32_t)a->S + 1) : 0;
    p.dh = a->dh;
    p.rot = a->rot;
    p.interleaved = a->interleaved != 0;
    p.eps = a->eps;
    p.inv_dh = 1.0f / (float)a->dh;
    p.pos = a->positions;
    p.pos0 = a->pos0;
    // Frequencies in turns, their fraction in 64-bit fixed point.  The geometric series is built by one
    // power and long double products (128 steps lose less than 2^-56 of each).
    const long double tau = 6.283185307179586476925286766559L;
    long double f = 1.0L, ratio = 1.0L;
    if (!a->inv_freq && a->rot) ratio = powl((long double)a->theta, -2.0L / (long double)a->rot);
    for (int i = 0; i < kMaxDh / 2; ++i) {
        p.freq[i] = 0;
        if (i >= a->rot / 2) continue;
        long double t = (a->inv_freq ? (long double)a->inv_freq[i] : f) / tau;
        if (t < 0.0L || t >= 1.0L) t -= floorl(t);                   // positions are whole: turns drop out
        t *= 18446744073709551616.0L;
        p.freq[i] = t >= 18446744073709551616.0L ? 0 : (unsigned long long)t;
        f *= ratio;
    }
    // A head's lanes, and the heads of a step.  Two tokens at a time where that leaves fewer lane steps.
    const int slots = (a->dh + 15) / 16;
    const int lanes = slots <= 6 ? slots : slots <= 8 ? 8 : slots <= 10 ? 10 : 16;
    const auto steps_of = [](int heads, int per) { return (heads + per - 1) / per; };
    const int one = 32 / lanes, two = 16 / lanes;
    const int T = steps_of(H[0], two) + steps_of(H[1], two) < 2 * (steps_of(H[0], one) + steps_of(H[1], one)) ? 2 : 1;
    const int hps = T == 2 ? two : one;
    // A warp takes all heads of a token where there are tokens for every warp, so that a token's angles are
    // computed once; with fewer tokens its heads are shared out over up to kMaxParts warps.
    const int most = per_sm(lanes, T, BWD) * ctx->num_sms;
    const int max_blocks = std::min(most, kMaxRows - 2 * kMaxParts / kWarps);
    const bool all = (long long)tokens * 2 >= (long long)max_blocks * kWarps * T;
    long long need[2];
    for (int i = 0; i < 2; ++i) {
        Side& s = p.side[i];
        s.H = H[i];
        s.x = heads(*x[i]);
        s.o = heads(*o[i]);
        s.dy = heads(*dy[i]);
        s.gain = (const half*)(i ? a->gk : a->gq);
        const int steps = steps_of(H[i], hps);
        s.heads_per_part = hps * (all ? steps : steps_of(steps, kMaxParts));
        s.parts = steps ? steps_of(H[i], s.heads_per_part) : 1;
        need[i] = steps ? (((long long)tokens + T - 1) / T * s.parts + kWarps - 1) / kWarps : 0;
    }
    cudaStream_t st = as_stream(stream);
    long long nb[2] = {need[0], need[1]};
    if (nb[0] + nb[1] > max_blocks) {
        // In proportion to the work: a token's steps, and half a step for its angles and addresses (by heads alone, 16
        // query heads beside one key head, 16384 tokens of heads of 128: 54 us, and 31 so).
        long long cost[2];
        for (int i = 0; i < 2; ++i) cost[i] = need[i] ? 2 * steps_of(H[i], hps) + 1 : 0;
        nb[0] = max_blocks * cost[0] / (cost[0] + cost[1]);
        nb[1] = max_blocks - nb[0];
        for (int i = 0; i < 2; ++i)                                  // a warp for each part of a token
            if (need[i]) nb[i] = std::max(nb[i], (long long)(p.side[i].parts + kWarps - 1) / kWarps);
    }
    p.blocks0 = (int)nb[0];
    const int grid = (int)(nb[0] + nb[1]);
    p.part = nullptr;
    if (BWD) {
        void* ws = a->ws;
        if (!ws) RBK_TRY(ctx_scratch(ctx, RBK_QK_BWD_WS_BYTES, &ws));
        p.part = (float*)ws;
    }
    const double n = (double)tokens * (a->Hq + a->Hk) * a->dh;
    ProfScope prof(ctx, st, kCatOther, (BWD ? 6.0 : 4.0) * n);
    if (grid) {
        const int status = a->interleaved ? (T == 2 ? launch<2, true, BWD>(p, lanes, grid, st)
                                                    : launch<1, true, BWD>(p, lanes, grid, st))
                                          : (T == 2 ? launch<2, false, BWD>(p, lanes, grid, st)
                                                    : launch<1, false, BWD>(p, lanes, grid, st));
        if (status != RBK_OK) return status;
    }
    if (BWD && (a->dgq || a->dgk)) {
        // one gradient for both: its first side's rows are all rows, and it has no second
        const bool one_gain = a->dgq == a->dgk;
        RBK_CUDA(launch_pdl(qk_gain_kernel, dim3((a->dh + 31) / 32, 2), dim3(kThreads), 0, st, a->dgq,
                            one_gain ? nullptr : a->dgk, (const float*)p.part, a->dh, one_gain ? grid : p.blocks0, grid,
                            a->accumulate));
        RBK_LAUNCHED("qk_gain_kernel");
    }
    return RBK_OK;
}

}  // namespace qk
}  // namespace rbk

extern "C" {

int rbk_qk_norm_rope_fwd(rbk_ctx* ctx, const rbk_qk_args* args, void* stream) {
    return rbk::qk::entry<false>(ctx, args, stream);
}

int rbk_qk_norm_rope_bwd(rbk_ctx* ctx, const rbk_qk_args* args, void* stream) {
    return rbk::qk::entry<true>(ctx, args, stream);
}

}  // extern "C"
