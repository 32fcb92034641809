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
// Memory bound: 4 bytes per element forward, 6 backward, each touched once.
// Layout: a head is split over G lanes (the power of two >= dh / 16), a lane holding two
// 16-byte chunks of it, chosen so that both members of every rotated pair are in the
// same lane: no exchange is needed for the rotation.  A warp works on 32 / G heads of one
// token at a time, so a token's angles are computed once for all of its heads, each by one
// of the lanes that need it (they get it by shuffle).  The loads of a warp's next heads are in
// flight while it works on its present ones, across tokens too.
#include <algorithm>
#include <cmath>

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
    int blocks0;                             // blocks [0, blocks0) work on side 0, the others on side 1
    float eps, inv_dh;
    const int* pos;
    int pos0;
    float* part;                             // [gridDim.x][dh] partial gain gradients (backward)
    unsigned long long freq[kMaxDh / 2];     // fractions of a turn per position, 2^-64; zero where nothing rotates
};

// cos and sin of position p's angle for a frequency of `freq` 2^-64 turns per position.  The product wraps
// modulo 2^64 = modulo a turn, exactly; its top 32 bits, rounded, are the angle to 2^-33 turns.
__device__ __forceinline__ void turn(int p, unsigned long long freq, float& c, float& s) {
    const unsigned long long t = (unsigned long long)(long long)p * freq + 0x80000000ull;
    sincospif((float)(int)(t >> 32) * 4.656612873077393e-10f, &s, &c);      // 2^-31: half turns
}

// What a lane holds of a head: chunks (8 channels, one vector each) a and b.
struct Lane {
    int a, b;
    bool has_a, has_b, rot_a, rot_b;
};
__device__ __forceinline__ Lane lane_of(const Params& p, int j) {
    Lane l;
    const int chunks = p.dh >> 3, rs = p.rot >> 4;
    if (p.interleaved) {
        l.a = 2 * j;
        l.b = l.a + 1;
        l.rot_a = l.a < (p.rot >> 3);
        l.rot_b = l.b < (p.rot >> 3);
    } else {
        l.a = j < rs ? j : 2 * j;
        l.b = j < rs ? j + rs : 2 * j + 1;
        l.rot_a = l.rot_b = j < rs;
    }
    l.has_a = l.a < chunks;
    l.has_b = l.b < chunks;
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
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Blocks of an SM: 24 warps at 80 registers forward, 16 at 128 backward.
template <bool BWD>
constexpr int kPerSm = BWD ? 2 : 3;

template <int G, bool INTER, bool BWD>
__global__ void __launch_bounds__(kThreads, kPerSm<BWD>) qk_kernel(const __grid_constant__ Params p) {
    constexpr int HPW = 32 / G;                                     // heads of a token per warp and step
    constexpr int ANG = HPW >= 8 ? 1 : 8 / HPW;                     // angles that a lane computes of its slot's 8
    __shared__ float acc_s[BWD ? kWarps : 1][BWD ? kMaxDh : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int which = (int)blockIdx.x >= p.blocks0;
    const Side& sd = p.side[which];
    const int w = (which ? blockIdx.x - p.blocks0 : blockIdx.x) * kWarps + warp;
    const int stride = max(1, (int)(which ? gridDim.x - p.blocks0 : p.blocks0) * kWarps / sd.parts);   // tokens of a round
    const int g = lane / G, j = lane % G;
    const Lane l = lane_of(p, j);
    unsigned long long freq[ANG];
#pragma unroll
    for (int i = 0; i < ANG; ++i) freq[i] = p.freq[8 * j + (g * ANG + i) % 8];
    grid_dependency_sync();

    Row gain;
    {
        const uint4 one = make_uint4(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u);
        const uint4* gp = reinterpret_cast<const uint4*>(sd.gain);
        tc::h8_to_p(gp ? load8(gp + l.a, l.has_a) : one, gain.v);
        tc::h8_to_p(gp ? load8(gp + l.b, l.has_b) : one, gain.v + 4);
    }
    Row acc = {};                                                   // gain gradient

    // The heads in flight: token (bi, si), this lane's head and pointers to its chunk a.
    const int part = w % sd.parts, h0 = part * sd.heads_per_part + g;
    const int h1 = min(sd.H, (part + 1) * sd.heads_per_part) + g;   // of the group's heads: h - g < h1 - g
    const int ab = l.b - l.a;
    int token = w / sd.parts < stride ? w / sd.parts : p.tokens, h = 0, pos = 0;
    const uint4 *xp = nullptr, *ep = nullptr;
    uint4* op = nullptr;
    uint4 xa, xb, ea, eb;
    auto at = [&](const Heads& t, int bi, int si) {
        return t.p + ((long long)bi * t.sb + (long long)si * t.ss + (long long)h0 * t.sh + l.a);
    };
    auto start = [&] {
        const int bi = (int)((unsigned)token / (unsigned)p.S), si = token - bi * p.S;
        pos = p.pos ? p.pos[token] : p.pos0 + si;
        xp = at(sd.x, bi, si);
        op = at(sd.o, bi, si);
        if (BWD) ep = at(sd.dy, bi, si);
        h = h0;
    };
    auto fetch = [&] {
        const bool on = h < sd.H;
        xa = load8(xp, on && l.has_a);
        xb = load8(xp + ab, on && l.has_b);
        if (BWD) {
            ea = load8(ep, on && l.has_a);
            eb = load8(ep + ab, on && l.has_b);
        }
    };
    if (token < p.tokens) {
        start();
        fetch();
    }
    bool fresh = true;
    uint64_t cs[4], sn[4];
    while (token < p.tokens) {
        Row x, e;
        tc::h8_to_p(xa, x.v);
        tc::h8_to_p(xb, x.v + 4);
        if (BWD) {
            tc::h8_to_p(ea, e.v);
            tc::h8_to_p(eb, e.v + 4);
        }
        const bool on = h < sd.H;
        uint4* const o = op;
        if (fresh) {                                                // a new token: its angles
            float c[ANG], s[ANG];
#pragma unroll
            for (int i = 0; i < ANG; ++i) turn(pos, freq[i], c[i], s[i]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int s0 = i / ANG * G + j, s1 = (i + 1) / ANG * G + j;
                cs[i / 2] = pk2(__shfl_sync(0xffffffffu, c[i % ANG], s0), __shfl_sync(0xffffffffu, c[(i + 1) % ANG], s1));
                sn[i / 2] = pk2(__shfl_sync(0xffffffffu, s[i % ANG], s0), __shfl_sync(0xffffffffu, s[(i + 1) % ANG], s1));
            }
        }
        h += HPW;
        xp += HPW * (long long)sd.x.sh;
        op += HPW * (long long)sd.o.sh;
        if (BWD) ep += HPW * (long long)sd.dy.sh;
        fresh = h >= h1;                                            // the same in all lanes
        if (fresh) {
            token = p.tokens - token > stride ? token + stride : p.tokens;
            if (token < p.tokens) start();
        }
        if (token < p.tokens) fetch();

        uint64_t ss = 0;                                            // two zeros
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = pfma2(x.v[i], x.v[i], ss);
        if constexpr (!BWD) {
            const float rstd = rsqrtf(group_sum<G>(lo2(ss) + hi2(ss)) * p.inv_dh + p.eps);
            const uint64_t r2 = pk2(rstd, rstd);
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = pmul2(pmul2(x.v[i], r2), gain.v[i]);
            rotate<INTER, false>(l, x, cs, sn);
        } else {
            rotate<INTER, true>(l, e, cs, sn);
            uint64_t wx = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) wx = pfma2(pmul2(e.v[i], gain.v[i]), x.v[i], wx);
            const float rstd = rsqrtf(group_sum<G>(lo2(ss) + hi2(ss)) * p.inv_dh + p.eps);
            const float t = -group_sum<G>(lo2(wx) + hi2(wx)) * rstd * p.inv_dh;   // -mean(w xhat)
            const uint64_t r2 = pk2(rstd, rstd), t2 = pk2(t, t);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint64_t xh = pmul2(x.v[i], r2);
                acc.v[i] = pfma2(e.v[i], xh, acc.v[i]);
                x.v[i] = pmul2(pfma2(xh, t2, pmul2(e.v[i], gain.v[i])), r2);
            }
        }
        if (on && l.has_a) o[0] = tc::p_to_h8(x.v);
        if (on && l.has_b) o[ab] = tc::p_to_h8(x.v + 4);
    }
    if constexpr (BWD) {
        // lanes of the same slot, then the warps, in a fixed order
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float a = lo2(acc.v[i]), b = hi2(acc.v[i]);
#pragma unroll
            for (int o = G; o < 32; o <<= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                b += __shfl_xor_sync(0xffffffffu, b, o);
            }
            const int c = i < 4 ? 8 * l.a + 2 * i : 8 * l.b + 2 * (i - 4);
            if (g == 0 && (i < 4 ? l.has_a : l.has_b)) {
                acc_s[warp][c] = a;
                acc_s[warp][c + 1] = b;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.dh; c += kThreads) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v += acc_s[w][c];
            p.part[(size_t)blockIdx.x * p.dh + c] = v;
        }
    }
}

// dgain[c] (+)= sum over the side's partial rows: a block takes 32 channels, its warps every eighth row, and the
// warps' sums are added in order.
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

template <bool INTER, bool BWD>
int run(const Params& p, int grid, cudaStream_t st) {
    const int slots = (p.dh + 15) / 16;
    const dim3 gd(grid), bd(kThreads);
    if (slots <= 1) RBK_CUDA(launch_pdl(qk_kernel<1, INTER, BWD>, gd, bd, 0, st, p));
    else if (slots <= 2) RBK_CUDA(launch_pdl(qk_kernel<2, INTER, BWD>, gd, bd, 0, st, p));
    else if (slots <= 4) RBK_CUDA(launch_pdl(qk_kernel<4, INTER, BWD>, gd, bd, 0, st, p));
    else if (slots <= 8) RBK_CUDA(launch_pdl(qk_kernel<8, INTER, BWD>, gd, bd, 0, st, p));
    else RBK_CUDA(launch_pdl(qk_kernel<16, INTER, BWD>, gd, bd, 0, st, p));
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
    RBK_REQUIRE((long long)a->B * a->S <= 0x7fffffffLL, "%s: more than 2^31 - 1 tokens", who);
    RBK_REQUIRE(a->dh >= 8 && a->dh <= kMaxDh && a->dh % 8 == 0, "%s: dh must be a multiple of 8 in [8, %d], got %d",
                who, kMaxDh, a->dh);
    RBK_REQUIRE(a->rot >= 0 && a->rot <= a->dh && a->rot % (a->interleaved ? 8 : 16) == 0,
                "%s: rot must be a multiple of %d in [0, dh], got %d", who, a->interleaved ? 8 : 16, a->rot);
    RBK_REQUIRE(a->eps > 0.0f && std::isfinite(a->eps), "%s: eps must be positive", who);
    RBK_REQUIRE(a->inv_freq || a->rot == 0 || (a->theta > 0.0 && std::isfinite(a->theta)),
                "%s: theta must be positive", who);
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
        t -= floorl(t);                                              // positions are whole: turns drop out
        t = roundl(t * 18446744073709551616.0L);
        p.freq[i] = t >= 18446744073709551616.0L ? 0 : (unsigned long long)t;
        f *= ratio;
    }
    // A warp takes all heads of a token where there are tokens for every warp, so that a token's angles are
    // computed once; with fewer tokens its heads are shared out over up to kMaxParts warps.
    const int slots = (a->dh + 15) / 16;
    const int hpw = slots <= 1 ? 32 : slots <= 2 ? 16 : slots <= 4 ? 8 : slots <= 8 ? 4 : 2;
    const int most = kPerSm<BWD> * ctx->num_sms;
    const int max_blocks = std::min(most, kMaxRows - 2 * kMaxParts / kWarps);
    const bool all = (long long)tokens * 2 >= (long long)max_blocks * kWarps;
    long long need[2];
    for (int i = 0; i < 2; ++i) {
        Side& s = p.side[i];
        s.H = H[i];
        s.x = heads(*x[i]);
        s.o = heads(*o[i]);
        s.dy = heads(*dy[i]);
        s.gain = (const half*)(i ? a->gk : a->gq);
        const int steps = (H[i] + hpw - 1) / hpw;
        s.heads_per_part = hpw * (all ? steps : (steps + kMaxParts - 1) / kMaxParts);
        s.parts = steps ? (H[i] + s.heads_per_part - 1) / s.heads_per_part : 1;
        need[i] = steps ? ((long long)tokens * s.parts + kWarps - 1) / kWarps : 0;
    }
    cudaStream_t st = as_stream(stream);
    long long nb[2] = {need[0], need[1]};
    if (nb[0] + nb[1] > max_blocks) {                                // in proportion to the heads
        nb[0] = (long long)max_blocks * a->Hq / ((long long)a->Hq + a->Hk);
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
        const int status = a->interleaved ? run<true, BWD>(p, grid, st) : run<false, BWD>(p, grid, st);
        if (status != RBK_OK) return status;
    }
    if (BWD && (a->dgq || a->dgk)) {
        RBK_CUDA(launch_pdl(qk_gain_kernel, dim3((a->dh + 31) / 32, 2), dim3(kThreads), 0, st, a->dgq, a->dgk,
                            (const float*)p.part, a->dh, p.blocks0, grid, a->accumulate));
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
