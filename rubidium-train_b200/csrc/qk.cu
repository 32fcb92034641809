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
// token at a time, so a token's angles are computed once for all of its heads.
#include <cmath>

#include "common.cuh"

namespace rbk {
namespace qk {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxDh = 256;
constexpr int kMaxRows = 1024;               // partial rows of the gain gradients (RBK_QK_BWD_WS_BYTES)

struct Heads {
    half* p;
    long long sb, ss, sh;
};
struct Side {                                // the queries or the keys
    int H;
    int units_per_token, heads_per_unit;     // a warp takes heads_per_unit heads of one token at a time
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

// What a lane holds of a head: chunks (8 channels each) a and b.
struct Lane {
    int a, b;                                // channel offsets
    bool has_a, has_b, rot_a, rot_b;
};
__device__ __forceinline__ Lane lane_of(const Params& p, int j) {
    Lane l;
    const int chunks = p.dh >> 3, rs = p.rot >> 4;
    int ca, cb;
    if (p.interleaved) {
        ca = 2 * j;
        cb = ca + 1;
        l.rot_a = ca < (p.rot >> 3);
        l.rot_b = cb < (p.rot >> 3);
    } else {
        ca = j < rs ? j : 2 * j;
        cb = j < rs ? j + rs : 2 * j + 1;
        l.rot_a = l.rot_b = j < rs;
    }
    l.has_a = ca < chunks;
    l.has_b = cb < chunks;
    l.a = 8 * ca;
    l.b = 8 * cb;
    return l;
}

// The rotation (sign = 1) or its transpose (sign = -1) on a lane's channels.
__device__ __forceinline__ void rotate(const Params& p, const Lane& l, float* a, float* b, const float* c,
                                       const float* s, float sign) {
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (l.rot_a) {
                const float x = a[2 * i], y = a[2 * i + 1], sn = sign * s[i];
                a[2 * i] = x * c[i] - y * sn;
                a[2 * i + 1] = x * sn + y * c[i];
            }
            if (l.rot_b) {
                const float x = b[2 * i], y = b[2 * i + 1], sn = sign * s[4 + i];
                b[2 * i] = x * c[4 + i] - y * sn;
                b[2 * i + 1] = x * sn + y * c[4 + i];
            }
        }
    } else if (l.rot_a) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = a[i], y = b[i], sn = sign * s[i];
            a[i] = x * c[i] - y * sn;
            b[i] = x * sn + y * c[i];
        }
    }
}

__device__ __forceinline__ uint4 load8(const half* p, bool on) {
    return on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int G, bool BWD>
__global__ void __launch_bounds__(kThreads) qk_kernel(const __grid_constant__ Params p) {
    constexpr int HPW = 32 / G;                                     // heads of a token per warp and step
    __shared__ float acc_s[BWD ? kWarps : 1][BWD ? kMaxDh : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int which = (int)blockIdx.x >= p.blocks0;
    const Side& sd = p.side[which];
    const int block = which ? blockIdx.x - p.blocks0 : blockIdx.x;
    const int blocks = which ? gridDim.x - p.blocks0 : p.blocks0;
    const int g = lane / G, j = lane % G;
    const Lane l = lane_of(p, j);
    grid_dependency_sync();

    float ga[8], gb[8];
    if (sd.gain) {
        h8_to_f(load8(sd.gain + l.a, l.has_a), ga);
        h8_to_f(load8(sd.gain + l.b, l.has_b), gb);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) ga[i] = gb[i] = 1.0f;
    }
    float da[8] = {}, db[8] = {};

    const long long units = (long long)p.tokens * sd.units_per_token;
    for (long long u = (long long)block * kWarps + warp; u < units; u += (long long)blocks * kWarps) {
        const int token = (int)(u / sd.units_per_token), part = (int)(u - (long long)token * sd.units_per_token);
        const int bi = token / p.S, si = token - bi * p.S;
        const int pos = p.pos ? p.pos[token] : p.pos0 + si;
        float c[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) turn(pos, p.freq[8 * j + i], c[i], s[i]);
        const half* xt = sd.x.p + bi * sd.x.sb + si * sd.x.ss;
        half* ot = sd.o.p + bi * sd.o.sb + si * sd.o.ss;
        const half* dt = BWD ? sd.dy.p + bi * sd.dy.sb + si * sd.dy.ss : nullptr;
        const int h0 = part * sd.heads_per_unit, h1 = min(sd.H, h0 + sd.heads_per_unit);
        for (int hb = h0; hb < h1; hb += HPW) {                     // the same trip count in every lane
            const int h = hb + g;
            const bool on = h < h1;
            float a[8], b[8];
            h8_to_f(load8(xt + h * sd.x.sh + l.a, on && l.has_a), a);
            h8_to_f(load8(xt + h * sd.x.sh + l.b, on && l.has_b), b);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
            if constexpr (!BWD) {
                const float rstd = rsqrtf(group_sum<G>(ss) * p.inv_dh + p.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[i] = a[i] * rstd * ga[i];
                    b[i] = b[i] * rstd * gb[i];
                }
                rotate(p, l, a, b, c, s, 1.0f);
            } else {
                float ea[8], eb[8];
                h8_to_f(load8(dt + h * sd.dy.sh + l.a, on && l.has_a), ea);
                h8_to_f(load8(dt + h * sd.dy.sh + l.b, on && l.has_b), eb);
                rotate(p, l, ea, eb, c, s, -1.0f);
                float wx = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) wx += ea[i] * ga[i] * a[i] + eb[i] * gb[i] * b[i];
                const float rstd = rsqrtf(group_sum<G>(ss) * p.inv_dh + p.eps);
                const float t = group_sum<G>(wx) * rstd * p.inv_dh;  // mean(w xhat)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[i] *= rstd;
                    b[i] *= rstd;
                    da[i] += ea[i] * a[i];
                    db[i] += eb[i] * b[i];
                    a[i] = rstd * (ea[i] * ga[i] - a[i] * t);
                    b[i] = rstd * (eb[i] * gb[i] - b[i] * t);
                }
            }
            if (on && l.has_a) *reinterpret_cast<uint4*>(ot + h * sd.o.sh + l.a) = f_to_h8(a);
            if (on && l.has_b) *reinterpret_cast<uint4*>(ot + h * sd.o.sh + l.b) = f_to_h8(b);
        }
    }
    if constexpr (BWD) {
        // lanes of the same slot, then the warps, in a fixed order
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int o = G; o < 32; o <<= 1) {
                da[i] += __shfl_xor_sync(0xffffffffu, da[i], o);
                db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
            }
        }
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (l.has_a) acc_s[warp][l.a + i] = da[i];
                if (l.has_b) acc_s[warp][l.b + i] = db[i];
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

// dgain[c] (+)= sum over the side's partial rows, one warp per channel.
__global__ void __launch_bounds__(kThreads) qk_gain_kernel(float* dgq, float* dgk, const float* part, int dh, int rows0,
                                                           int rows, int accumulate) {
    grid_dependency_sync();
    const int ch = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int which = blockIdx.y;
    float* out = which ? dgk : dgq;
    if (ch >= dh || !out) return;
    float v = 0.0f;
    for (int r = (which ? rows0 : 0) + lane; r < (which ? rows : rows0); r += 32) v += part[(size_t)r * dh + ch];
    v = warp_sum(v);
    if (lane == 0) out[ch] = accumulate ? out[ch] + v : v;
}

template <bool BWD>
int run(rbk_ctx* ctx, const Params& p, int grid, cudaStream_t st) {
    const int slots = (p.dh + 15) / 16;
    if (slots <= 1) RBK_CUDA(launch_pdl(qk_kernel<1, BWD>, dim3(grid), dim3(kThreads), 0, st, p));
    else if (slots <= 2) RBK_CUDA(launch_pdl(qk_kernel<2, BWD>, dim3(grid), dim3(kThreads), 0, st, p));
    else if (slots <= 4) RBK_CUDA(launch_pdl(qk_kernel<4, BWD>, dim3(grid), dim3(kThreads), 0, st, p));
    else if (slots <= 8) RBK_CUDA(launch_pdl(qk_kernel<8, BWD>, dim3(grid), dim3(kThreads), 0, st, p));
    else RBK_CUDA(launch_pdl(qk_kernel<16, BWD>, dim3(grid), dim3(kThreads), 0, st, p));
    RBK_LAUNCHED("qk_kernel");
    return RBK_OK;
}

static int check_heads(const char* who, const char* what, const rbk_heads& t, const rbk_qk_args* a, int H, bool out) {
    RBK_REQUIRE(t.p, "%s: %s is NULL", who, what);
    RBK_REQUIRE(aligned16(t.p), "%s: %s must be 16-byte aligned", who, what);
    RBK_REQUIRE(t.sb % 8 == 0 && t.ss % 8 == 0 && t.sh % 8 == 0, "%s: strides of %s must be multiples of 8 elements",
                who, what);
    RBK_REQUIRE(!out || ((t.sb || a->B <= 1) && (t.ss || a->S <= 1) && (t.sh || H <= 1)),
                "%s: %s is written and must not repeat elements (zero stride)", who, what);
    return RBK_OK;
}

static Heads heads(const rbk_heads& t) { return {(half*)t.p, t.sb, t.ss, t.sh}; }

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
    // Enough warps to fill the machine first, then as many heads of a token per warp as there are, so that
    // a token's angles are computed once.
    const int hpw = [&] {
        const int slots = (a->dh + 15) / 16;
        return slots <= 1 ? 32 : slots <= 2 ? 16 : slots <= 4 ? 8 : slots <= 8 ? 4 : 2;
    }();
    const int max_blocks = 4 * ctx->num_sms < kMaxRows ? 4 * ctx->num_sms : kMaxRows;
    long long need[2];
    for (int i = 0; i < 2; ++i) {
        Side& s = p.side[i];
        s.H = H[i];
        s.x = heads(*x[i]);
        s.o = heads(*o[i]);
        s.dy = heads(*dy[i]);
        s.gain = (const half*)(i ? a->gk : a->gq);
        const int steps = (H[i] + hpw - 1) / hpw;
        const bool all = (long long)tokens * 2 >= (long long)max_blocks * kWarps;
        s.heads_per_unit = all && steps ? steps * hpw : hpw;
        s.units_per_token = all ? (steps ? 1 : 0) : steps;
        need[i] = ((long long)tokens * s.units_per_token + kWarps - 1) / kWarps;
    }
    cudaStream_t st = as_stream(stream);
    long long nb[2] = {need[0], need[1]};
    if (nb[0] + nb[1] > max_blocks) {                                // in proportion to the heads
        nb[0] = need[0] ? (long long)max_blocks * a->Hq / (a->Hq + a->Hk) : 0;
        nb[0] = need[0] && nb[0] < 1 ? 1 : nb[0];
        nb[1] = max_blocks - nb[0];
        if (need[1] && nb[1] < 1) { nb[1] = 1; nb[0] = max_blocks - 1; }
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
    if (grid) RBK_TRY(run<BWD>(ctx, p, grid, st));
    if (BWD && (a->dgq || a->dgk)) {
        RBK_CUDA(launch_pdl(qk_gain_kernel, dim3((a->dh + kWarps - 1) / kWarps, 2), dim3(kThreads), 0, st, a->dgq, a->dgk,
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
