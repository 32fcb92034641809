// ffn.cu — the gated feed-forward block, forward and backward.
//
//   gate = x Wg^T + bg,  up = x Wu^T + bu,  h = act(gate) * up,  y = h Wd^T + bd + residual
//   dh = dy Wd,  dgate = dh up act'(gate),  dup = dh act(gate),  dx = dgate Wg + dup Wu
//
// Many rows: tensor bound (6 N D F FLOP each way).  The CTA-pair GEMM of gemm.cu with epilogues of its own
// makes h (gate and up tiles share one accumulator) and dgu; the other products are plain GEMMs.  8192 rows,
// D 2048, F 5632: forward 425 to 510 us (280 + 142 its two kernels alone; the power limit does the rest), backward without
// weight gradients 500 to 560 (174 + 280), with them 1010 to 1050 (283 + 147 more); in a stream of calls 498 and 552.
// Where those tiles are too few for the machine, smaller ones (ffn_mid.cu).
// Few rows: the weights, 6 D F bytes, are read once and that is the cost.  The kernels below stream them.
#include <algorithm>

#include "tc.cuh"

namespace rbk {
namespace ffn {

// ---------------------------------------------------------------- few rows ----
// out[n, r] = sum_k w[r, k] x[n, k] for up to 8 NT rows n.  A tile is 16 MT weight rows (GLU: of each 16, eight
// of the gate and the same eight of the up projection, so that a lane ends up with both of its elements); a CTA
// goes through its tiles, its warps share k out in rounds of 64, and their sums are added in warp order through
// shared memory.  mma.sync m16n8k16 with the weights as the 16-row operand: the tensor pipe is idle next to the
// memory, what matters is that a lane's fragment is a whole 16-byte vector.  The k order within a half round is
// permuted for that, alike on both sides: lane 4 g + t holds k = 8 t .. 8 t + 7 of row g, and MMA m of the two
// that use them takes elements 4 m .. 4 m + 3.
// A lane copies its vectors of the next DEPTH - 1 rounds, across tiles, into slots of its own with cp.async and
// waits for its own copies only: the weights stream without registers or barriers.  Bound by HBM where the weights
// are large (1 row, D 2048, F 5632: 14.6 us for both kernels, 69 MB, 4740 GB/s with two ramps; plain loads in
// the loop took 22.4), by latency where they are not (D 768, F 2048: 5.5 us), and from 16 rows on also by x, which
// every tile reads from L2 (32 rows: 26.7 us), and by SMs without work: 21 rows, D 1000, F 2664 are 167 tiles of gate and
// up on 148 SMs and 63 of the down projection (13.8 us, floor 2.5).

// Which calls they serve: up to 32 rows, and up to 64 of a narrow block, where the launches and waits of the tiles are
// most of their time.  Measured at 48 rows, these kernels against the tiles: D 512, F 1024: 7.5 us against 9.8;
// D 768, F 2048: 12.6 against 12.9; D 1024, F 2816: 21 against 16.5; D 256, F 5632: 22 against 15.  At 32 rows:
// D 1024, F 2816: 12.3 against 15.7; D 2048, F 5632: 27 both.
static bool few(int N, int D, int F) {
    return N <= 32 || (N <= 64 && std::max(D, F) <= 2048 && (int64_t)D * F <= (3 << 19));
}

// WIDE: at most one tile per SM, so a CTA has all of its shared memory for what is in flight; else two CTAs share
// an SM (1 row, D 4096, F 11264: 48 to 49.5 us; three of four warps with deeper slots 52.8), and a tile is 32 weight
// rows where x, which comes from L2 for each, is more than the weights (16 rows n, D 1888, F 4312: 21.5 us with 16
// weight rows, 16.6 with 32).
template <int NT, bool WIDE>
struct Few {
    static constexpr int MT = NT > 1 && !WIDE ? 2 : 1;
    static constexpr int WARPS = WIDE || NT == 1 ? 8 : 4, THREADS = 32 * WARPS;
    static constexpr int DEPTH = WIDE ? (NT == 1 ? 8 : NT == 2 ? 6 : NT == 4 ? 4 : 2) : NT == 2 ? 4 : 3;
    static constexpr int VECS = 4 * MT + 2 * NT;         // 16-byte vectors of a lane and round
    static constexpr int ROUND = VECS * 512;
    static constexpr int RING = WARPS * DEPTH * ROUND;
    static constexpr int SUMS = WARPS * MT * 16 * (8 * NT + 1) * 4;
    static constexpr int SMEM = RING + SUMS;
    static constexpr int PER_SM = WIDE || NT == 8 ? 1 : 2;
    static_assert(PER_SM * (SMEM + 1024) <= 233472, "shared memory of an SM");
};

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const half* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}

struct Params {
    int N, R, K;                   // tokens, weight rows (of one of the two matrices when gated), inner extent
    const half* w;                 // [R, K]; gated: [2R, K]
    const half* x;
    long long ldx;
    const half* bias;              // [R]; gated: [2R]
    const half* residual;          // [N, R]
    long long ldr;
    half* out;                     // [N, R]
    long long ldo;
    half* gu;                      // gated: [N, 2R] or NULL
    int act;
    int early;                     // the weights may be read before the kernel before this one has ended
};

template <int NT, bool WIDE, bool GLU>
__global__ void __launch_bounds__(Few<NT, WIDE>::THREADS) few_rows_kernel(const Params p) {
    using C = Few<NT, WIDE>;
    constexpr int MT = C::MT, DEPTH = C::DEPTH;
    constexpr int OUT = GLU ? 8 * MT : 16 * MT;          // output columns of a tile
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = tc::su32(smem) + warp * (DEPTH * C::ROUND) + lane * 16;
    auto sums = reinterpret_cast<float(*)[MT][16][8 * NT + 1]>(smem + C::RING);
    const int tiles = (p.R + OUT - 1) / OUT;
    const int k0 = 64 * warp + 8 * t;                    // this lane's first k

    // the copies: tile ft, k fk, rows' pointers, x's pointer
    int ft = blockIdx.x, fk = k0;
    const half *wp[MT][2], *xp = nullptr;
    uint32_t fd = ring;
    auto rows = [&] {                                    // of tile ft; past the end, the last row: not stored
        if (ft >= tiles) return;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int r = ft * OUT + (GLU ? 8 : 16) * m + g;
            wp[m][0] = p.w + (size_t)min(r, p.R - 1) * p.K + k0;
            wp[m][1] = p.w + (GLU ? (size_t)p.R + min(r, p.R - 1) : (size_t)min(r + 8, p.R - 1)) * p.K + k0;
        }
    };
    auto fetch_w = [&](uint32_t d) {
        if (ft >= tiles) return;
        const bool on0 = fk < p.K, on1 = fk + 32 < p.K;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                copy16(d + (4 * m + 2 * h) * 512, wp[m][h], on0);
                copy16(d + (4 * m + 2 * h + 1) * 512, wp[m][h] + 32, on1);
                wp[m][h] += 64 * C::WARPS;
            }
    };
    auto fetch_x = [&](uint32_t d) {
        if (ft < tiles) {
            const bool on0 = fk < p.K, on1 = fk + 32 < p.K;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const bool row = 8 * j + g < p.N;
                copy16(d + (4 * MT + 2 * j) * 512, xp + 8 * j * p.ldx, row && on0);
                copy16(d + (4 * MT + 2 * j + 1) * 512, xp + 8 * j * p.ldx + 32, row && on1);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto advance = [&] {                                 // to the round after; every warp has the same number
        fk += 64 * C::WARPS;
        xp += 64 * C::WARPS;
        fd = fd + C::ROUND == ring + DEPTH * C::ROUND ? ring : fd + C::ROUND;
        if (fk - k0 >= p.K) {
            ft += gridDim.x;
            fk = k0;
            xp = p.x + (size_t)g * p.ldx + k0;
            rows();
        }
    };
    xp = p.x + (size_t)g * p.ldx + k0;
    rows();
    if (p.early) {
        // the weights of the first rounds, then x behind them in the same slots
        const half* x1 = xp;
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) { fetch_w(fd); advance(); }
        grid_dependency_sync();
        ft = blockIdx.x; fk = k0; xp = x1; fd = ring;
        rows();
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) {
            fetch_x(fd);
#pragma unroll
            for (int m = 0; m < MT; ++m) { wp[m][0] += 64 * C::WARPS; wp[m][1] += 64 * C::WARPS; }
            advance();
        }
    } else {
        grid_dependency_sync();
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) { fetch_w(fd); fetch_x(fd); advance(); }
    }

    uint32_t d = ring;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        float acc[MT][NT][4] = {};
        for (int k = 0; k < p.K; k += 64 * C::WARPS) {
            asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
            uint4 a[MT][4], b[NT][2];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) a[m][i] = lds16(d + (4 * m + i) * 512);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) b[j][i] = lds16(d + (4 * MT + 2 * j + i) * 512);
            d = d + C::ROUND == ring + DEPTH * C::ROUND ? ring : d + C::ROUND;
            fetch_w(fd);                                 // into the slot of the round before
            fetch_x(fd);
            advance();
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        mma_16816(acc[m][j], a[m][i].x, a[m][2 + i].x, a[m][i].y, a[m][2 + i].y, b[j][i].x, b[j][i].y);
                        mma_16816(acc[m][j], a[m][i].z, a[m][2 + i].z, a[m][i].w, a[m][2 + i].w, b[j][i].z, b[j][i].w);
                    }
        }
        if (tile != blockIdx.x) __syncthreads();         // the sums of the tile before have been read
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sums[warp][m][g + 8 * (e >> 1)][8 * j + 2 * t + (e & 1)] = acc[m][j][e];
        __syncthreads();
        for (int i = threadIdx.x; i < OUT * p.N; i += C::THREADS) {
            const int c = i % OUT, n = i / OUT, col = tile * OUT + c;
            if (col >= p.R) continue;
            const int m = c / (GLU ? 8 : 16), r = c % (GLU ? 8 : 16);
            float v = 0.0f, u = 0.0f;
#pragma unroll
            for (int w = 0; w < C::WARPS; ++w) {
                v += sums[w][m][r][n];
                if (GLU) u += sums[w][m][r + 8][n];
            }
            if (p.bias) v += __half2float(p.bias[col]);
            if constexpr (GLU) {
                if (p.bias) u += __half2float(p.bias[p.R + col]);
                if (p.gu) {
                    p.gu[(size_t)n * 2 * p.R + col] = __float2half_rn(v);
                    p.gu[(size_t)n * 2 * p.R + p.R + col] = __float2half_rn(u);
                }
                v = glu_act(v, p.act) * u;
            } else if (p.residual) {
                v += __half2float(p.residual[n * p.ldr + col]);
            }
            p.out[n * p.ldo + col] = __float2half_rn(v);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int NT, bool WIDE, bool GLU>
int launch_few(rbk_ctx* ctx, const Params& p, cudaStream_t st) {
    using C = Few<NT, WIDE>;
    static int configured_device = -1;   // attribute is per device; one device per process
    if (configured_device != ctx->device) {
        RBK_CUDA(cudaFuncSetAttribute(few_rows_kernel<NT, WIDE, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        configured_device = ctx->device;
    }
    // the same number of tiles, or one fewer, for every CTA
    const int out = (GLU ? 8 : 16) * C::MT, tiles = (p.R + out - 1) / out, slots = C::PER_SM * ctx->num_sms;
    const int each = (tiles + slots - 1) / slots;
    RBK_CUDA(launch_pdl(few_rows_kernel<NT, WIDE, GLU>, dim3((tiles + each - 1) / each), dim3(C::THREADS), C::SMEM, st, p));
    RBK_LAUNCHED("few_rows_kernel");
    return RBK_OK;
}

static bool few_wide(rbk_ctx* ctx, int R, bool glu) { return (R + (glu ? 7 : 15)) / (glu ? 8 : 16) <= ctx->num_sms; }

template <bool GLU>
int few_rows(rbk_ctx* ctx, const Params& p, cudaStream_t st) {
    ProfScope prof(ctx, st, kCatGemm, (GLU ? 4.0 : 2.0) * p.N * (double)p.R * p.K, 0);
    const bool wide = few_wide(ctx, p.R, GLU);
    if (p.N <= 8) return wide ? launch_few<1, true, GLU>(ctx, p, st) : launch_few<1, false, GLU>(ctx, p, st);
    if (p.N <= 16) return wide ? launch_few<2, true, GLU>(ctx, p, st) : launch_few<2, false, GLU>(ctx, p, st);
    if (p.N <= 32) return wide ? launch_few<4, true, GLU>(ctx, p, st) : launch_few<4, false, GLU>(ctx, p, st);
    // 33 to 64 rows: D is at most 2048, which is 128 of the down projection's tiles
    if constexpr (GLU)
        if (!wide) return launch_few<8, false, GLU>(ctx, p, st);
    return launch_few<8, true, GLU>(ctx, p, st);
}

static int check_sizes(const char* who, int N, int D, int F, int act) {
    RBK_REQUIRE(N >= 0, "%s: negative N", who);
    RBK_REQUIRE(N <= (1 << 30), "%s: more than 2^30 rows", who);         // rounded up to tiles they stay an int
    RBK_REQUIRE(D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0 && D <= (1 << 29) && F <= (1 << 29),
                "%s: D and F must be positive multiples of 8, at most 2^29 (D=%d F=%d)", who, D, F);
    // the kernels count the tiles of an output in an int
    const auto blocks = [](int n) { return ((long long)n + 127) / 128; };
    RBK_REQUIRE(blocks(N) * blocks(std::max(D, 2 * F)) <= 0x7fffffffLL && blocks(2 * F) * blocks(D) <= 0x7fffffffLL,
                "%s: more than 2^31 - 1 tiles of 128 x 128 (N=%d D=%d F=%d)", who, N, D, F);
    RBK_REQUIRE(act == RBK_ACT_SILU || act == RBK_ACT_GELU, "%s: act must be RBK_ACT_SILU or RBK_ACT_GELU", who);
    return RBK_OK;
}
// A required (or, with optional, possibly NULL) pointer and the row stride of its [N, cols] rows (cols 0: none).
static int check_ptr(const char* who, const char* what, const void* p, bool optional, int ld = 0, int cols = 0) {
    RBK_REQUIRE(p || optional, "%s: %s is NULL", who, what);
    RBK_REQUIRE(aligned16(p), "%s: %s must be 16-byte aligned", who, what);
    RBK_REQUIRE(!p || !cols || (ld >= cols && ld % 8 == 0), "%s: row stride of %s must be a multiple of 8, at least %d", who,
                what, cols);
    return RBK_OK;
}

// The FP32 planes of the down projection (backward: of dx), if the call splits it.
static int64_t plane_bytes(rbk_ctx* ctx, int M, int N, int K, int b_mn) {
    if (mid_serves(ctx, kMidStore, M, N, K, b_mn)) return 0;
    const int s = gemm_store_splits(ctx, M, N, K);
    return s > 1 ? (int64_t)s * M * N * 4 : 0;
}
static int check_ws(const char* who, const void* ws, int64_t ws_bytes, int64_t need) {
    RBK_REQUIRE(!ws || ws_bytes >= need, "%s: ws has %lld bytes, %lld are needed", who, (long long)ws_bytes,
                (long long)need);
    return RBK_OK;
}

}  // namespace ffn
}  // namespace rbk

using namespace rbk;

extern "C" {

int64_t rbk_gated_ffn_ws_bytes(rbk_ctx* ctx, int N, int D, int F, int backward) {
    const char* who = "rbk_gated_ffn_ws_bytes";
    RBK_TRY(ffn::check_sizes(who, N, D, F, RBK_ACT_SILU));
    RBK_REQUIRE(ctx, "%s: ctx is NULL", who);
    if (N == 0 || (!backward && ffn::few(N, D, F))) return 0;
    return ffn::plane_bytes(ctx, N, D, backward ? 2 * F : F, backward != 0);
}

int rbk_gated_ffn_plan(rbk_ctx* ctx, int N, int D, int F, int backward, rbk_ffn_plan* plan) {
    const char* who = "rbk_gated_ffn_plan";
    RBK_TRY(ffn::check_sizes(who, N, D, F, RBK_ACT_SILU));
    RBK_REQUIRE(ctx && plan, "%s: ctx or plan is NULL", who);
    RBK_REQUIRE(N > 0, "%s: no rows", who);
    if (!backward && ffn::few(N, D, F)) {
        for (int i = 0; i < 2; ++i) plan->product[i] = {RBK_FFN_ROWS, ffn::few_wide(ctx, i ? D : F, i == 0), 1};
        return RBK_OK;
    }
    const int K = backward ? 2 * F : F;                      // of the second product
    auto& p = plan->product;
    p[0] = {RBK_FFN_PAIRS, 256, 1};
    if (mid_serves(ctx, backward ? kMidGluBwd : kMidGlu, N, F, D, backward != 0, &p[0].cols, &p[0].parts))
        p[0].kernel = RBK_FFN_TILES;
    p[1] = {RBK_FFN_PAIRS, 256, gemm_store_splits(ctx, N, D, K)};
    if (mid_serves(ctx, kMidStore, N, D, K, backward != 0, &p[1].cols, &p[1].parts)) p[1].kernel = RBK_FFN_TILES;
    return RBK_OK;
}

int rbk_gated_ffn_fwd(rbk_ctx* ctx, const rbk_ffn_args* a, void* stream) {
    const char* who = "rbk_gated_ffn_fwd";
    RBK_REQUIRE(a, "%s: args is NULL", who);
    RBK_TRY(ffn::check_sizes(who, a->N, a->D, a->F, a->act));
    RBK_TRY(ffn::check_ptr(who, "bgu", a->bgu, true));
    RBK_TRY(ffn::check_ptr(who, "bd", a->bd, true));
    if (a->N) {
        RBK_TRY(ffn::check_ptr(who, "x", a->x, false, a->ldx, a->D));
        RBK_TRY(ffn::check_ptr(who, "wgu", a->wgu, false));
        RBK_TRY(ffn::check_ptr(who, "wd", a->wd, false));
        RBK_TRY(ffn::check_ptr(who, "residual", a->residual, true, a->ldr, a->D));
        RBK_TRY(ffn::check_ptr(who, "y", a->y, false, a->ldy, a->D));
        RBK_TRY(ffn::check_ptr(who, "gu", a->gu, true));
        RBK_TRY(ffn::check_ptr(who, "h", a->h, false));
        RBK_TRY(ffn::check_ptr(who, "ws", a->ws, true));
    }
    RBK_TRY(check_device(ctx, who));
    if (!a->N) return RBK_OK;
    cudaStream_t st = as_stream(stream);
    if (ffn::few(a->N, a->D, a->F)) {
        ffn::Params p = {};
        p.N = a->N; p.R = a->F; p.K = a->D;
        p.w = (const half*)a->wgu;
        p.x = (const half*)a->x; p.ldx = a->ldx;
        p.bias = (const half*)a->bgu;
        p.out = (half*)a->h; p.ldo = a->F;
        p.gu = (half*)a->gu;
        p.act = a->act;
        RBK_TRY(ffn::few_rows<true>(ctx, p, st));
        ffn::Params d = {};
        d.N = a->N; d.R = a->D; d.K = a->F;
        d.w = (const half*)a->wd;
        d.x = (const half*)a->h; d.ldx = a->F;
        d.bias = (const half*)a->bd;
        d.residual = (const half*)a->residual; d.ldr = a->ldr;
        d.out = (half*)a->y; d.ldo = a->ldy;
        // The kernel before is the one above, which began only when everything before it had ended and writes no
        // weights: wd is as it will be, h is not.
        d.early = 1;
        return ffn::few_rows<false>(ctx, d, st);
    }
    void* ws = a->ws;
    const int64_t need = ffn::plane_bytes(ctx, a->N, a->D, a->F, 0);
    RBK_TRY(ffn::check_ws(who, ws, a->ws_bytes, need));
    if (!ws && need) RBK_TRY(ctx_scratch(ctx, need, &ws));
    RBK_TRY(mid_glu_fwd(ctx, a->h, a->gu, a->x, a->ldx, a->wgu, a->bgu, a->N, a->D, a->F, a->act, st));
    rbk_gemm_desc d = {};
    d.M = a->N; d.N = a->D; d.K = a->F;
    d.A = a->h; d.lda = a->F;
    d.B = a->wd; d.ldb = a->F;
    d.C = a->y; d.ldc = a->ldy;
    d.epilogue = RBK_EPI_STORE_F16;
    d.bias = a->bd;
    d.aux = a->residual; d.ld_aux = a->residual ? a->ldr : 0;
    d.alpha = 1.0f;
    // wd is as it will be: the kernel before, of this call, began after all before it had ended and writes none of it
    return mid_store(ctx, &d, (float*)ws, 1, st);
}

int rbk_gated_ffn_bwd(rbk_ctx* ctx, const rbk_ffn_bwd_args* a, void* stream) {
    const char* who = "rbk_gated_ffn_bwd";
    RBK_REQUIRE(a, "%s: args is NULL", who);
    RBK_TRY(ffn::check_sizes(who, a->N, a->D, a->F, a->act));
    RBK_REQUIRE(a->dwgu || !a->dbgu, "%s: dbgu needs dwgu", who);
    RBK_REQUIRE(a->dwd || !a->dbd, "%s: dbd needs dwd", who);
    RBK_TRY(ffn::check_ptr(who, "dwgu", a->dwgu, true));
    RBK_TRY(ffn::check_ptr(who, "dwd", a->dwd, true));
    if (a->N) {
        RBK_TRY(ffn::check_ptr(who, "dy", a->dy, false, a->lddy, a->D));
        RBK_TRY(ffn::check_ptr(who, "x", a->x, !a->dwgu, a->ldx, a->D));
        RBK_TRY(ffn::check_ptr(who, "gu", a->gu, false));
        RBK_TRY(ffn::check_ptr(who, "wgu", a->wgu, !a->dx));
        RBK_TRY(ffn::check_ptr(who, "wd", a->wd, false));
        RBK_TRY(ffn::check_ptr(who, "h", a->h, !a->recompute_h && !a->dwd));
        RBK_TRY(ffn::check_ptr(who, "dgu", a->dgu, false));
        RBK_TRY(ffn::check_ptr(who, "dx", a->dx, true, a->lddx, a->D));
        RBK_TRY(ffn::check_ptr(who, "ws", a->ws, true));
    }
    RBK_TRY(check_device(ctx, who));
    if (!a->N) return RBK_OK;
    const int64_t need = a->dx ? ffn::plane_bytes(ctx, a->N, a->D, 2 * a->F, 1) : 0;
    RBK_TRY(ffn::check_ws(who, a->ws, a->ws_bytes, need));
    cudaStream_t st = as_stream(stream);
    RBK_TRY(mid_glu_bwd(ctx, a->dgu, a->recompute_h ? a->h : nullptr, a->dy, a->lddy, a->wd, a->gu, a->N, a->D, a->F,
                          a->act, st));
    // the weight gradients before dx, which may then lie over dy or x
    rbk_gemm_desc d = {};
    d.K = a->N;
    d.a_major = d.b_major = 1;
    d.epilogue = RBK_EPI_ACC_F32;
    d.alpha = 1.0f;
    if (a->dwgu) {
        d.M = 2 * a->F; d.N = a->D;
        d.A = a->dgu; d.lda = 2 * a->F;
        d.B = a->x; d.ldb = a->ldx;
        d.C = a->dwgu; d.ldc = a->D;
        d.dbias_rows = a->dbgu;
        RBK_TRY(rbk_gemm(ctx, &d, stream));
    }
    if (a->dwd) {
        d.M = a->D; d.N = a->F;
        d.A = a->dy; d.lda = a->lddy;
        d.B = a->h; d.ldb = a->F;
        d.C = a->dwd; d.ldc = a->F;
        d.dbias_rows = a->dbd;
        RBK_TRY(rbk_gemm(ctx, &d, stream));
    }
    if (!a->dx) return RBK_OK;
    void* ws = a->ws;
    if (!ws && need) RBK_TRY(ctx_scratch(ctx, need, &ws));        // after the GEMMs above, which may move it
    rbk_gemm_desc e = {};
    e.M = a->N; e.N = a->D; e.K = 2 * a->F;
    e.A = a->dgu; e.lda = 2 * a->F;
    e.B = a->wgu; e.ldb = a->D; e.b_major = 1;                // B(n, k = gate or up row) = Wgu[k, n]
    e.C = a->dx; e.ldc = a->lddx;
    e.epilogue = RBK_EPI_STORE_F16;
    e.alpha = 1.0f;
    return mid_store(ctx, &e, (float*)ws, !a->dwgu && !a->dwd, st);
}

}  // extern "C"
