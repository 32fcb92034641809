// ffn.cu — the gated feed-forward block, forward and backward.
//
//   gate = x Wg^T + bg,  up = x Wu^T + bu,  h = act(gate) * up,  y = h Wd^T + bd + residual
//   dh = dy Wd,  dgate = dh up act'(gate),  dup = dh act(gate),  dx = dgate Wg + dup Wu
//
// Many rows: tensor bound (6 N D F FLOP each way).  The CTA-pair GEMM of gemm.cu with epilogues of its own
// makes h (gate and up tiles share one accumulator) and dgu; the other products are plain GEMMs.
// Few rows: the weights, 6 D F bytes, are read once and that is the cost.  The kernels below stream them.
#include "common.cuh"

namespace rbk {
namespace ffn {

// ---------------------------------------------------------------- few rows ----
// out[n, r] = sum_k w[r, k] x[n, k] for up to 8 NT rows n: a CTA takes 16 rows r of the weights (GLU: 16 of
// the gate and the same 16 of the up projection), its 8 warps take every eighth 64-wide block of k, and the
// warps' sums are added in warp order through shared memory.  mma.sync m16n8k16 with the weights as the
// 16-row operand: the tensor pipe is idle next to the memory, what matters is that a lane's fragment is a
// whole 16-byte load.  The k order within a block is permuted for that, alike on both sides: lane 4 g + t
// holds k = 8 t .. 8 t + 7 (and 32 + 8 t ..) of row g, and MMA m of the two that use it takes its elements
// 4 m .. 4 m + 3.
constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kRows = 16;                                // weight rows of a CTA
constexpr int kMaxTokens = 32;

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ldg_stream(const half* p, bool on) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (on)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p));
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
};

template <int NT, bool GLU>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const Params p) {
    constexpr int MATS = GLU ? 2 : 1;
    __shared__ float sums[kWarps][MATS][kRows][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.x * kRows;
    grid_dependency_sync();
    // rows past the end read the last row; what they give is not stored
    const half* w0 = p.w + (size_t)min(r0 + g, p.R - 1) * p.K;
    const half* w1 = p.w + (size_t)min(r0 + g + 8, p.R - 1) * p.K;
    const size_t up = (size_t)p.R * p.K;
    float acc[MATS][NT][4] = {};
    for (int kb = warp * 64; kb < p.K; kb += kWarps * 64) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int k = kb + 32 * hf + 8 * t;
            const bool on = k < p.K;
            uint4 a[MATS][2], b[NT];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                a[m][0] = ldg_stream(w0 + m * up + k, on);
                a[m][1] = ldg_stream(w1 + m * up + k, on);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int n = 8 * j + g;
                b[j] = on && n < p.N ? *reinterpret_cast<const uint4*>(p.x + n * p.ldx + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_16816(acc[m][j], a[m][0].x, a[m][1].x, a[m][0].y, a[m][1].y, b[j].x, b[j].y);
                    mma_16816(acc[m][j], a[m][0].z, a[m][1].z, a[m][0].w, a[m][1].w, b[j].z, b[j].w);
                }
        }
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            sums[warp][m][g][8 * j + 2 * t] = acc[m][j][0];
            sums[warp][m][g][8 * j + 2 * t + 1] = acc[m][j][1];
            sums[warp][m][g + 8][8 * j + 2 * t] = acc[m][j][2];
            sums[warp][m][g + 8][8 * j + 2 * t + 1] = acc[m][j][3];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * 8 * NT; i += kThreads) {
        const int r = i % kRows, n = i / kRows, row = r0 + r;
        if (n >= p.N || row >= p.R) continue;
        float v[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            v[m] = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) v[m] += sums[w][m][r][n];
            if (p.bias) v[m] += __half2float(p.bias[m * p.R + row]);
        }
        if constexpr (GLU) {
            if (p.gu) {
                p.gu[(size_t)n * 2 * p.R + row] = __float2half_rn(v[0]);
                p.gu[(size_t)n * 2 * p.R + p.R + row] = __float2half_rn(v[1]);
            }
            v[0] = glu_act(v[0], p.act) * v[1];
        } else if (p.residual) {
            v[0] += __half2float(p.residual[n * p.ldr + row]);
        }
        p.out[n * p.ldo + row] = __float2half_rn(v[0]);
    }
}

template <bool GLU>
int few_rows(rbk_ctx* ctx, const Params& p, cudaStream_t st) {
    const dim3 grid((p.R + kRows - 1) / kRows), block(kThreads);
    ProfScope prof(ctx, st, kCatGemm, (GLU ? 4.0 : 2.0) * p.N * (double)p.R * p.K, 0);
    if (p.N <= 8) RBK_CUDA(launch_pdl(few_rows_kernel<1, GLU>, grid, block, 0, st, p));
    else if (p.N <= 16) RBK_CUDA(launch_pdl(few_rows_kernel<2, GLU>, grid, block, 0, st, p));
    else RBK_CUDA(launch_pdl(few_rows_kernel<4, GLU>, grid, block, 0, st, p));
    RBK_LAUNCHED("few_rows_kernel");
    return RBK_OK;
}

static int check_sizes(const char* who, int N, int D, int F, int act) {
    RBK_REQUIRE(N >= 0, "%s: negative N", who);
    RBK_REQUIRE(D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0 && F <= (1 << 29),
                "%s: D and F must be positive multiples of 8 (D=%d F=%d)", who, D, F);
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

}  // namespace ffn
}  // namespace rbk

using namespace rbk;

extern "C" {

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
    }
    RBK_TRY(check_device(ctx, who));
    if (!a->N) return RBK_OK;
    cudaStream_t st = as_stream(stream);
    if (a->N <= ffn::kMaxTokens) {
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
        return ffn::few_rows<false>(ctx, d, st);
    }
    RBK_TRY(glu_fwd_tiles(ctx, a->h, a->gu, a->x, a->ldx, a->wgu, a->bgu, a->N, a->D, a->F, a->act, st));
    rbk_gemm_desc d = {};
    d.M = a->N; d.N = a->D; d.K = a->F;
    d.A = a->h; d.lda = a->F;
    d.B = a->wd; d.ldb = a->F;
    d.C = a->y; d.ldc = a->ldy;
    d.epilogue = RBK_EPI_STORE_F16;
    d.bias = a->bd;
    d.aux = a->residual; d.ld_aux = a->residual ? a->ldr : 0;
    d.alpha = 1.0f;
    return rbk_gemm(ctx, &d, stream);
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
    }
    RBK_TRY(check_device(ctx, who));
    if (!a->N) return RBK_OK;
    RBK_TRY(glu_bwd_tiles(ctx, a->dgu, a->recompute_h ? a->h : nullptr, a->dy, a->lddy, a->wd, a->gu, a->N, a->D, a->F,
                          a->act, as_stream(stream)));
    if (a->dx) {
        rbk_gemm_desc d = {};
        d.M = a->N; d.N = a->D; d.K = 2 * a->F;
        d.A = a->dgu; d.lda = 2 * a->F;
        d.B = a->wgu; d.ldb = a->D; d.b_major = 1;            // B(n, k = gate or up row) = Wgu[k, n]
        d.C = a->dx; d.ldc = a->lddx;
        d.epilogue = RBK_EPI_STORE_F16;
        d.alpha = 1.0f;
        RBK_TRY(rbk_gemm(ctx, &d, stream));
    }
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
    return RBK_OK;
}

}  // extern "C"
