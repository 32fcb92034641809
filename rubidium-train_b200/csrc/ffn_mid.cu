// ffn_mid.cu — the gated feed-forward block's products where the 256 x 256 tiles of gemm.cu are too few for the
// machine: some tens to a few hundred rows, or narrow blocks.
//
// One CTA has 128 rows and `bn` columns of a product (kGlu: bn / 2 of the gate and the same of the up projection),
// and of K one part of S (gate and up: all of it; dgu: up to 2 parts; y and dx: up to 8): the S CTAs of a tile are a
// cluster.  Each leaves its FP32 sums in its own shared memory, and every CTA of the cluster adds a part of the tile
// from all of them, in order, through distributed shared memory, applies the epilogue and stores it: one launch, no
// planes in global memory, and two runs give the same bits.
// Bound by latency: the first loads, a chain of K blocks with what an SM has in flight (96 KB, 200 where one CTA has
// it), the exchange and the drain.  100 rows, D 2048, F 5632: 28 us for the forward's two launches (floor 10.7); each
// uses 11 to 19% of the tensor pipe and 16 to 30% of L2 and HBM.
#include <algorithm>

#include "tc.cuh"

namespace rbk {
namespace mid {

using namespace tc;

constexpr int kLong = 17;                                    // k blocks of a CTA from which on it is better off alone
constexpr int BM = 128, BK = 64, kThreads = 320;             // a TMA warp, an MMA warp, eight that read TMEM
constexpr int kHead = 1024;                                  // barriers
// Shared memory of which two CTAs fit an SM (228 KB, 1 KB of each for the system), the least that one takes: a CTA
// holds up to 256 columns of TMEM while it waits for the others of its cluster, so that no SM may take more CTAs than
// its 512 columns serve, this kernel's or the CTA pairs' (512 columns, at least 193 KB) of another stream.
constexpr int kHalfSm = 113 << 10, kAllSm = 227 << 10;
enum { kGlu = kMidGlu, kGluBwd = kMidGluBwd, kStore = kMidStore };

struct Params {
    int M, N, K;                   // rows, output columns (F; store: D), inner extent
    int bn, m_blocks, k_blocks, kb_per, stages, rows_box;
    uint32_t tx;                   // bytes of a K block's loads
    int b_mn;                      // B(n, k) is contiguous in n
    int early;                     // B may be read before the kernel before this one has ended
    int act;
    const half *bias, *bias2;      // of the output columns; kGlu: of gate and up
    const half* aux; long long ld_aux;       // kStore: residual; kGluBwd: gate | up, [M, 2N]
    half* out; long long ldo;      // y or dx; kGlu, kGluBwd: h, [M, N], or NULL
    half* gu;                      // kGlu: gate | up, or NULL; kGluBwd: dgate | dup; [M, 2N]
    int* err;
    uint64_t wait_ns;              // limit of a wait
};

// act(z) and act'(z), glu_act's formulas.
__device__ __forceinline__ void glu_both(float z, int act, float& a, float& da) {
    const float zz = z * z;
    const float r = act == RBK_ACT_GELU ? kGluC * z * (1.0f + kGluA * zz) : z;
    const float s = rcp_fast(1.0f + ex2_fast(-kGluLog2e * r));
    a = z * s;
    float e = a * (1.0f - s);
    if (act == RBK_ACT_GELU) e *= kGluC + 3.0f * kGluC * kGluA * zz;
    da = s + e;
}

__device__ __forceinline__ float4 lds_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// Eight sums at offset `off` of the cluster's tiles, in the order of its CTAs.
template <int S>
__device__ __forceinline__ void sum8(float* v, const uint32_t* tile, uint32_t off) {
    float4 a[S], b[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        a[s] = lds_cluster(tile[s] + off);
        b[s] = lds_cluster(tile[s] + off + 16);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        v[0] += a[s].x; v[1] += a[s].y; v[2] += a[s].z; v[3] += a[s].w;
        v[4] += b[s].x; v[5] += b[s].y; v[6] += b[s].z; v[7] += b[s].w;
    }
}
__device__ __forceinline__ void add8(float* v, const half* p) {
    float t[8];
    h8_to_f(*reinterpret_cast<const uint4*>(p), t);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += t[e];
}

template <int EPI, int S>
__global__ void __launch_bounds__(kThreads, 2) mid_kernel(const __grid_constant__ CUtensorMap tmA,
                                                          const __grid_constant__ CUtensorMap tmB, const Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = su32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    const uint32_t ring = base + kHead;
    const int stage_bytes = BM * BK * 2 + p.bn * BK * 2, pitch = p.bn + 4;
    auto full_bar = [&](int s) { return base + 8u * s; };
    auto empty_bar = [&](int s) { return base + 64u + 8u * s; };
    const uint32_t done_bar = base + 128u;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + 136);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + 144);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % S, tile = blockIdx.x / S;
    const int m0 = tile % p.m_blocks * BM, nt = tile / p.m_blocks;
    const int n0 = nt * (EPI == kGlu ? p.bn / 2 : p.bn);     // first output column
    const int kb0 = split * p.kb_per, kb1 = min(p.k_blocks, kb0 + p.kb_per);
    const int rows = min(BM, p.M - m0);
    uint32_t cols = 32;                                      // of TMEM: a power of two
    while ((int)cols < p.bn) cols *= 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    }
    if (warp == 1) tmem_alloc(tmem_slot, cols);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    auto load_b = [&](int s, int kb) {
        const uint32_t sb = ring + s * stage_bytes + BM * BK * 2;
        if (EPI == kGlu) {                                   // gate rows, then the same up rows
            tma_load_2d(sb, &tmB, full_bar(s), kb * BK, n0);
            tma_load_2d(sb + p.bn / 2 * BK * 2, &tmB, full_bar(s), kb * BK, p.N + n0);
        } else if (!p.b_mn) {
            tma_load_2d(sb, &tmB, full_bar(s), kb * BK, n0);
        } else {
            for (int j = 0; j < p.bn / 64; ++j) tma_load_2d(sb + 8192 * j, &tmB, full_bar(s), n0 + 64 * j, kb * BK);
        }
    };
    auto load_a = [&](int s, int kb) { tma_load_2d(ring + s * stage_bytes, &tmA, full_bar(s), kb * BK, m0); };
    int issued = 0;                                          // K blocks whose loads thread 0 has issued

    // Everybody but the producer waits here for what came before; bounded waits start after that.
    if (warp != 0 || lane != 0) grid_dependency_sync();
    if (warp == 0) {
        if (lane == 0) {
            const int nk = kb1 - kb0, first = min(nk, p.stages);
            if (!p.early) grid_dependency_sync();
            for (int i = 0; i < first; ++i) {
                mbar_expect_tx(full_bar(i), p.tx);
                load_b(i, kb0 + i);
            }
            if (p.early) grid_dependency_sync();
            for (int i = 0; i < first; ++i) load_a(i, kb0 + i);
            int s = 0;
            uint32_t phase = 0;
            for (issued = first; issued < nk; ++issued) {
                if (!mbar_wait(empty_bar(s), phase, abort_flag, p.wait_ns)) break;
                mbar_expect_tx(full_bar(s), p.tx);
                load_b(s, kb0 + issued);
                load_a(s, kb0 + issued);
                if (++s == p.stages) { s = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_f16(p.bn, 0, p.b_mn);
            const uint32_t lbo = p.b_mn ? 8192u : 16u, step = p.b_mn ? 2048u : 32u;
            int s = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(full_bar(s), phase, abort_flag, p.wait_ns)) break;
                fence_after();
                const uint32_t sa = ring + s * stage_bytes, sb = sa + BM * BK * 2;
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                    mma_f16(tmem, sdesc(sa + k * 32, 16, 1024), sdesc(sb + k * step, lbo, 1024), idesc, kb > kb0 || k > 0);
                mma_commit(empty_bar(s));
                if (++s == p.stages) { s = 0; phase ^= 1; }
            }
            mma_commit(done_bar);
        }
    }
    __syncwarp();
    if (warp >= 2) {
        // the tile's sums to shared memory, over the operands' slots: all MMAs have read them
        if (__all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag, p.wait_ns) && !*abort_flag)) {
            fence_after();
            const int q = warp & 3, row = q * 32 + lane;
            if (q * 32 < rows) {
                const uint32_t t = tmem + ((uint32_t)(q * 32) << 16);
                const uint32_t dst = ring + row * pitch * 4;
                for (int c = (warp - 2) / 4 * 16; c < p.bn; c += 32) {
                    uint32_t r[16];
                    tmem_ld16(t + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; k += 4)          // a warp's 32 rows have room, those behind the last too
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (c + k) * 4), "r"(r[k]),
                                     "r"(r[k + 1]), "r"(r[k + 2]), "r"(r[k + 3]) : "memory");
                }
            }
            fence_before();
        }
    }
    __syncwarp();
    if (S > 1) cluster_sync();
    else __syncthreads();
    fence_after();

    uint32_t part[S];
#pragma unroll
    for (int s = 0; s < S; ++s) part[s] = mapa_shared(ring, s);
    const int per_row = (EPI == kGlu ? p.bn / 2 : p.bn) / 8;
    for (int i = split * kThreads + threadIdx.x; i < rows * per_row; i += S * kThreads) {
        const int row = i / per_row, c = (i - row * per_row) * 8, n = n0 + c, m = m0 + row;
        if (n >= p.N) continue;
        const uint32_t off = (row * pitch + c) * 4;
        float v[8];
        sum8<S>(v, part, off);
        if constexpr (EPI == kGlu) {
            float u[8];
            sum8<S>(u, part, off + p.bn / 2 * 4);
            if (p.bias) {
                add8(v, p.bias + n);
                add8(u, p.bias2 + n);
            }
            if (p.gu) {
                half* g = p.gu + (size_t)m * 2 * p.N + n;
                *reinterpret_cast<uint4*>(g) = f_to_h8(v);
                *reinterpret_cast<uint4*>(g + p.N) = f_to_h8(u);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = glu_act(v[e], p.act) * u[e];
            *reinterpret_cast<uint4*>(p.out + (size_t)m * p.ldo + n) = f_to_h8(v);
        } else if constexpr (EPI == kGluBwd) {
            const half* src = p.aux + (size_t)m * 2 * p.N + n;
            float g[8], u[8], h[8];
            h8_to_f(*reinterpret_cast<const uint4*>(src), g);
            h8_to_f(*reinterpret_cast<const uint4*>(src + p.N), u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float a, da;
                glu_both(g[e], p.act, a, da);
                h[e] = a * u[e];
                g[e] = v[e] * u[e] * da;
                u[e] = v[e] * a;
            }
            half* dst = p.gu + (size_t)m * 2 * p.N + n;
            *reinterpret_cast<uint4*>(dst) = f_to_h8(g);
            *reinterpret_cast<uint4*>(dst + p.N) = f_to_h8(u);
            if (p.out) *reinterpret_cast<uint4*>(p.out + (size_t)m * p.ldo + n) = f_to_h8(h);
        } else {
            if (p.bias) add8(v, p.bias + n);
            if (p.aux) add8(v, p.aux + (size_t)m * p.ld_aux + n);
            *reinterpret_cast<uint4*>(p.out + (size_t)m * p.ldo + n) = f_to_h8(v);
        }
    }

    __syncwarp();                                            // lanes leave the loop at different times
    if (S > 1) cluster_sync();                               // the other CTAs have read this one's sums
    else __syncthreads();
    // Every role has ended, so the flag is what it will be.  After a timeout the copies under way, which may be the last
    // that were issued for each slot, land before the CTA ends, or 4 ms pass.
    if (threadIdx.x == 0 && *abort_flag) {
        for (int n = max(0, issued - p.stages), t = 0; n < issued; ++n)
            while (t < 200 && !mbar_try_suspend(full_bar(n % p.stages), n / p.stages & 1, 20000u)) ++t;
        atomicExch(p.err, RBK_ERR_TIMEOUT);
    }
    if (warp == 1) tmem_free(tmem, cols);
}

template <int EPI, int S>
int launch_s(rbk_ctx* ctx, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int tiles, int smem,
             cudaStream_t st) {
    static int configured_device = -1;   // attribute is per device; one device per process
    if (configured_device != ctx->device) {
        RBK_CUDA(cudaFuncSetAttribute(mid_kernel<EPI, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kAllSm));
        configured_device = ctx->device;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(tiles * S);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = set_pdl(attr, 1);
    RBK_CUDA(cudaLaunchKernelEx(&cfg, mid_kernel<EPI, S>, ta, tb, p));
    RBK_LAUNCHED("mid_kernel");
    return RBK_OK;
}

template <int EPI>
int launch(rbk_ctx* ctx, int S, const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int tiles, int smem,
           cudaStream_t st) {
    // the parts of K that plan() gives: gate and up one, dgu one or two, y and dx up to eight
    if (S == 1) return launch_s<EPI, 1>(ctx, ta, tb, p, tiles, smem, st);
    if constexpr (EPI != kGlu)
        if (S == 2) return launch_s<EPI, 2>(ctx, ta, tb, p, tiles, smem, st);
    if constexpr (EPI == kStore) {
        if (S == 4) return launch_s<EPI, 4>(ctx, ta, tb, p, tiles, smem, st);
        if (S == 8) return launch_s<EPI, 8>(ctx, ta, tb, p, tiles, smem, st);
    }
    set_error("mid_kernel: no instance for %d parts of K", S);
    return RBK_ERR_INVALID;
}

// The tiles of a call, or bn 0: those of gemm.cu.  Two CTAs fit an SM; what is wanted is one round of them with the
// widest spread, and of K parts that are still worth a cluster's exchange.  Measured, whole calls, forward:
//   D 768, F 2048: 100 rows 20.9 -> 13.8 us, 384 rows 21.6 -> 18.7; 1024 rows 23.8 -> 20.8
//   D 2048, F 5632: 100 rows 34.8 -> 28.2, 384 rows 48.9 -> 38.7; 640 rows stay (50.9; tiles of 192 columns 74)
//   D 512, F 1024: 100 rows 17.6 -> 10.9, 1024 rows 18.4 -> 14.1
// backward (dgu, h, dx):
//   D 768, F 2048: 100 rows 25.1 -> 15.7; 1024 rows 30.2 -> 27.0
//   D 2048, F 5632: 100 rows 40.3 -> 32.5, 384 rows 48.2 -> 45.0; 512 rows stay (49.9; 53.3 with 64 columns)
//   D 512, F 1024: 384 rows 22.8 -> 17.7
// Over 96 shapes (33 to 2048 rows, D 256 to 2048, F 256 to 5632) the forward took 0.79 of its time and the backward
// 0.76 (geometric means), the worst 1.07 (353 rows, D 760, F 3832: 27.6 us, 25.8 on the larger tiles).
struct Plan {
    int bn, S;
};
static Plan plan(rbk_ctx* ctx, int epi, int M, int N, int K, int b_mn) {
    const long long m = (M + BM - 1) / BM, slots = 2LL * ctx->num_sms;
    const int kb = (K + BK - 1) / BK;
    const auto ctas = [&](long long cols, int bn) { return m * ((cols + bn - 1) / bn); };
    // Clusters of four do not fill the machine: 288 CTAs of them are two rounds (dx of 768 rows, D 768,
    // F 2048: 36 us and 29 with the tiles of gemm.cu), 264 are one.
    const auto fit = [&](long long cols, int least, int most, int S, long long slots) {   // the narrowest one-round tiles
        for (int bn = least; bn <= most; bn += 16)
            if (ctas(cols, bn) * S <= (S >= 4 ? slots * 9 / 10 : slots)) return bn;
        return 0;
    };
    // Microseconds by what bounds each: here an SM's loads, 100 KB a microsecond (rows of K that do not start on 128 bytes
    // cost a third more), there 0.45 us a k block and wave and, if K is split, the planes.
    const bool ragged = K % 64 != 0;
    const auto here = [&](int bn, int S, long long n) {
        return 4.0 + (S > 1) + (n > ctx->num_sms ? 2 : 1) * ((kb + S - 1) / S) * (16.0 + bn / 8.0) / 100.0 * (ragged ? 1.35 : 1.0);
    };
    const auto there = [&](long long units, int splits) {
        const int pairs = ctx->num_sms / 2;
        return 7.5 + (units * splits + pairs - 1) / pairs * ((kb + splits - 1) / splits) * (ragged ? 0.495 : 0.45) +
               (splits > 1 ? 2.5 + 8e-7 * splits * M * N : 0.0);
    };
    const long long m2 = (M + 2 * BM - 1) / (2 * BM);
    Plan p = {0, 1};
    if (epi == kGlu) {
        // long in K: one CTA for an SM, or two (286 rows, D 1192, F 2040, whole call: 23.7 us so, 28.1 with two)
        if (kb >= kLong) p.bn = fit(2LL * N, 48, 256, 1, slots / 2);
        if (!p.bn) p.bn = fit(2LL * N, kb >= 24 ? 64 : 48, 160, 1, slots);
        if (p.bn && here(p.bn, 1, ctas(2LL * N, p.bn)) > there(m2 * ((N + 127) / 128), 1)) p.bn = 0;
    } else if (epi == kGluBwd) {
        // One round of two CTAs an SM with two parts of K; else one round of CTAs alone in an SM (192 columns); else one of
        // two an SM with K whole.  Whole backwards, 64 columns x 2 parts | 192 x 2 | 64 whole | CTA pairs:
        //   100 rows, D 1024, F 2048:  18.0 | 21.7 | 20.0 | 26.4        200 rows, D 2048, F 4736:  35.4 | 36.5 | 37.0 | 41.0
        //   200 rows, D 2048, F 5632:  45.7 | 39.3 | 42.2 | 44.1        300 rows, D 1024, F 4736:  36.5 | 34.5 | 30.4 | 33.8
        // Over 119 shapes (100 to 1500 rows, D 256 to 4096) within 0.2% of the best of the four on average, the worst
        // 14% off it (200 rows, D 256, F 5632: 25.9, 22.6 with 64 columns in two parts, two rounds).
        if (2 * ctas(N, 64) <= slots) p = {64, 2};
        else if (4 * ctas(N, 192) <= slots) p = {192, 2};
        else if (ctas(N, 64) <= slots) p = {64, 1};
    } else if (!b_mn) {
        p.S = m <= 2 || kb > 48 ? 4 : 2;
        while (p.S < 8 && kb >= 32 * p.S && ctas(N, 32) * 2 * p.S <= (m <= 2 ? slots / 2 : slots)) p.S *= 2;
        if (m <= 2 || kb <= 32 * p.S) p.bn = fit(N, m <= 2 ? 32 : 48, 80, p.S, slots);
        if (p.bn && here(p.bn, p.S, ctas(N, p.bn) * p.S) > there(m2 * ((N + 255) / 256), gemm_store_splits(ctx, M, N, K))) p.bn = 0;
    } else {
        // dx: K is twice F, and its rows of B come 64 columns at a time.  t tiles.  Two parts where K is short and the
        // tiles many; eight where they are few and K is worth the exchange; four between; CTA pairs, which share K out
        // over planes, where K is long or the tiles are enough for them.  Whole backwards, 2 | 4 | 8 parts | CTA pairs:
        //   t 64, 500 rows, D 1024, F 1024:  17.4 | 20.1 | 33.3 | 20.5     t 8, 100 rows, D 512, F 2304:  20.8 | 15.9 | 14.9 | 17.4
        //   t 48, 300 rows, D 1024, F 2560:  26.9 | 24.5 | 35.5 | 25.6     t 48, 300 rows, D 1024, F 5632:  43.8 | 34.4 | 45.9 | 32.1
        // Over 143 shapes (t 8 to 144, 8 to 176 k blocks) within 2% of the best of the four on average and 0.94 of the
        // pairs' time; the worst 19% off it (t 24, 200 rows, D 768, F 1792: 20.3, and 17.0 with four parts).
        const long long t = ctas(N, 64);
        if (kb <= 32 && 8 * t > slots) {
            if (2 * t <= slots) p = {64, 2};
        } else if (8 * t <= slots && kb >= 32 && kb <= 72) {
            p = {64, 16 * t <= slots + slots / 3 ? 8 : 4};
        } else if (16 * t <= 3 * slots + slots / 2 && kb <= 96) {
            p = {64, 4};
        }
    }
    while (p.S > 1 && (kb < 4 * p.S || (p.S - 1) * ((kb + p.S - 1) / p.S) >= kb)) p.S /= 2;
    return p;
}

template <int EPI>
int run(rbk_ctx* ctx, Params p, const Plan& pl, const void* A, int64_t lda, const void* B, int64_t ldb, cudaStream_t st) {
    p.bn = pl.bn;
    p.m_blocks = (p.M + BM - 1) / BM;
    p.k_blocks = (p.K + BK - 1) / BK;
    p.kb_per = (p.k_blocks + pl.S - 1) / pl.S;
    p.rows_box = std::min(BM, (p.M + 7) / 8 * 8);
    const int per = EPI == kGlu ? p.bn / 2 : p.bn;
    const int tiles = p.m_blocks * ((p.N + per - 1) / per);
    const int stage = BM * BK * 2 + p.bn * BK * 2;
    // At most one CTA for an SM, and long in K: all of its shared memory for what is in flight (629 rows, D 1736, F 864:
    // forward 27.4 -> 21.6 us; 131 rows, D 1448, F 992 23.4 -> 18.8).  Short ones are better off beside the next
    // kernel's (100 rows, D 768, F 2048: 13.8, and 14.9 alone), and so are few (dx of 100 rows, D 1024, F 2816, 64 CTAs:
    // backward 18.9, and 20.1 alone; of 200 rows, 128 CTAs: 24.4, and 22.0 alone).
    const int ctas = tiles * pl.S, room = pl.S >= 4 ? ctx->num_sms * 9 / 10 : ctx->num_sms;
    const bool alone = p.kb_per >= kLong && ctas <= room && (EPI != kStore || 2 * ctas > ctx->num_sms);
    p.stages = std::min({8, p.kb_per, std::max(3, ((alone ? kAllSm : kHalfSm) - 1024 - kHead) / stage)});
    p.err = ctx->tickets + kGemmError;
    p.wait_ns = ctx->test_ffn_wait_ns ? ctx->test_ffn_wait_ns : kWaitTimeoutNs;
    p.tx = (p.rows_box + p.bn) * BK * 2 + (ctx->test_ffn_wait_ns ? 16 : 0);   // armed: more than will come
    ctx->test_ffn_wait_ns = 0;                               // the test setting covers one launch
    const int smem = std::max(kHalfSm, 1024 + kHead + std::max(p.stages * stage, (p.rows_box + 31) / 32 * 32 * (p.bn + 4) * 4));
    CUtensorMap ta, tb;
    RBK_TRY(make_tmap(&ta, A, p.K, p.M, lda, 64, p.rows_box));
    if (p.b_mn) RBK_TRY(make_tmap(&tb, B, p.N, p.K, ldb, 64, 64));
    else RBK_TRY(make_tmap(&tb, B, p.K, EPI == kGlu ? 2 * (uint64_t)p.N : p.N, ldb, 64, per));
    return launch<EPI>(ctx, pl.S, ta, tb, p, tiles, smem, st);
}

}  // namespace mid

bool mid_serves(rbk_ctx* ctx, int product, int M, int N, int K, int b_mn, int* cols, int* parts) {
    const mid::Plan p = mid::plan(ctx, product, M, N, K, b_mn);
    if (p.bn && cols) *cols = p.bn;
    if (p.bn && parts) *parts = p.S;
    return p.bn > 0;
}

int mid_glu_fwd(rbk_ctx* ctx, void* h, void* gu, const void* x, int ldx, const void* wgu, const void* bgu, int N, int D,
                int F, int act, cudaStream_t st) {
    const mid::Plan pl = mid::plan(ctx, mid::kGlu, N, F, D, 0);
    if (!pl.bn) return glu_fwd_tiles(ctx, h, gu, x, ldx, wgu, bgu, N, D, F, act, st);
    mid::Params p = {};
    p.M = N; p.N = F; p.K = D;
    p.act = act;
    p.bias = (const half*)bgu;
    p.bias2 = bgu ? p.bias + F : nullptr;
    p.out = (half*)h; p.ldo = F;
    p.gu = (half*)gu;
    ProfScope prof(ctx, st, kCatGemm, 4.0 * N * (double)D * F, 0);
    return mid::run<mid::kGlu>(ctx, p, pl, x, ldx, wgu, D, st);
}

int mid_glu_bwd(rbk_ctx* ctx, void* dgu, void* h, const void* dy, int lddy, const void* wd, const void* gu, int N, int D,
                int F, int act, cudaStream_t st) {
    const mid::Plan pl = mid::plan(ctx, mid::kGluBwd, N, F, D, 1);
    if (!pl.bn) return glu_bwd_tiles(ctx, dgu, h, dy, lddy, wd, gu, N, D, F, act, st);
    mid::Params p = {};
    p.M = N; p.N = F; p.K = D;
    p.b_mn = 1;                                              // B(n = f, k = d) = Wd[d, f]
    p.act = act;
    p.aux = (const half*)gu;
    p.out = (half*)h; p.ldo = F;
    p.gu = (half*)dgu;
    ProfScope prof(ctx, st, kCatGemm, 2.0 * N * (double)D * F, 1);
    return mid::run<mid::kGluBwd>(ctx, p, pl, dy, lddy, wd, F, st);
}

int mid_store(rbk_ctx* ctx, const rbk_gemm_desc* d, float* ws, int early, cudaStream_t st) {
    const mid::Plan pl = mid::plan(ctx, mid::kStore, d->M, d->N, d->K, d->b_major);
    if (!pl.bn) return gemm_store(ctx, d, ws, st);
    mid::Params p = {};
    p.M = d->M; p.N = d->N; p.K = d->K;
    p.b_mn = d->b_major;
    p.early = early;
    p.bias = (const half*)d->bias;
    p.aux = (const half*)d->aux; p.ld_aux = d->ld_aux;
    p.out = (half*)d->C; p.ldo = d->ldc;
    ProfScope prof(ctx, st, kCatGemm, 2.0 * d->M * (double)d->N * d->K, d->b_major ? 1 : 0);
    return mid::run<mid::kStore>(ctx, p, pl, d->A, d->lda, d->B, d->ldb, st);
}

}  // namespace rbk
