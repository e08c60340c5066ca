// k_xent.cu -- softmax cross entropy of the linear layer z = x w^T over a large
// vocabulary, and its gradient, without ever holding z.
//
//   x [n, dim], w [vocab, dim] (one row per class), label_i
//   lse_i  = log sum_v exp z_iv,      loss_i = lse_i - z_i,label
//   G_iv   = (exp(z_iv - lse_i) - [v = label_i]) dloss_i
//   dx     = G w  [n, dim],           dw = G^T x  [vocab, dim]
// A label outside [0, vocab) marks a row without a target: loss 0, G row 0.
//
// Three matrix products of 2 n vocab dim operations each, and z once more in
// the backward pass because it is not kept: 8 n vocab dim in all, on the
// tcgen05 tensor cores.  All go through one kernel, k_xgemm, with an epilogue
// each:
//   LSE  the maximum and the sum of exponentials of every row over the tile's
//        classes (8 bytes per row and tile instead of the logits) and the
//        label's logit; a small kernel joins the tiles;
//   G    G as bf16 for one piece of the vocabulary at a time;
//   OUT  dx += G_piece w_piece in f32, and dw_piece = G_piece^T x.
//
// Types.  bf16: the operands go to the tensor core as they are; G is rounded
// to bf16 once (2^-8 relative to each entry at most, like the operands of the
// products that follow it), sums are f32.  f32: every f32 value is the sum
// of three bf16 values, b0 = bf16(v), b1 = bf16(v - b0), b2 = bf16(v - b0 - b1)
// (exact but for values below 2^-110), and a product is the six partial
// products b_i b_j with i + j <= 2, the smallest first; the three left out are
// below 2^-24 of the product.  bf16 has f32's exponent range, so no scaling is
// needed, and six bf16 products cost what three TF32 products cost.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include "kernels.h"

#include <algorithm>

namespace nxv {

namespace {

using bf16 = __nv_bfloat16;

constexpr int BM = 128, BN = 256, BK = 64;  // BK bf16 = one 128-byte swizzle row
constexpr int ST = 4;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, ST_BYTES = A_BYTES + B_BYTES;
constexpr int SMEM = ST * ST_BYTES + 1024 + 256;
constexpr uint32_t TMEM_COLS = 512;  // two 128 x 256 f32 accumulators

__device__ int g_xent_error;

// ---- PTX ----------------------------------------------------------------------

__device__ __forceinline__ uint32_t su32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(su32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait (a few seconds at most); false when it runs out or when another
// warp of the CTA has given up.
__device__ __noinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* err) {
    for (uint32_t i = 0; i < (1u << 24); i++) {
        if (mbar_try(b, parity)) return true;
        if (i > 256) {
            if (*err) return false;
            __nanosleep(100);
        }
    }
    *err = 1;
    atomicExch(&g_xent_error, 1);
    return false;
}

__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(su32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(su32(bar))
        : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle (layout type 2), sm_100
// format (version 1).
//   K-major: rows of 64 K elements; 8-row groups 1024 bytes apart (stride
//     offset); a K step of 16 advances the address by 32 bytes.
//   MN-major: blocks of 64 M (or N) elements x BK rows of K; the blocks are
//     BK * 128 bytes apart (leading offset), 8-row groups along K 1024 bytes
//     apart (stride offset); a K step of 16 advances by two groups.
template <bool MN>
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(MN ? (BK * 128) >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <bool MN>
constexpr uint64_t kstep() { return MN ? 2048 >> 4 : 32 >> 4; }

// Instruction descriptor, kind::f16: D f32 (bits 4-5 = 1), A and B bf16
// (bits 7-9, 10-12 = 1), bits 15 / 16: A / B MN-major, N >> 3 at bit 17,
// M >> 4 at bit 24.
template <bool A_MN, bool B_MN>
constexpr uint32_t idesc() {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id,
                                          uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(id), "r"(acc));
}
__device__ __forceinline__ void umma_commit(uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     su32(b))
                 : "memory");
}

#define TC_BEFORE() asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory")
#define TC_AFTER() asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory")

// 32 consecutive accumulator columns of the warp's 32 lanes (one row per lane).
__device__ __forceinline__ void tmem_ld32(float (&v)[32], uint32_t addr) {
    uint32_t r[32];
    __syncwarp();  // the load is a warp's: lanes that parted in the caller meet
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int e = 0; e < 32; e++) v[e] = __uint_as_float(r[e]);
}

constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// v as the sum of three bf16 values.  A finite v that would round to infinity
// is truncated instead; an infinity keeps zero in the lower two.
__device__ __forceinline__ void split3(float v, bf16& b0, bf16& b1, bf16& b2) {
    b0 = __float2bfloat16_rn(v);
    if (__hisinf(b0) && isfinite(v)) b0 = __float2bfloat16_rz(v);
    const float r = __fsub_rn(v, __bfloat162float(b0));
    b1 = __float2bfloat16_rn(isinf(v) ? 0.0f : r);
    b2 = __float2bfloat16_rn(isinf(v) ? 0.0f : __fsub_rn(r, __bfloat162float(b1)));
}

__device__ __forceinline__ long long label_at(const void* labels, int bytes, size_t i) {
    return bytes == 8 ? ((const long long*)labels)[i] : (long long)((const int*)labels)[i];
}

// ---- the product kernel ---------------------------------------------------------

enum Epi : int { EPI_LSE = 0, EPI_G = 1, EPI_OUT = 2 };

struct GemmArgs {
    int M, N, K;       // D[M, N] = A[M, K] B[N, K]^T (either may be stored K-first)
    int nprod;         // 1, or 6 for operands in three planes
    long long col0;    // LSE, G: the class of column 0
    // LSE
    float* part_m;     // [column tile][M]
    float* part_s;
    float* zlabel;     // [M]
    // LSE, G
    const void* labels;
    int index_bytes;
    long long vocab;
    // G
    const float* lse;
    const float* dloss;
    bf16* g;           // planes of [M][ldg]
    long long ldg, gplane;
    int planes;
    // OUT
    float* acc;        // f32 [M][ldo]
    void* out;         // f32 or bf16 [M][ldo]
    int out_bf16;
    long long ldo;
    int mode;          // 0 out = D, 1 acc = D, 2 acc += D, 3 out = acc + D
};

__device__ __forceinline__ int prod_a(int p, int nprod) { return nprod == 1 ? 0 : (0x001102 >> (4 * p)) & 3; }
__device__ __forceinline__ int prod_b(int p, int nprod) { return nprod == 1 ? 0 : (0x010120 >> (4 * p)) & 3; }

// The row's maximum and sum of exponentials over the tile's columns.
__device__ __forceinline__ void epi_lse(const GemmArgs& g, uint32_t tm, int row, int n0, int nt) {
    float m = -INFINITY, s = 0.0f, zl = 0.0f;
    const int left = min(BN, g.N - n0);
    const bool live = row < g.M;
    const long long lab =
        live ? label_at(g.labels, g.index_bytes, row) - (g.col0 + n0) : -1;  // column of the tile
    for (int c0 = 0; c0 < left; c0 += 32) {
        float v[32];
        tmem_ld32(v, tm + c0);
        if (c0 + 32 > left) {
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (c0 + e >= left) v[e] = -INFINITY;
        }
        if (lab >= c0 && lab < c0 + 32) {
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (c0 + e == lab) zl = v[e];
        }
        float cm = v[0];
#pragma unroll
        for (int e = 1; e < 32; e++) cm = fmaxf(cm, v[e]);
        if (cm > m) {
            s *= ex2((m - cm) * kLog2e);  // m = -inf: s is 0
            m = cm;
        }
        // while every logit is -inf (or NaN), terms are taken against 0
        const float ref = m == -INFINITY ? 0.0f : m * kLog2e;
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 32; e++) t[e & 3] += ex2(fmaf(v[e], kLog2e, -ref));
        s += (t[0] + t[1]) + (t[2] + t[3]);
    }
    if (live) {
        g.part_m[(size_t)nt * g.M + row] = m;
        g.part_s[(size_t)nt * g.M + row] = s;
        if (lab >= 0 && lab < left) g.zlabel[row] = zl;
    }
}

__device__ __forceinline__ void epi_g(const GemmArgs& g, uint32_t tm, int row, int n0) {
    const int left = min(BN, g.N - n0);
    const bool live = row < g.M;
    float lse = 0.0f, dl = 0.0f;
    long long lab = -1;
    bool has = false;
    if (live) {
        const long long l = label_at(g.labels, g.index_bytes, row);
        has = l >= 0 && l < g.vocab;
        lab = has ? l - (g.col0 + n0) : -1;
        lse = g.lse[row];
        dl = g.dloss[row];
    }
    for (int c0 = 0; c0 < left; c0 += 32) {
        float v[32];
        tmem_ld32(v, tm + c0);
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 32; e++) {
            float p = ex2((v[e] - lse) * kLog2e);
            if (c0 + e == lab) p -= 1.0f;
            v[e] = has ? p * dl : 0.0f;
        }
        bf16* dst = g.g + (size_t)row * g.ldg + n0 + c0;
        if (g.planes == 1) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint4 o;
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    h[e] = __floats2bfloat162_rn(v[q * 8 + 2 * e], v[q * 8 + 2 * e + 1]);
                reinterpret_cast<uint4*>(dst)[q] = o;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint4 o[3];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    bf16 b[3];
                    split3(v[q * 8 + e], b[0], b[1], b[2]);
#pragma unroll
                    for (int k = 0; k < 3; k++) reinterpret_cast<bf16*>(&o[k])[e] = b[k];
                }
#pragma unroll
                for (int k = 0; k < 3; k++) reinterpret_cast<uint4*>(dst + k * g.gplane)[q] = o[k];
            }
        }
    }
}

__device__ __forceinline__ void epi_out(const GemmArgs& g, uint32_t tm, int row, int n0) {
    const int left = min(BN, g.N - n0);
    const bool live = row < g.M;
    const bool vec = (g.ldo & 7) == 0 &&
                     ((((uintptr_t)(g.mode == 0 || g.mode == 3 ? g.out : g.acc)) |
                       ((uintptr_t)(g.mode == 0 ? nullptr : g.acc))) & 15) == 0;
    for (int c0 = 0; c0 < left; c0 += 32) {
        float v[32];
        tmem_ld32(v, tm + c0);
        if (!live) continue;
        const size_t at = (size_t)row * g.ldo + n0 + c0;
        const bool whole = vec && c0 + 32 <= left;
        if (g.mode >= 2) {
            if (whole) {
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float4 a = reinterpret_cast<const float4*>(g.acc + at)[q];
                    v[4 * q] += a.x, v[4 * q + 1] += a.y, v[4 * q + 2] += a.z, v[4 * q + 3] += a.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c0 + e < left) v[e] += g.acc[at + e];
            }
        }
        const bool to_acc = g.mode == 1 || g.mode == 2;
        if (to_acc || !g.out_bf16) {
            float* o = to_acc ? g.acc + at : (float*)g.out + at;
            if (whole) {
#pragma unroll
                for (int q = 0; q < 8; q++)
                    reinterpret_cast<float4*>(o)[q] =
                        make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c0 + e < left) o[e] = v[e];
            }
        } else {
            bf16* o = (bf16*)g.out + at;
            if (whole) {
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint4 u;
                    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        h[e] = __floats2bfloat162_rn(v[q * 8 + 2 * e], v[q * 8 + 2 * e + 1]);
                    reinterpret_cast<uint4*>(o)[q] = u;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c0 + e < left) o[e] = __float2bfloat16_rn(v[e]);
            }
        }
    }
}

// Persistent: CTA b computes tiles b, b + gridDim.x, ... (row tile fastest, so
// that the CTAs at work share the column operand's tiles in L2).
//   warp 0 lane 0: TMA producer, ST stages of A (128 x 64) and B (256 x 64);
//   warp 1 lane 0: MMA issuer into one of two accumulators in tensor memory;
//   warps 4-7: epilogue of the other accumulator (warp q reads lanes 32 q ..).
// Every wait is bounded; on a timeout each role stops, outstanding loads and
// products are waited for (bounded), tensor memory is freed and g_xent_error set.
template <int EPI, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(256, 1)
k_xgemm(const __grid_constant__ CUtensorMap mA, const __grid_constant__ CUtensorMap mB,
        const GemmArgs g) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (su32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * ST_BYTES);
    uint64_t* empty = full + ST;
    uint64_t* acc_full = empty + ST;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    __shared__ volatile int s_err;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int KB = (g.K + BK - 1) / BK, KT = KB * g.nprod;
    const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
    const long long tiles = (long long)tm * tn;

    if (tid == 0) {
        s_err = 0;
        for (int s = 0; s < ST; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 128);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         su32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    TC_BEFORE();
    __syncthreads();
    TC_AFTER();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        int it = 0;
        bool ok = true;
        for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            const int m0 = (int)(t % tm) * BM, n0 = (int)(t / tm) * BN;
            for (int v = 0; v < KT; v++, it++) {
                const int s = it % ST;
                if (it >= ST && !mbar_wait(&empty[s], ((it / ST) + 1) & 1, &s_err)) {
                    ok = false;
                    break;
                }
                const int p = v / KB, k0 = (v - p * KB) * BK;
                const int za = prod_a(p, g.nprod), zb = prod_b(p, g.nprod);
                unsigned char* a = smem + s * ST_BYTES;
                unsigned char* b = a + A_BYTES;
                mbar_expect_tx(&full[s], ST_BYTES);
                if constexpr (A_MN) {
#pragma unroll
                    for (int j = 0; j < BM / 64; j++)
                        tma_load(a + j * (BK * 128), &mA, m0 + j * 64, k0, za, &full[s]);
                } else {
                    tma_load(a, &mA, k0, m0, za, &full[s]);
                }
                if constexpr (B_MN) {
#pragma unroll
                    for (int j = 0; j < BN / 64; j++)
                        tma_load(b + j * (BK * 128), &mB, n0 + j * 64, k0, zb, &full[s]);
                } else {
                    tma_load(b, &mB, k0, n0, zb, &full[s]);
                }
            }
        }
        // every load lands before the CTA's shared memory goes away (at once,
        // unless a role has given up)
        for (int i = it > ST ? it - ST : 0; i < it; i++)
            for (uint32_t w = 0; w < (1u << 22) && !mbar_try(&full[i % ST], (i / ST) & 1); w++)
                __nanosleep(100);
    } else if (warp == 1 && lane == 0) {
        int it = 0, i = 0;
        bool ok = true;
        for (long long t = blockIdx.x; t < tiles && ok; t += gridDim.x, i++) {
            const int buf = i & 1;
            if (i >= 2 && !mbar_wait(&acc_empty[buf], ((i >> 1) + 1) & 1, &s_err)) {
                ok = false;
                break;
            }
            TC_AFTER();
            const uint32_t d = tmem + buf * BN;
            for (int v = 0; v < KT; v++, it++) {
                const int s = it % ST;
                if (!mbar_wait(&full[s], (it / ST) & 1, &s_err)) {
                    ok = false;
                    break;
                }
                TC_AFTER();
                const uint32_t a = su32(smem + s * ST_BYTES);
                const uint64_t da = sdesc<A_MN>(a), db = sdesc<B_MN>(a + A_BYTES);
#pragma unroll
                for (int k = 0; k < BK / 16; k++)
                    umma_bf16(d, da + k * kstep<A_MN>(), db + k * kstep<B_MN>(),
                              idesc<A_MN, B_MN>(), (v | k) ? 1u : 0u);
                umma_commit(&empty[s]);
            }
            if (ok) umma_commit(&acc_full[buf]);
        }
        if (!ok) {  // products in flight end before tensor memory is freed
            umma_commit(drain);
            for (uint32_t w = 0; w < (1u << 22) && !mbar_try(drain, 0); w++) __nanosleep(100);
        }
    } else if (warp >= 4) {
        const int q = warp - 4;
        int i = 0;
        for (long long t = blockIdx.x; t < tiles; t += gridDim.x, i++) {
            const int m0 = (int)(t % tm) * BM, nt = (int)(t / tm), n0 = nt * BN;
            const int buf = i & 1;
            const bool ok = mbar_wait(&acc_full[buf], (i >> 1) & 1, &s_err);
            if (!__all_sync(0xffffffffu, ok)) break;
            TC_AFTER();
            const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
            const int row = m0 + q * 32 + lane;
            if constexpr (EPI == EPI_LSE) epi_lse(g, src, row, n0, nt);
            else if constexpr (EPI == EPI_G) epi_g(g, src, row, n0);
            else epi_out(g, src, row, n0);
            TC_BEFORE();
            mbar_arrive(&acc_empty[buf]);
        }
    }
    __syncwarp();
    TC_BEFORE();
    __syncthreads();
    if (warp == 2) {
        TC_AFTER();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(TMEM_COLS)
                     : "memory");
    }
}

// ---- small kernels -----------------------------------------------------------------

// Rows of src [rows][dim] as bf16 planes [planes][rows][ld] (1 plane: copied,
// 3: split3); with labels, a row without a target becomes zeros, so that what
// its x holds (NaN, infinities) never meets the zeros of its G row.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
k_pack(bf16* __restrict__ dst, const T* __restrict__ src, long long rows, int dim, int ld,
       const void* labels, int index_bytes, long long vocab) {
    const long long total = rows * ld, plane = rows * ld;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / ld;
        const int c = (int)(i - r * ld);
        bool live = c < dim;
        if (labels) {
            const long long l = label_at(labels, index_bytes, r);
            live = live && l >= 0 && l < vocab;
        }
        if constexpr (PLANES == 1) {
            dst[i] = live ? (bf16)src[r * dim + c] : __float2bfloat16_rn(0.0f);
        } else {
            bf16 b0, b1, b2;
            split3(live ? (float)src[r * dim + c] : 0.0f, b0, b1, b2);
            dst[i] = b0;
            dst[plane + i] = b1;
            dst[2 * plane + i] = b2;
        }
    }
}

// lse and loss of every row from its tiles' maxima and sums: 8 strided
// groups of tiles per row joined in a fixed order.
__global__ void __launch_bounds__(256)
k_xent_join(float* __restrict__ loss, float* __restrict__ lse, const float* __restrict__ part_m,
            const float* __restrict__ part_s, const float* __restrict__ zlabel,
            const void* labels, int index_bytes, long long vocab, long long n, int tiles) {
    __shared__ float sm[8][33], ss[8][33];
    const long long row = (long long)blockIdx.x * 32 + threadIdx.x;
    float m = -INFINITY, s = 0.0f;
    auto join = [&](float om, float os) {
        if (om > m) {
            s = s * expf(m - om) + os;
            m = om;
        } else {
            s += om == -INFINITY ? os : os * expf(om - m);
        }
    };
    if (row < n)
        for (int t = threadIdx.y; t < tiles; t += 8)
            join(part_m[(size_t)t * n + row], part_s[(size_t)t * n + row]);
    sm[threadIdx.y][threadIdx.x] = m;
    ss[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && row < n) {
        for (int k = 1; k < 8; k++) join(sm[k][threadIdx.x], ss[k][threadIdx.x]);
        // no finite maximum (a row of -inf or NaN): log 0 would say -inf
        const float ls = logf(s);
        lse[row] = m == -INFINITY ? NAN : m + ls;
        const long long l = label_at(labels, index_bytes, row);
        // (m - z_label) + log s keeps small losses exact where lse - z_label cancels
        loss[row] = l >= 0 && l < vocab ? (m == -INFINITY ? NAN : (m - zlabel[row]) + ls) : 0.0f;
    }
}

// ---- host ---------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = []() {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        cudaGetLastError();
        return (PFN_cuTensorMapEncodeTiled_v12000) nullptr;
    }();
    return fn;
}

// bf16 planes [planes][rows][ld] of which `cols` columns count; boxes of 64
// columns x box_rows rows, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, const void* base, size_t cols, size_t rows, size_t ld, int planes,
             size_t plane, int box_rows) {
    auto fn = encode_fn();
    if (!fn) {
        set_error("cuTensorMapEncodeTiled unavailable");
        return E_CUDA;
    }
    cuuint64_t dims[3] = {cols, rows, (cuuint64_t)planes};
    cuuint64_t strides[2] = {ld * 2, plane * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides,
                    box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
        return E_CUDA;
    }
    return OK;
}

template <int EPI, bool A_MN, bool B_MN>
int run_gemm(Ctx& c, const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& g) {
    NXV_CK(cudaFuncSetAttribute(k_xgemm<EPI, A_MN, B_MN>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    const long long tiles = (long long)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    const unsigned grid = (unsigned)std::min<long long>(tiles, c.dev->sm_count);
    k_xgemm<EPI, A_MN, B_MN><<<grid, 256, SMEM, c.stream>>>(a, b, g);
    count_launch();
    return OK;
}

size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// How a call uses its workspace.  The vocabulary is cut into pieces of vp
// classes (a multiple of the column tile) so that the piece's G, and its
// packed w where w cannot be read in place, stay within a fixed budget.
struct Plan {
    int planes;
    size_t dp;               // packed row length
    size_t vp, pieces;
    size_t xp, wp, g, ldg, acc, pm, ps, zl, total;  // byte offsets; ldg in elements
};

constexpr size_t kPieceBytes = (size_t)256 << 20;

Plan make_plan(const XentP& p, bool grad) {
    Plan q{};
    q.planes = p.dt == F32 ? 3 : 1;
    q.dp = up(p.dim, 8);
    const size_t per_class = (size_t)q.planes * 2 * (q.dp + (grad ? (size_t)p.n : 0));
    size_t vp = std::max<size_t>(kPieceBytes / per_class / BN * BN, 4 * BN);
    const size_t all = up(p.vocab, BN);
    vp = std::min(vp, all);
    q.pieces = (p.vocab + vp - 1) / vp;
    q.vp = up((p.vocab + q.pieces - 1) / q.pieces, BN);
    q.pieces = (p.vocab + q.vp - 1) / q.vp;
    q.ldg = q.vp;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up(bytes, 1024);
        return o;
    };
    q.xp = take((size_t)q.planes * 2 * p.n * q.dp);
    q.wp = take((size_t)q.planes * 2 * q.vp * q.dp);
    if (grad) {
        q.g = take((size_t)q.planes * 2 * p.n * q.ldg);
        q.acc = take(p.dt == BF16 ? (size_t)4 * p.n * p.dim : 0);
    } else {
        const size_t tiles = all / BN;
        q.pm = take(4 * tiles * p.n);
        q.ps = take(4 * tiles * p.n);
        q.zl = take((size_t)4 * p.n);
    }
    q.total = at;
    return q;
}

void pack(Ctx& c, const XentP& p, bf16* dst, const void* src, size_t rows, int ld, bool masked) {
    const unsigned grid = grid_for(c, rows * ld, 256, 16);
    const void* lab = masked ? p.labels : nullptr;
    if (p.dt == F32)
        k_pack<float, 3><<<grid, 256, 0, c.stream>>>(dst, (const float*)src, rows, p.dim, ld, lab,
                                                     p.index_bytes, p.vocab);
    else
        k_pack<bf16, 1><<<grid, 256, 0, c.stream>>>(dst, (const bf16*)src, rows, p.dim, ld, lab,
                                                    p.index_bytes, p.vocab);
    count_launch();
}

// w can feed TMA where it lies when its rows start on 16-byte boundaries.
bool in_place(const XentP& p, const void* t) {
    return p.dt == BF16 && p.dim % 8 == 0 && ((uintptr_t)t & 15) == 0;
}

}  // namespace

size_t xent_workspace(const XentP& p, bool grad) { return make_plan(p, grad).total; }

int xent_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_xent_error, sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (v) {
        int z = 0;
        cudaMemcpyToSymbol(g_xent_error, &z, sizeof(int));
    }
    return v;
}

int launch_xent(Ctx& c, const XentP& p, void* loss, void* lse, void* ws) {
    if (p.n == 0) return OK;
    const Plan q = make_plan(p, false);
    char* base = (char*)ws;
    const bool wip = in_place(p, p.w), xip = in_place(p, p.x);
    const bf16* xp = (const bf16*)p.x;
    if (!xip) {
        xp = (bf16*)(base + q.xp);
        pack(c, p, (bf16*)xp, p.x, p.n, (int)q.dp, false);
    }
    CUtensorMap ma, mb;
    int rc;
    if ((rc = make_map(&ma, xp, p.dim, p.n, q.dp, q.planes, (size_t)p.n * q.dp, BM))) return rc;
    GemmArgs g{};
    g.M = (int)p.n;
    g.K = (int)p.dim;
    g.nprod = q.planes == 3 ? 6 : 1;
    g.zlabel = (float*)(base + q.zl);
    g.labels = p.labels;
    g.index_bytes = p.index_bytes;
    g.vocab = p.vocab;
    const size_t vp = wip ? (size_t)p.vocab : q.vp;
    for (size_t v0 = 0; v0 < p.vocab; v0 += vp) {
        const size_t nv = std::min<size_t>(vp, p.vocab - v0);
        const bf16* wp = (const bf16*)p.w;
        if (!wip) {
            wp = (bf16*)(base + q.wp);
            pack(c, p, (bf16*)wp, (const char*)p.w + v0 * p.dim * dtype_bytes(p.dt), nv, (int)q.dp,
                 false);
        }
        if ((rc = make_map(&mb, wp, p.dim, nv, q.dp, q.planes, nv * q.dp, BN))) return rc;
        g.N = (int)nv;
        g.col0 = (long long)v0;
        g.part_m = (float*)(base + q.pm) + v0 / BN * p.n;
        g.part_s = (float*)(base + q.ps) + v0 / BN * p.n;
        if ((rc = run_gemm<EPI_LSE, false, false>(c, ma, mb, g))) return rc;
    }
    k_xent_join<<<(p.n + 31) / 32, dim3(32, 8), 0, c.stream>>>(
        (float*)loss, (float*)lse, (const float*)(base + q.pm), (const float*)(base + q.ps),
        (const float*)(base + q.zl), p.labels, p.index_bytes, p.vocab, p.n,
        (int)((p.vocab + BN - 1) / BN));
    count_launch();
    pdl_record_all(c);
    return finish(c);
}

int launch_xent_grad(Ctx& c, const XentP& p, void* dx, void* dw, const void* dloss,
                     const void* lse, void* ws) {
    if (p.n == 0) {
        NXV_CK(cudaMemsetAsync(dw, 0, (size_t)p.vocab * p.dim * dtype_bytes(p.dt), c.stream));
        return finish(c);
    }
    const Plan q = make_plan(p, true);
    char* base = (char*)ws;
    const bool wip = in_place(p, p.w);
    bf16* xp = (bf16*)(base + q.xp);
    bf16* gp = (bf16*)(base + q.g);
    pack(c, p, xp, p.x, p.n, (int)q.dp, true);
    const size_t xplane = (size_t)p.n * q.dp, gplane = (size_t)p.n * q.ldg;
    CUtensorMap mxk, mxn, mwk, mwn, mgk, mgm;
    int rc;
    // x: K-major A of z = x w^T, and N-major B of dw = G^T x
    if ((rc = make_map(&mxk, xp, p.dim, p.n, q.dp, q.planes, xplane, BM))) return rc;
    if ((rc = make_map(&mxn, xp, p.dim, p.n, q.dp, q.planes, xplane, BK))) return rc;
    GemmArgs z{};
    z.M = (int)p.n;
    z.K = (int)p.dim;
    z.nprod = q.planes == 3 ? 6 : 1;
    z.labels = p.labels;
    z.index_bytes = p.index_bytes;
    z.vocab = p.vocab;
    z.lse = (const float*)lse;
    z.dloss = (const float*)dloss;
    z.g = gp;
    z.ldg = (long long)q.ldg;
    z.gplane = (long long)gplane;
    z.planes = q.planes;
    for (size_t v0 = 0, i = 0; v0 < p.vocab; v0 += q.vp, i++) {
        const size_t nv = std::min<size_t>(q.vp, p.vocab - v0);
        const bf16* wp = (const bf16*)p.w + (wip ? v0 * p.dim : 0);
        if (!wip) {
            wp = (bf16*)(base + q.wp);
            pack(c, p, (bf16*)wp, (const char*)p.w + v0 * p.dim * dtype_bytes(p.dt), nv, (int)q.dp,
                 false);
        }
        if ((rc = make_map(&mwk, wp, p.dim, nv, q.dp, q.planes, nv * q.dp, BN))) return rc;
        if ((rc = make_map(&mwn, wp, p.dim, nv, q.dp, q.planes, nv * q.dp, BK))) return rc;
        if ((rc = make_map(&mgk, gp, nv, p.n, q.ldg, q.planes, gplane, BM))) return rc;
        if ((rc = make_map(&mgm, gp, nv, p.n, q.ldg, q.planes, gplane, BK))) return rc;
        z.N = (int)nv;
        z.col0 = (long long)v0;
        if ((rc = run_gemm<EPI_G, false, false>(c, mxk, mwk, z))) return rc;
        GemmArgs o{};
        o.nprod = z.nprod;
        o.out_bf16 = p.dt == BF16;
        o.ldo = p.dim;
        // dx += G w: K runs over the piece's classes
        o.M = (int)p.n;
        o.N = (int)p.dim;
        o.K = (int)nv;
        const bool first = i == 0, last = v0 + nv == p.vocab;
        o.out = dx;
        o.acc = p.dt == BF16 ? (float*)(base + q.acc) : (float*)dx;
        o.mode = p.dt == F32 ? (first ? 1 : 2) : first ? (last ? 0 : 1) : (last ? 3 : 2);
        if ((rc = run_gemm<EPI_OUT, false, true>(c, mgk, mwn, o))) return rc;
        // dw = G^T x: K runs over the tokens
        o.M = (int)nv;
        o.K = (int)p.n;
        o.out = (char*)dw + v0 * p.dim * dtype_bytes(p.dt);
        o.acc = nullptr;
        o.mode = 0;
        if ((rc = run_gemm<EPI_OUT, true, true>(c, mgm, mxn, o))) return rc;
    }
    pdl_record_all(c);
    return finish(c);
}

}  // namespace nxv
