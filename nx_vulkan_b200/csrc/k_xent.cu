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
// tcgen05 tensor cores (few rows and small problems have kernels of their own, further
// down).  All go through one kernel, k_xgemm, with an epilogue each:
//   LSE   the maximum and the sum of exponentials of every row over a segment
//         of classes (8 bytes per row and segment instead of the logits) and
//         the label's logit; a small kernel joins the segments;
//   GRAD  P = exp(z - lse) - [v = label] for one piece of the vocabulary at a
//         time, as bf16;
//   OUT   dx = dloss (sum over pieces of P w), the sum in f32, and
//         dw_piece = P^T (dloss x).
//
// Types.  bf16: the operands go to the tensor core as they are; sums are f32, all of K
// in the tensor core's accumulator, which may lose up to 2^-23 of the running sum per 16
// products, towards zero (8192 x 65536 x 2048: the loss is 6.7e-7 from its formula in 64
// bits, in f32 sums that round to nearest 7e-8).
// Two roundings to bf16 stand between the inputs and the sums of the gradient
// (2^-8 relative to each term at most, like the rounding of the inputs): P
// without the factor dloss, so that the label's entry, near -1, is nearly exact
// (with it, all rows of a mean loss would round the same value, by up to 2^-8),
// and dloss x, in units of the largest dloss, which leaves x as it is for a mean.
// Against 64 bits, P's rounding adds 2.7e-4 to dx and dw (2-norms), beside the 1.65e-3
// of their own rounding to bf16.  Few rows and small problems keep both in f32.
// f32: every f32 value is the sum of three bf16 values, b0 = bf16(v),
// b1 = bf16(v - b0), b2 = bf16(v - b0 - b1) (exact but for values below 2^-110),
// and a product is the six partial products b_i b_j with i + j <= 2; the three
// left out are below 2^-24 of the product.  bf16 has f32's exponent range, so
// no scaling is needed, and six bf16 products cost what three TF32 products cost.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include "kernels.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace nxv {

namespace {

using bf16 = __nv_bfloat16;

// A CTA stages 128 rows of A and 128 of B, 64 of K deep.  Alone (CG = 1) it
// makes a 128 x 128 tile; a pair of CTAs (CG = 2, tcgen05 cta_group::2) makes a
// 256 x 256 tile, each holding the accumulator of its own 128 rows.
constexpr int BT = 128, BK = 64;  // BK bf16 = one 128-byte swizzle row
constexpr int ST = 6;
constexpr int OP_BYTES = BT * BK * 2, ST_BYTES = 2 * OP_BYTES;
constexpr int TR_BYTES = 8 * 32 * 33 * 4;  // a 32 x 32 transpose buffer per epilogue warp
constexpr int SMEM = ST * ST_BYTES + 1024 + 256 + TR_BYTES;
static_assert(SMEM <= 227 * 1024, "shared memory of a CTA");
constexpr int kThreads = 384;  // producer of A, MMA issuer, allocator, producer of B, 8 epilogue warps

// ---- PTX ----------------------------------------------------------------------

__device__ __forceinline__ uint32_t su32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes)
                 : "memory");
}
// The address of the same shared-memory object in the pair's CTA 0.
__device__ __forceinline__ uint32_t in_leader(uint32_t p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(p));
    return r;
}
__device__ __forceinline__ void mbar_arrive_leader(uint32_t b) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(b), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait (seconds at most); false when it runs out or when another
// warp of the CTA has given up.
__device__ __noinline__ bool mbar_wait_long(uint32_t b, uint32_t parity, volatile int* err) {
    for (uint32_t i = 0; i < (1u << 22); i++) {
        if (mbar_try(b, parity)) return true;
        if (i > 256) {
            if (*err) return false;
            __nanosleep(100);
        }
    }
    *err = 1;
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t b, uint32_t parity, volatile int* err) {
    return mbar_try(b, parity) || mbar_wait_long(b, parity, err);
}

// Into this CTA's shared memory; the bytes count on the leader's barrier.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            ".cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
            "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle (layout type 2), sm_100
// format (version 1).
//   K-major: rows of 64 K elements; 8-row groups 1024 bytes apart (stride
//     offset); a K step of 16 advances the address by 32 bytes.
//   MN-major: blocks of 64 M (or N) elements x BK rows of K; the blocks are
//     BK * 128 bytes apart (leading offset), 8-row groups along K 1024 bytes
//     apart (stride offset); a K step of 16 advances by two groups.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, bool mn) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(mn ? (BK * 128) >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ uint64_t kstep(bool mn) { return mn ? 2048 >> 4 : 32 >> 4; }

// Instruction descriptor, kind::f16: D f32 (bits 4-5 = 1), A and B bf16
// (bits 7-9, 10-12 = 1), bits 15 / 16: A / B MN-major, N >> 3 at bit 17,
// M >> 4 at bit 24.
template <int CG>
__device__ __forceinline__ uint32_t idesc(bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(BT * CG >> 3) << 17) | ((uint32_t)(BT * CG >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t id,
                                          uint32_t acc) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(acc));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(id), "r"(acc));
}
// Arrives on the barrier (of both CTAs of a pair) when every product issued
// so far has completed.
template <int CG>
__device__ __forceinline__ void umma_commit(uint32_t b) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
            "[%0], %1;" ::"r"(b),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(b)
                     : "memory");
}
// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
// A whole warp's wait: the same answer in every lane, so that the loops around
// it stay uniform and their addresses in uniform registers.
__device__ __forceinline__ bool warp_wait(uint32_t b, uint32_t parity, volatile int* err) {
    return __all_sync(0xffffffffu, mbar_wait(b, parity, err));
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
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

enum Kind : int { LSE = 0, GRAD = 1, OUT = 2 };

struct Job {
    int kind;
    int M, N, K;          // D[M, N] = A[M, K] B[N, K]^T
    int a_mn, b_mn;       // the operand is stored K rows of M (N) values
    uint32_t tm, tiles;   // row tiles, all tiles
    uint32_t plane;       // tiles of one slice of K
    int kslice;           // the K of a slice, a multiple of BK
    long long col0;       // LSE, GRAD: the class of column 0
    // LSE
    float* part_m;        // [column segment of 64 CG classes][M]
    float* part_s;
    float* zlabel;        // [M]
    // LSE, GRAD
    const void* labels;
    int index_bytes;
    long long vocab;
    // GRAD
    const float* lse;
    bf16* g;              // planes of [M][ldg]
    long long ldg, gplane;
    // OUT: with slices, out and acc_in are f32 [slice][M][ldo]
    const float* acc_in;  // f32 [M][ldo] to add, or null
    const float* dloss;   // [M]: the rows' factors, 0 for a row without a target; or null
    const float* factor;  // one factor of all, or null
    void* out;            // [M][ldo]
    int out_bf16;
    long long ldo;
};

// K blocks of tile lt of the job.
__device__ __forceinline__ int k_blocks(const Job& g, uint32_t lt) {
    const int first = (int)(lt / g.plane) * g.kslice;
    return (min(g.K - first, g.kslice) + BK - 1) / BK;
}

constexpr int kMaxJobs = 3;
struct alignas(64) Work {
    CUtensorMap map[2 * kMaxJobs];  // A, B of every job
    Job job[kMaxJobs];
    int jobs;
    uint32_t tiles;
    int* err;             // wait_flag(c)
};

// The six partial products of f32, the smallest first.
__device__ __forceinline__ int prod_a(int p) { return (0x001102 >> (4 * p)) & 3; }
__device__ __forceinline__ int prod_b(int p) { return (0x010120 >> (4 * p)) & 3; }

// 16 bytes x 2 of a row, with the widest store its address allows.
__device__ __forceinline__ void store32(void* p, const uint32_t (&u)[8], int align) {
    if (align >= 32) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]),
                     "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

// One thread's row of a tile: 32 columns at a time go through chunk().
// n0: the columns' first column of D; left: columns of D from there.
// SIX: no transpose buffer (its code costs registers that hold the sums).
template <bool SIX>
struct Row {
    const Job& g;
    const int row, n0, left;
    const bool live;
    // LSE
    float m = -INFINITY, s = 0.0f, zl = 0.0f;
    long long lab = -1;  // the label's column, from n0
    // GRAD
    float lse = 0.0f;
    // OUT
    size_t row_at = 0;  // the row's first element in out and acc_in
    float dl = 0.0f;
    int align = 0;
    bool has = false;

    float* const tr;  // the warp's transpose buffer

    __device__ __forceinline__ Row(const Job& j, int r, int n, uint32_t slice, float* t)
        : g(j), row(r), n0(n), left(j.N - n), live(r < j.M), tr(t) {
        row_at = ((size_t)slice * g.M + row) * g.ldo;
        if (g.kind == OUT) {
            const int es = g.out_bf16 ? 2 : 4;
            const uintptr_t a = (uintptr_t)g.out | (uintptr_t)(g.ldo * es) | (uintptr_t)g.acc_in |
                                (uintptr_t)(g.acc_in ? g.ldo * 4 : 0);
            align = (a & 31) == 0 ? 32 : (a & 15) == 0 ? 16 : 4;
        }
        if (live && (g.kind != OUT || g.dloss)) {
            const long long l = label_at(g.labels, g.index_bytes, row);
            has = l >= 0 && l < g.vocab;
            lab = has ? l - (g.col0 + n0) : -1;
            if (g.kind == GRAD) lse = g.lse[row];
            if (g.kind == OUT) dl = g.dloss[row];
        }
    }

    __device__ __forceinline__ void chunk(float (&v)[32], int c0) {
        if (c0 >= left) return;
        if (g.kind == LSE) chunk_lse(v, c0);
        else if (g.kind == GRAD) chunk_grad(v, c0);
        else chunk_out(v, c0);
    }

    __device__ __forceinline__ void chunk_lse(float (&v)[32], int c0) {
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
        // While every logit is -inf (or NaN), terms are taken against 0.  The difference first:
        // the largest term is 1 then and the sum not below it, so no loss is negative (one
        // fma with m log2e, rounded, puts all terms off by half a step of that product).
        const float ref = m == -INFINITY ? 0.0f : m;
        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 32; e++) t[e & 3] += ex2((v[e] - ref) * kLog2e);
        s += (t[0] + t[1]) + (t[2] + t[3]);
    }

    __device__ __forceinline__ void chunk_grad(float (&v)[32], int c0) {
        if (!live) return;
#pragma unroll
        for (int e = 0; e < 32; e++) {
            float p = ex2((v[e] - lse) * kLog2e);
            if (c0 + e == lab) p -= 1.0f;
            v[e] = has ? p : 0.0f;
        }
        // ldg covers whole tiles, so the columns past N have room; no product reads them
        bf16* dst = g.g + (size_t)row * g.ldg + n0 + c0;
        if constexpr (!SIX) {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t u[8];
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = pack2(v[q * 16 + 2 * e], v[q * 16 + 2 * e + 1]);
                store32(dst + q * 16, u, 32);
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t u[3][8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    bf16 a[3], b[3];
                    split3(v[q * 16 + 2 * e], a[0], a[1], a[2]);
                    split3(v[q * 16 + 2 * e + 1], b[0], b[1], b[2]);
#pragma unroll
                    for (int k = 0; k < 3; k++) {
                        __nv_bfloat162 h = __halves2bfloat162(a[k], b[k]);
                        u[k][e] = *reinterpret_cast<uint32_t*>(&h);
                    }
                }
#pragma unroll
                for (int k = 0; k < 3; k++) store32(dst + k * g.gplane + q * 16, u[k], 32);
            }
        }
    }

    // Whole aligned rows of 32 columns: a lane stores its own row, 32 bytes at a
    // time.  Else through the warp's transpose buffer: a row's columns are the
    // lanes', so that what cannot be a wide store is at least a whole line.
    __device__ __forceinline__ void chunk_out(float (&v)[32], int c0) {
        if (align >= 16 && c0 + 32 <= left) out_rows(v, c0);
        else if constexpr (SIX) out_single(v, c0);
        else out_columns(v, c0);
    }

    __device__ __forceinline__ void out_single(float (&v)[32], int c0) {
        if (!live) return;
        finish(v, c0, false);
        float* o = (float*)g.out + row_at + n0 + c0;
#pragma unroll
        for (int e = 0; e < 32; e++)
            if (c0 + e < left) o[e] = v[e];
    }

    // The sum so far and the factors.
    __device__ __forceinline__ void finish(float (&v)[32], int c0, bool wide) {
        if (g.acc_in) {
            const float* in = g.acc_in + row_at + n0 + c0;
            if (wide) {
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float4 a = reinterpret_cast<const float4*>(in)[q];
                    v[4 * q] += a.x, v[4 * q + 1] += a.y, v[4 * q + 2] += a.z, v[4 * q + 3] += a.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (c0 + e < left) v[e] += in[e];
            }
        }
        if (g.dloss) {
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] = has ? v[e] * dl : 0.0f;
        }
        if (g.factor) {
            const float f = *g.factor;
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] *= f;
        }
    }

    __device__ __forceinline__ void out_columns(float (&v)[32], int c0) {
        const int lane = threadIdx.x & 31, r0 = row - lane;
        __syncwarp();  // the buffer's last chunk has been read
#pragma unroll
        for (int e = 0; e < 32; e++) tr[lane * 33 + e] = v[e];
        __syncwarp();
        const size_t at0 = row_at - (size_t)lane * g.ldo + n0 + c0 + lane;
        const float f = g.factor ? *g.factor : 1.0f;
        const bool in = c0 + lane < left;
#pragma unroll 4
        for (int r = 0; r < 32; r++) {
            const float rdl = __shfl_sync(0xffffffffu, dl, r);
            const bool rhas = __shfl_sync(0xffffffffu, has, r);
            if (!in || r0 + r >= g.M) continue;
            const size_t at = at0 + (size_t)r * g.ldo;
            float x = tr[r * 33 + lane];
            if (g.acc_in) x += g.acc_in[at];
            if (g.dloss) x = rhas ? x * rdl : 0.0f;
            x *= f;
            if (g.out_bf16) ((bf16*)g.out)[at] = __float2bfloat16_rn(x);
            else ((float*)g.out)[at] = x;
        }
    }

    __device__ __forceinline__ void out_rows(float (&v)[32], int c0) {
        if (!live) return;
        const size_t at = row_at + n0 + c0;
        finish(v, c0, true);
        if (!SIX && g.out_bf16) {
            bf16* o = (bf16*)g.out + at;
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t u[8];
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = pack2(v[q * 16 + 2 * e], v[q * 16 + 2 * e + 1]);
                store32(o + q * 16, u, align);
            }
        } else {
            float* o = (float*)g.out + at;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint32_t u[8];
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] = __float_as_uint(v[q * 8 + e]);
                store32(o + q * 8, u, align);
            }
        }
    }

    // width: the columns of the segment
    __device__ __forceinline__ void done(int width) {
        if (g.kind != LSE || !live || left <= 0) return;
        const size_t at = (size_t)(n0 / width) * g.M + row;
        g.part_m[at] = m;
        g.part_s[at] = s;
        if (lab >= 0 && lab < min(width, left)) g.zlabel[row] = zl;
    }
};

__device__ __forceinline__ uint32_t tile_of(uint32_t round, uint32_t first, uint32_t step) {
    return round * step + (round & 1 ? step - 1 - first : first);
}

// Persistent: the CTAs (pairs) take the tiles of the jobs in rounds (row tile fastest,
// so that the CTAs at work share the column operand's tiles in L2).  Jobs of one
// launch do not depend on each other; the host puts the one with the longest K first,
// and every other round goes backwards, so that the last round's tiles go to those
// whose first tile was short (2048 x 10007 x 1000 f32 gradient 612 us instead of 666).
//   warps 0 and 3, lane 0: TMA producers, ST stages of 128 rows of A and of B;
//   warp 1 lane 0 (of the leader): MMA issuer into one of two accumulators;
//   warps 4-11: epilogue of the other (warp w: lanes 32 (w % 4), column half (w - 4) / 4).
// SIX (f32): the six partial products, one k-block of all of them at a time:
// the tensor core's sums lose up to a step of the running sum per product,
// with a bias, so every k-block's sum is added to f32 registers by the
// epilogue warps (round to nearest) while the next one is made.  Measured for
// 2048 x 10007 x 1000: error of the gradients 1.9e-5 without, 2.6e-7 with.
// Bound by the tensor pipe, at the clock that its power leaves.  What it took: pair
// tiles (a stage's 32 KB for 512 cycles of products), and issue loops without
// divisions, one warp per operand and uniform (a stage took its one thread
// ~1000 cycles to load before, whatever its size or the ring's depth, and ~500 to
// multiply).  Measured, 8192 x 65536 x 2048 bf16: loss 1.30 ms in short runs (1.69
// PFLOP/s), 1.44 to 1.51 in a loop (1.5; the library's bare product of these sizes 1.47);
// gradient 4.8 ms at first, 5.5 to 5.6 in a loop, 1.6 PFLOP/s over its four products;
// 8192 x 32768 x 1024 f32 2.2 and 8.1 ms (2.35 and 8.2 in a loop), 1.6 PFLOP/s over the six partial products.
// Every wait is bounded; on a timeout each role stops, loads and products in
// flight are waited for (bounded), tensor memory is freed and the host's flag set.
template <int CG, bool SIX>
__global__ void __launch_bounds__(kThreads, 1)
k_xgemm(const __grid_constant__ Work W) {
    constexpr int NC = BT * CG;       // accumulator columns
    constexpr int HALF = NC / 2;      // columns of one epilogue warp
    constexpr uint32_t COLS = 2 * NC; // tensor memory columns
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (su32(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * ST_BYTES);
    uint64_t* empty = full + ST;
    uint64_t* acc_full = empty + ST;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drain = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int& s_err = *reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int rank = CG == 2 ? (blockIdx.x & 1) : 0;
    const uint32_t first = blockIdx.x / CG, step = gridDim.x / CG;

    if (tid == 0) {
        s_err = 0;
        for (int s = 0; s < ST; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 8 * CG);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             su32(tmem_slot)),
                         "r"(COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             su32(tmem_slot)),
                         "r"(COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    TC_BEFORE();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();  // the peer's barriers are ready
    TC_AFTER();
    const uint32_t tmem = *tmem_slot;

    // shared-memory addresses of the barriers (8 bytes each)
    const uint32_t b_full = su32(full), b_empty = su32(empty), b_accf = su32(acc_full),
                   b_acce = su32(acc_empty), ring = su32(smem);

    if (warp == 0 || warp == 3) {
        // One warp per operand, one lane of it issuing: two loads of a stage
        // by one thread would take as long as the stage's products.
        const int is_b = warp == 3;
        const bool one = elect_one();
        const uint32_t b_out = CG == 2 ? in_leader(b_full) : b_full;
        uint32_t s = 0, par = 1, issued = 0;  // the first pass over the ring finds it empty
        bool ok = true;
        for (uint32_t round = 0; ok; round++) {
            uint32_t j = 0, lt = tile_of(round, first, step);
            if (lt >= W.tiles) break;
            while (lt >= W.job[j].tiles) lt -= W.job[j++].tiles;
            const uint32_t tm = W.job[j].tm, slice = lt / W.job[j].plane;
            lt -= slice * W.job[j].plane;
            const CUtensorMap* map = &W.map[2 * j + is_b];
            const bool mn = is_b ? W.job[j].b_mn : W.job[j].a_mn;
            const int r0 = (int)((is_b ? lt / tm : lt % tm) * NC + rank * BT);
            const int first_k = (int)slice * W.job[j].kslice;
            const int K = min(W.job[j].K, first_k + W.job[j].kslice);
            for (int k0 = first_k; k0 < K && ok; k0 += BK) {
#pragma unroll
                for (int p = 0; p < (SIX ? 6 : 1); p++) {
                    ok = warp_wait(b_empty + s * 8, par, &s_err);
                    if (!ok) break;
                    const int z = !SIX ? 0 : is_b ? prod_b(p) : prod_a(p);
                    const uint32_t dst = ring + s * ST_BYTES + is_b * OP_BYTES, bar = b_out + s * 8;
                    if (one) {
                        if (rank == 0 && !is_b) mbar_expect_tx(b_full + s * 8, ST_BYTES * CG);
                        if (mn) {
                            tma_load<CG>(dst, map, r0, k0, z, bar);
                            tma_load<CG>(dst + BK * 128, map, r0 + 64, k0, z, bar);
                        } else {
                            tma_load<CG>(dst, map, k0, r0, z, bar);
                        }
                    }
                    issued++;
                    if (++s == ST) s = 0, par ^= 1;
                }
            }
        }
        // The last stages are read (and the pair's arrivals here made) before
        // the CTA's shared memory goes away; after a timeout, the loads land.
        for (uint32_t i = 0; i < ST && i < issued && ok; i++) {
            if (s == 0) s = ST, par ^= 1;
            s--;
            ok = warp_wait(b_empty + s * 8, par ^ 1, &s_err);
        }
        if (!ok)  // a millisecond, in which every load in flight has long landed
            for (int w = 0; w < 1000; w++) __nanosleep(1000);
    } else if (warp == 1 && rank == 0) {
        const bool one = elect_one();
        uint32_t s = 0, par = 0, ph = 0;
        bool ok = true;
        for (uint32_t round = 0; ok; round++) {
            uint32_t j = 0, lt = tile_of(round, first, step);
            if (lt >= W.tiles) break;
            while (lt >= W.job[j].tiles) lt -= W.job[j++].tiles;
            const bool a_mn = W.job[j].a_mn, b_mn = W.job[j].b_mn;
            const uint32_t id = idesc<CG>(a_mn, b_mn);
            const uint64_t ka = kstep(a_mn), kb = kstep(b_mn);
            const uint64_t da0 = sdesc(ring, a_mn), db0 = sdesc(ring + OP_BYTES, b_mn);
            const int KB = k_blocks(W.job[j], lt);
            const int phases = SIX ? KB : 1, per = SIX ? 6 : KB;
            for (int f = 0; f < phases && ok; f++, ph++) {
                const uint32_t buf = ph & 1;
                // the first two phases find the accumulators free
                ok = warp_wait(b_acce + buf * 8, ((ph >> 1) + 1) & 1, &s_err);
                if (!ok) break;
                TC_AFTER();
                const uint32_t d = tmem + buf * NC;
                for (int v = 0; v < per; v++) {
                    ok = warp_wait(b_full + s * 8, par, &s_err);
                    if (!ok) break;
                    TC_AFTER();
                    if (one) {
                        const uint64_t at = (uint64_t)(s * (ST_BYTES >> 4));
                        const uint64_t da = da0 + at, db = db0 + at;
#pragma unroll
                        for (int k = 0; k < BK / 16; k++)
                            umma_bf16<CG>(d, da + k * ka, db + k * kb, id, (v | k) ? 1u : 0u);
                        umma_commit<CG>(b_empty + s * 8);
                    }
                    if (++s == ST) s = 0, par ^= 1;
                }
                if (ok && one) umma_commit<CG>(b_accf + buf * 8);
            }
        }
        if (!ok && one) {  // products in flight end before tensor memory is freed
            umma_commit<CG>(su32(drain));
            for (uint32_t w = 0; w < (1u << 14) && !mbar_try(su32(drain), 0); w++) __nanosleep(100);
        }
    } else if (warp >= 4) {
        const int q = warp & 3, h = (warp - 4) >> 2;
        const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + h * HALF;
        const uint32_t b_free = in_leader(b_acce);
        float* tr = reinterpret_cast<float*>(smem + ST * ST_BYTES + 256) + (warp - 4) * (32 * 33);
        uint32_t ph = 0;
        bool ok = true;
        for (uint32_t round = 0; ok; round++) {
            uint32_t j = 0, lt = tile_of(round, first, step);
            if (lt >= W.tiles) break;
            while (lt >= W.job[j].tiles) lt -= W.job[j++].tiles;
            const Job& g = W.job[j];
            const int KB = k_blocks(g, lt);
            const uint32_t slice = lt / g.plane;
            lt -= slice * g.plane;
            const int row = (int)(lt % g.tm * NC) + rank * BT + q * 32 + lane;
            const int n0 = (int)(lt / g.tm * NC) + h * HALF;
            if constexpr (SIX) {
                float acc[HALF / 32][32];
#pragma unroll
                for (int c = 0; c < HALF / 32; c++)
#pragma unroll
                    for (int e = 0; e < 32; e++) acc[c][e] = 0.0f;
                for (int f = 0; f < KB; f++, ph++) {
                    const uint32_t buf = ph & 1;
                    ok = warp_wait(b_accf + buf * 8, (ph >> 1) & 1, &s_err);
                    if (!ok) break;
                    TC_AFTER();
#pragma unroll
                    for (int c = 0; c < HALF / 32; c++) {
                        float v[32];
                        tmem_ld32(v, lanes + buf * NC + c * 32);
#pragma unroll
                        for (int e = 0; e < 32; e++) acc[c][e] += v[e];
                    }
                    TC_BEFORE();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_leader(b_free + buf * 8);
                }
                if (!ok) break;
                Row<SIX> r(g, row, n0, slice, tr);
#pragma unroll
                for (int c = 0; c < HALF / 32; c++) r.chunk(acc[c], c * 32);
                r.done(HALF);
            } else {
                const uint32_t buf = ph & 1;
                Row<SIX> r(g, row, n0, slice, tr);
                ok = warp_wait(b_accf + buf * 8, (ph >> 1) & 1, &s_err);
                if (!ok) break;
                ph++;
                TC_AFTER();
#pragma unroll 1
                for (int c = 0; c < HALF / 32; c++) {
                    float v[32];
                    tmem_ld32(v, lanes + buf * NC + c * 32);
                    r.chunk(v, c * 32);
                }
                TC_BEFORE();
                __syncwarp();
                if (lane == 0) mbar_arrive_leader(b_free + buf * 8);
                r.done(HALF);
            }
        }
    }
    __syncwarp();
    TC_BEFORE();
    __syncthreads();
    if (tid == 0 && s_err) atomicExch_system(W.err, 1);
    if constexpr (CG == 2) cluster_sync();
    if (warp == 2) {
        TC_AFTER();
        if constexpr (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS)
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS)
                         : "memory");
    }
    if constexpr (CG == 2) cluster_sync();
}

// ---- small kernels -----------------------------------------------------------------

// The largest |dloss| of the rows with a target, 1 where there is none that is
// positive and finite: the unit that dloss x is taken in, so that the equal
// dloss of a mean leaves x as it is, with no rounding.  The whole CTA.
template <int THREADS>
__device__ __forceinline__ float largest_dloss(const float* __restrict__ dloss, const void* labels,
                                               int index_bytes, long long vocab, long long n) {
    __shared__ float s[THREADS / 32];
    float m = 0.0f;
#pragma unroll 4
    for (long long i = threadIdx.x; i < n; i += THREADS) {
        const long long l = label_at(labels, index_bytes, i);
        const float v = fabsf(dloss[i]);
        if (l >= 0 && l < vocab) m = fmaxf(m, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = m;
    __syncthreads();
    m = s[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m > 0.0f && m < INFINITY ? m : 1.0f;
}
__global__ void __launch_bounds__(1024)
k_xent_unit(float* __restrict__ unit, const float* __restrict__ dloss, const void* labels,
            int index_bytes, long long vocab, long long n) {
    const float u = largest_dloss<1024>(dloss, labels, index_bytes, vocab, n);
    if (threadIdx.x == 0) *unit = u;
}

// Up to this many rows k_pack finds the unit itself, every CTA for itself, which costs
// less than a launch.
constexpr long long kOwnUnit = 2048;

// Tensors [rows][dim] as bf16 planes [planes][rows][ld], ld = dim rounded up to 64, one
// after the other: a warp per row, a lane 8 consecutive values at a time (the columns
// from dim on are written as zeros).  1 plane: rounded to bf16; 3: split3.
// A scaled tensor's (the first job's) row i becomes (dloss_i / *unit) x_i in f32 first,
// and a row without a target becomes zeros, so that what its x holds (NaN, infinities)
// never meets the zeros of its G row.
struct PackJob {
    bf16* dst;
    const void* src;
    long long rows;
    int vec;  // rows on 16-byte boundaries
    int scaled;
};
struct PackWork {
    PackJob job[3];
    int jobs, dim, ld;
    const float* dloss;
    float* unit;
    const void* labels;
    int index_bytes;
    long long vocab, n;
};
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
k_pack(const __grid_constant__ PackWork w) {
    long long all = 0;
    for (int i = 0; i < w.jobs; i++) all += w.job[i].rows;
    const int lane = threadIdx.x & 31, dim = w.dim, ld = w.ld;
    float unit = 1.0f;
    if (w.job[0].scaled && (long long)blockIdx.x * 8 < w.n) {  // this CTA has scaled rows
        if (w.n <= kOwnUnit) {
            unit = largest_dloss<256>(w.dloss, w.labels, w.index_bytes, w.vocab, w.n);
            if (blockIdx.x == 0 && threadIdx.x == 0) *w.unit = unit;
        } else {
            unit = *w.unit;
        }
    }
    for (long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); at < all; at += (long long)gridDim.x * 8) {
        long long r = at;
        int ji = 0;
        while (r >= w.job[ji].rows) r -= w.job[ji++].rows;
        const PackJob& g = w.job[ji];
        const long long plane = g.rows * ld;
        float f = 1.0f;
        bool has = true;
        if (g.scaled) {
            const long long l = label_at(w.labels, w.index_bytes, r);
            has = l >= 0 && l < w.vocab;
            f = __fdiv_rn(w.dloss[r], unit);
        }
        const T* sr = (const T*)g.src + r * dim;
        bf16* dr = g.dst + r * ld;
        constexpr int U = 4;  // groups of 8 whose loads are in flight together
        for (int c0 = lane * 8; c0 < ld; c0 += 256 * U) {
            alignas(16) T in[U][8];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + 256 * u;
                if (g.vec && c + 8 <= dim) {
#pragma unroll
                    for (int q = 0; q < (int)(8 * sizeof(T) / 16); q++)
                        reinterpret_cast<uint4*>(in[u])[q] = reinterpret_cast<const uint4*>(sr + c)[q];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) in[u][e] = c + e < dim ? sr[c + e] : T(0.0f);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + 256 * u;
                if (c >= ld) break;
                alignas(16) bf16 o[PLANES][8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float v = (float)in[u][e];
                    if (g.scaled) v = has ? v * f : 0.0f;
                    if constexpr (PLANES == 1) o[0][e] = __float2bfloat16_rn(v);
                    else split3(v, o[0][e], o[1][e], o[2][e]);
                }
#pragma unroll
                for (int k = 0; k < PLANES; k++)
                    *reinterpret_cast<uint4*>(dr + k * plane + c) = *reinterpret_cast<uint4*>(o[k]);
            }
        }
    }
}

// lse and loss of every row from its segments' maxima and sums: 32 rows a
// CTA, the segments in 32 strided groups per row, each group's maximum first
// and then its sum against it (independent loads, no chain of exponentials),
// the groups joined in a fixed order.
__global__ void __launch_bounds__(1024)
k_xent_join(float* __restrict__ loss, float* __restrict__ lse, const float* __restrict__ part_m,
            const float* __restrict__ part_s, const float* __restrict__ zlabel,
            const void* labels, int index_bytes, long long vocab, long long n, int segs) {
    __shared__ float sm[32][33], ss[32][33];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const long long row = (long long)blockIdx.x * 32 + tx;
    float m = -INFINITY, s = 0.0f;
    if (row < n) {
#pragma unroll 4
        for (int t = ty; t < segs; t += 32) m = fmaxf(m, part_m[(size_t)t * n + row]);
        // while every segment's maximum is -inf, its sum is 0 or NaN: added as it is
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
        for (int t = ty; t < segs; t += 32) {
            const float om = part_m[(size_t)t * n + row], os = part_s[(size_t)t * n + row];
            s += om == -INFINITY ? os : os * ex2((om - ref) * kLog2e);
        }
    }
    sm[ty][tx] = m;
    ss[ty][tx] = s;
    __syncthreads();
    // warp ty joins row ty of the CTA: lane k takes group k
    const long long my = (long long)blockIdx.x * 32 + ty;
    float gm = sm[tx][ty], gs = ss[tx][ty], top = gm;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    gs = gm == -INFINITY ? gs : gs * expf(gm - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) gs += __shfl_xor_sync(0xffffffffu, gs, o);
    if (tx == 0 && my < n) {
        // no finite maximum (a row of -inf or NaN): log 0 would say -inf
        const float ls = top == -INFINITY ? NAN : logf(gs);
        lse[my] = top + ls;
        const long long l = label_at(labels, index_bytes, my);
        // (top - z_label) + log s keeps small losses exact where lse - z_label cancels
        loss[my] = l >= 0 && l < vocab ? (top - zlabel[my]) + ls : 0.0f;
    }
}

// The same for few rows: a CTA per row.
__global__ void __launch_bounds__(256)
k_xent_join_row(float* __restrict__ loss, float* __restrict__ lse, const float* __restrict__ part_m,
                const float* __restrict__ part_s, const float* __restrict__ zlabel,
                const void* labels, int index_bytes, long long vocab, long long n, int segs) {
    __shared__ float sh[8];
    const long long row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY, s = 0.0f;
#pragma unroll 4
    for (int t = threadIdx.x; t < segs; t += 256) m = fmaxf(m, part_m[(size_t)t * n + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) sh[warp] = m;
    __syncthreads();
    m = sh[lane & 7];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
    for (int t = threadIdx.x; t < segs; t += 256) {
        const float om = part_m[(size_t)t * n + row], os = part_s[(size_t)t * n + row];
        s += om == -INFINITY ? os : os * ex2((om - ref) * kLog2e);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();  // the maxima have been read
    if (lane == 0) sh[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = ((sh[0] + sh[1]) + (sh[2] + sh[3])) + ((sh[4] + sh[5]) + (sh[6] + sh[7]));
        const float ls = m == -INFINITY ? NAN : logf(s);  // as k_xent_join
        lse[row] = m + ls;
        const long long l = label_at(labels, index_bytes, row);
        loss[row] = l >= 0 && l < vocab ? (m - zlabel[row]) + ls : 0.0f;
    }
}

// ---- small problems ---------------------------------------------------------------
//
// For few multiply-adds per product the packing, the tensor maps and the
// pipeline's start cost more than the products.  k_small does them with f32 FMAs straight from the tensors, a
// TM x TN tile a CTA, KG groups of its threads taking every KG-th k of a chunk,
// added in order at the end: two launches forward (tiles, join) and two to four
// backward (P, both products, in one launch where they take the same tile, and
// where a long K is cut into slices, their sum).

// The limits on n vocab dim, from both paths' times in us (loss / gradient, this
// path's first): f32 16 x 200 x 100 12 / 13 and 18 / 27, 64 x 1001 x 1000 19 / 58 and
// 37 / 66, 100 x 100 x 1000 19 / 28 and 36 / 45, 256 x 512 x 512 21 / 53 and 25 / 41,
// 512 x 512 x 256 21 / 56 and 19 / 37; bf16 200 x 200 x 100 10 / 19 and 14 / 25 (not
// 16-byte rows), 64 x 300 x 400 12 / 19 and 12 / 23, 128 x 512 x 128 10 / 21 and 10 / 19,
// 64 x 1001 x 1000 21 / 60 and 14 / 29.  Above the f32 limit, 64 x 2000 x 1000 29 / 103
// and 37 / 70, 128 x 1001 x 1000 29 / 84 and 39 / 70, 64 x 4000 x 1000 51 / 187 and 41 /
// 85: the forward call alone would gain up to 2^27, one limit serves both.  Above the bf16
// limit, 64 x 1001 x 250 13 / 26 and 15 / 27, 128 x 512 x 256 12 / 27 and 13 / 19.
constexpr unsigned long long kSmallF32 = 1ull << 26, kSmallBf16 = 1ull << 23;  // f32 of more than 128 rows: half
constexpr int KSTEP = 128;  // slices of K are multiples of this, and of a tile's chunk KC

struct SmallJob {
    int kind;
    // LSE, GRAD: A [M][K] and B [N][K] of T; OUT: A f32, [M][K] or (a_mn) [K][M], B [K][N] of T
    const void *A, *B;
    int a_mn;
    long long lda, ldb;
    int M, N, K;
    int tm, tn, tiles;    // tiles of one slice, and of all
    int kslice;           // the k of a slice
    const float* bscale;  // OUT: a factor of B's row k, 0 without a target; or null
    // as in Job
    float *part_m, *part_s, *zlabel;
    const void* labels;
    int index_bytes;
    long long vocab;
    const float *lse, *dloss;
    float* p;             // GRAD: [M][N]
    void* out;            // OUT: T [M][N], or f32 [slice][M][N] where `partial`
    int partial;
};
struct SmallWork {
    SmallJob job[2];
    int jobs, tiles;
};

__device__ __forceinline__ float f32_of(float v) { return v; }
__device__ __forceinline__ float f32_of(bf16 v) { return __bfloat162float(v); }

// P: OUT jobs; else LSE or GRAD.
template <typename T, bool P, int TM, int TN, int RM, int RN, int KG, int KC>
__global__ void __launch_bounds__(TM / RM * (TN / RN) * KG)
k_small(const __grid_constant__ SmallWork w) {
    constexpr int GT = TM / RM * (TN / RN), NT = GT * KG;  // threads of a group, of the CTA
    constexpr int LA = TM * KC / NT, LB = TN * KC / NT;
    // the finished tile takes the place of the last chunk
    static_assert(RM == 4 && (RN == 2 || RN == 4) && KC % KG == 0 && KSTEP % KC == 0, "tile");
    __shared__ union alignas(16) {
        struct {
            float a[KC][TM + 4], b[KC][TN + 4];
        } in;
        float z[KG][TM][TN];
    } sh;
    auto& sa = sh.in.a;
    auto& sb = sh.in.b;
    auto& z = sh.z[0];
    const int tid = threadIdx.x;
    int lt = blockIdx.x, ji = 0;
    if (w.jobs > 1 && lt >= w.job[0].tiles) lt -= w.job[0].tiles, ji = 1;
    const SmallJob& g = w.job[ji];
    const int slice = lt / (g.tm * g.tn), in = lt - slice * (g.tm * g.tn);
    const int m0 = in % g.tm * TM, n0 = in / g.tm * TN;
    const int k_lo = slice * g.kslice, k_hi = min(g.K, k_lo + g.kslice);

    // A thread's elements of a chunk: where they lie, where they go, their k.  K-major
    // operands: a warp takes 4 rows x 8 k (whole sectors), and with a pitch of 4
    // mod 32 floats its transposed stores meet 32 banks.
    using TA = std::conditional_t<P, float, T>;
    const bool a_mn = P && g.a_mn;
    const TA* pa[LA];
    const T* pb[LB];
    int oa[LA], ob[LB], ka[LA], kb[LB];
#pragma unroll
    for (int i = 0; i < LA; i++) {
        const int x = tid + i * NT;
        const int r = a_mn ? x % TM : (x & 3) + 4 * ((x >> 5) / (KC / 8));
        const int k = a_mn ? x / TM : ((x >> 2) & 7) + 8 * ((x >> 5) % (KC / 8));
        pa[i] = (const TA*)g.A + (a_mn ? (size_t)(k_lo + k) * g.lda + m0 + r : (size_t)(m0 + r) * g.lda + k_lo + k);
        oa[i] = k * (TM + 4) + r;
        ka[i] = m0 + r < g.M ? k_lo + k : INT_MAX;
    }
#pragma unroll
    for (int i = 0; i < LB; i++) {
        const int x = tid + i * NT;
        const int r = P ? x % TN : (x & 3) + 4 * ((x >> 5) / (KC / 8));
        const int k = P ? x / TN : ((x >> 2) & 7) + 8 * ((x >> 5) % (KC / 8));
        pb[i] = (const T*)g.B + (P ? (size_t)(k_lo + k) * g.ldb + n0 + r : (size_t)(n0 + r) * g.ldb + k_lo + k);
        ob[i] = k * (TN + 4) + r;
        kb[i] = n0 + r < g.N ? k_lo + k : INT_MAX;
    }
    const size_t step_a = a_mn ? (size_t)KC * g.lda : KC, step_b = P ? (size_t)KC * g.ldb : KC;
    float ra[LA], rb[LB];
    // the next chunk, whose first k is kd further than the first one's
    auto fetch = [&](int kd) {
#pragma unroll
        for (int i = 0; i < LA; i++) {
            ra[i] = ka[i] < k_hi - kd ? f32_of(*pa[i]) : 0.0f;
            pa[i] += step_a;
        }
#pragma unroll
        for (int i = 0; i < LB; i++) {
            const bool in = kb[i] < k_hi - kd;
            float v = in ? f32_of(*pb[i]) : 0.0f;
            pb[i] += step_b;
            if (P && g.bscale && in) {
                // a row without a target counts as zeros, whatever it holds
                const long long l = label_at(g.labels, g.index_bytes, kb[i] + kd);
                v = l >= 0 && l < g.vocab ? v * g.bscale[kb[i] + kd] : 0.0f;
            }
            rb[i] = v;
        }
    };
    const int grp = tid / GT, gt = tid % GT;
    const int mr = gt % (TM / RM) * RM, nr = gt / (TM / RM) * RN;
    float acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; i++)
#pragma unroll
        for (int j = 0; j < RN; j++) acc[i][j] = 0.0f;
    fetch(0);
    for (int k0 = k_lo; k0 < k_hi; k0 += KC) {
        __syncthreads();  // the last chunk has been read
#pragma unroll
        for (int i = 0; i < LA; i++) sa[0][oa[i]] = ra[i];
#pragma unroll
        for (int i = 0; i < LB; i++) sb[0][ob[i]] = rb[i];
        __syncthreads();
        if (k0 + KC < k_hi) fetch(k0 + KC - k_lo);
#pragma unroll
        for (int k = grp; k < KC; k += KG) {
            float a[RM], b[RN];
            const float4 a4 = *reinterpret_cast<const float4*>(&sa[k][mr]);
            a[0] = a4.x, a[1] = a4.y, a[2] = a4.z, a[3] = a4.w;
            if constexpr (RN == 4) {
                const float4 b4 = *reinterpret_cast<const float4*>(&sb[k][nr]);
                b[0] = b4.x, b[1] = b4.y, b[2] = b4.z, b[3] = b4.w;
            } else {
                const float2 b2 = *reinterpret_cast<const float2*>(&sb[k][nr]);
                b[0] = b2.x, b[1] = b2.y;
            }
#pragma unroll
            for (int i = 0; i < RM; i++)
#pragma unroll
                for (int j = 0; j < RN; j++) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
    }
    // the groups' sums, in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RM; i++)
#pragma unroll
        for (int j = 0; j < RN; j++) sh.z[grp][mr + i][nr + j] = acc[i][j];
    __syncthreads();
    for (int x = tid; x < TM * TN; x += NT) {
        float v = sh.z[0][x / TN][x % TN];
#pragma unroll
        for (int q = 1; q < KG; q++) v += sh.z[q][x / TN][x % TN];
        z[x / TN][x % TN] = v;  // this thread's own element
    }
    __syncthreads();
    if (g.kind == LSE) {
        // a warp per row, a lane per column (and its 32nd next ones)
        const int lane = tid & 31;
        for (int r = tid >> 5; r < TM; r += NT / 32) {
            const int row = m0 + r;
            if (row >= g.M) break;
            float v[TN / 32], m = -INFINITY;
#pragma unroll
            for (int j = 0; j < TN / 32; j++) {
                const int c = lane + 32 * j;
                v[j] = n0 + c < g.N ? z[r][c] : -INFINITY;
                m = fmaxf(m, v[j]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float ref = m == -INFINITY ? 0.0f : m;  // as in chunk_lse
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < TN / 32; j++) s += ex2((v[j] - ref) * kLog2e);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const long long l = label_at(g.labels, g.index_bytes, row) - n0;
            if (lane == 0) {
                g.part_m[(size_t)(n0 / TN) * g.M + row] = m;
                g.part_s[(size_t)(n0 / TN) * g.M + row] = s;
                if (l >= 0 && l < TN && n0 + l < g.N) g.zlabel[row] = z[r][l];
            }
        }
        return;
    }
    for (int x = tid; x < TM * TN; x += NT) {
        const int row = m0 + x / TN, col = n0 + x % TN;
        if (row >= g.M || col >= g.N) continue;
        float v = z[x / TN][x % TN];
        const size_t at = (size_t)row * g.N + col;
        if (g.kind == GRAD) {
            const long long l = label_at(g.labels, g.index_bytes, row);
            v = ex2((v - g.lse[row]) * kLog2e) - (l == col ? 1.0f : 0.0f);
            g.p[at] = l >= 0 && l < g.vocab ? v : 0.0f;
        } else if (g.partial) {
            ((float*)g.out)[(size_t)slice * g.M * g.N + at] = v;
        } else {
            if (g.dloss) {
                const long long l = label_at(g.labels, g.index_bytes, row);
                v = l >= 0 && l < g.vocab ? v * g.dloss[row] : 0.0f;
            }
            if constexpr (sizeof(T) == 2) ((bf16*)g.out)[at] = __float2bfloat16_rn(v);
            else ((float*)g.out)[at] = v;
        }
    }
}

// out = the slices' partial products added in order, times the rows' dloss.
struct SumJob {
    const float* part;
    void* out;
    const float* dloss;   // or null
    const float* factor;  // of all, or null
    long long M, N;
    int slices;           // 0: no such job
};
struct SumWork {
    SumJob job[2];
    const void* labels;
    int index_bytes;
    long long vocab;
};
template <typename T>
__global__ void __launch_bounds__(256)
k_sum(const __grid_constant__ SumWork w) {
    const SumJob& g = w.job[blockIdx.y];
    const long long n = g.M * g.N;
    if (g.slices == 0) return;
    const float f = g.factor ? *g.factor : 1.0f;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float v = 0.0f;
#pragma unroll 4
        for (int s = 0; s < g.slices; s++) v += g.part[s * n + i];
        if (g.dloss) {
            const long long r = i / g.N, l = label_at(w.labels, w.index_bytes, r);
            v = l >= 0 && l < w.vocab ? v * g.dloss[r] : 0.0f;
        }
        v *= f;
        if constexpr (sizeof(T) == 2) ((bf16*)g.out)[i] = __float2bfloat16_rn(v);
        else ((float*)g.out)[i] = v;
    }
}

// ---- few rows ---------------------------------------------------------------------
//
// A few rows (one token's score, a handful of sequences): a product with them is a
// pass over w, bound by its bytes, and the tensor cores' 128-row tiles would be empty.
// k_few_z: x in shared memory as f32; a warp takes kFewC classes at a time, the lanes
// 16 bytes each of their rows, and every value of x that is read serves kFewC
// classes; then the lanes part the sums among them, one (class, row) each, which keeps
// its own running maximum and sum (forward) or stores P (backward).
// k_few_out: a thread holds (of up to 16 rows) some columns of x and of dx's sums in registers and goes
// down a slab of classes: dx += P w, dw = P^T (dloss x), w read and dw written once.
// All in f32, rounded once at the end.
// Measured, 1 x 65536 x 2048: f32 86 us forward (88 to 94 in a loop; w alone 82 at the measured copy rate),
// 272 us the gradient (w twice and dw 246); bf16 50 and 147 us (41 and 123).

constexpr unsigned kFewRows = 8, kFewC = 4;
constexpr unsigned kFewX = 16384;       // values of x: 64 KB of shared memory
constexpr unsigned kFewCtas = 148 * 2;  // fixed, as the workspace must not depend on the device

struct Few {
    const void *x, *w, *labels;
    int index_bytes;
    unsigned n, vocab, dim;
    float *part_m, *part_s, *zlabel;  // forward: [CTA][n], [CTA][n], [n]
    const float *lse, *dloss;
    float* p;     // backward: [vocab][ldp], ldp = the rows padded to k_few_out's NB
    unsigned ldp;
    float* part;  // [slab][n][dim]
    void *dx, *dw;
    unsigned parts;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(float (&v)[VEC], const T* p) {
    alignas(16) T e[VEC];
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    else {
#pragma unroll
        for (int i = 0; i < VEC; i++) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = f32_of(e[i]);
}

// VEC: 16 bytes of w where its rows are aligned, else 1.  blockIdx.y: NB of the rows.
template <typename T, int NB, int VEC, bool GRADIENT>
__global__ void __launch_bounds__(256, 2)
k_few_z(const __grid_constant__ Few f) {
    constexpr int C = kFewC, M = C * NB, U = VEC > 1 ? 2 : 4;
    extern __shared__ __align__(16) float xs[];  // [NB][dim]
    __shared__ float sm[8][M], ss[8][M];
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = f.dim;
    const unsigned r0 = blockIdx.y * NB, n = min(f.n - r0, (unsigned)NB);  // this CTA's rows
    for (unsigned i = threadIdx.x; i < NB * d; i += 256)
        xs[i] = i < n * d ? f32_of(((const T*)f.x)[(size_t)r0 * d + i]) : 0.0f;
    __syncthreads();
    // what the lane holds after the sums: class j of the C, row r
    constexpr int LG = M == 4 ? 2 : M == 8 ? 3 : M == 16 ? 4 : 5;
    const unsigned id = lane >> (5 - LG), j = id / NB, r = id % NB;
    const bool mine = (lane & ((1u << (5 - LG)) - 1)) == 0;  // of lanes with the same value
    const long long lab = r < n ? label_at(f.labels, f.index_bytes, r0 + r) : -1;
    const bool has = lab >= 0 && lab < f.vocab;
    const float lse = GRADIENT && r < n ? f.lse[r0 + r] : 0.0f;
    float m = -INFINITY, s = 0.0f;
    for (size_t v0 = ((size_t)blockIdx.x * 8 + warp) * C; v0 < f.vocab; v0 += (size_t)gridDim.x * 8 * C) {
        const T* w[C];
#pragma unroll
        for (int c = 0; c < C; c++) w[c] = (const T*)f.w + min(v0 + c, (size_t)f.vocab - 1) * d;
        float acc[M];
#pragma unroll
        for (int i = 0; i < M; i++) acc[i] = 0.0f;
#pragma unroll U
        for (unsigned k = lane * VEC; k < d; k += 32 * VEC) {
            float wv[C][VEC];
#pragma unroll
            for (int c = 0; c < C; c++) load_vec<T, VEC>(wv[c], w[c] + k);
#pragma unroll
            for (int q = 0; q < NB; q++) {
                float xv[VEC];
                if constexpr (VEC > 1) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 4) {
                        const float4 a = *reinterpret_cast<const float4*>(&xs[q * d + k + e]);
                        xv[e] = a.x, xv[e + 1] = a.y, xv[e + 2] = a.z, xv[e + 3] = a.w;
                    }
                } else {
                    xv[0] = xs[q * d + k];
                }
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) acc[c * NB + q] = fmaf(wv[c][e], xv[e], acc[c * NB + q]);
            }
        }
        // the lanes' sums: every step halves the values a lane holds
        __syncwarp();
#pragma unroll
        for (int h = M / 2, o = 16; o > 0; o >>= 1, h >>= 1) {
            if (h > 0) {
                const bool up = lane & o;
#pragma unroll
                for (int i = 0; i < M / 2; i++)
                    if (i < h) {
                        const float keep = up ? acc[i + h] : acc[i], give = up ? acc[i] : acc[i + h];
                        acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
            } else {
                acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
            }
        }
        const float z = acc[0];
        const size_t v = v0 + j;
        if (v < f.vocab) {
            if constexpr (GRADIENT) {
                float p = ex2((z - lse) * kLog2e);
                if ((long long)v == lab) p -= 1.0f;
                if (mine) f.p[v * f.ldp + r0 + r] = has ? p : 0.0f;
            } else {
                const float nm = fmaxf(m, z), ref = nm == -INFINITY ? 0.0f : nm;  // as in chunk_lse
                s = s * ex2((m - ref) * kLog2e) + ex2((z - ref) * kLog2e);
                m = nm;
                if (mine && (long long)v == lab) f.zlabel[r0 + r] = z;
            }
        }
    }
    if constexpr (!GRADIENT) {
        if (mine) sm[warp][id] = m, ss[warp][id] = s;
        __syncthreads();
        if (threadIdx.x < n) {
            m = -INFINITY, s = 0.0f;
            for (int i = 0; i < 8 * C; i++) m = fmaxf(m, sm[i / C][i % C * NB + threadIdx.x]);
            const float ref = m == -INFINITY ? 0.0f : m;
            for (int i = 0; i < 8 * C; i++) {
                const float om = sm[i / C][i % C * NB + threadIdx.x], os = ss[i / C][i % C * NB + threadIdx.x];
                s += om == -INFINITY ? os : os * ex2((om - ref) * kLog2e);
            }
            f.part_m[(size_t)blockIdx.x * f.n + r0 + threadIdx.x] = m;
            f.part_s[(size_t)blockIdx.x * f.n + r0 + threadIdx.x] = s;
        }
    }
}

// blockDim = (threads over columns, groups that take classes of their own), 256 in all;
// blockIdx.x: 256-thread block of columns, blockIdx.y: slab.
template <typename T, int NB, int VEC>
__global__ void __launch_bounds__(256, NB * VEC > 32 ? 1 : 2)
k_few_out(const __grid_constant__ Few f) {
    constexpr int U = 8;  // classes whose loads are in flight together
    __shared__ float red[256][VEC];
    const unsigned tx = blockDim.x, t = threadIdx.x, ty = blockDim.y, g = threadIdx.y, d = f.dim;
    const size_t c0 = ((size_t)blockIdx.x * tx + t) * VEC;
    const bool in = c0 < d;  // whole vectors: d is a multiple of VEC
    float x[NB][VEC], acc[NB][VEC];
#pragma unroll
    for (int r = 0; r < NB; r++) {
        const long long l = r < (int)f.n ? label_at(f.labels, f.index_bytes, r) : -1;
        const bool has = l >= 0 && l < f.vocab;
        const float dl = has ? f.dloss[r] : 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            // a row without a target counts as zeros, whatever it holds
            x[r][e] = in && has ? dl * f32_of(((const T*)f.x)[(size_t)r * d + c0 + e]) : 0.0f;
            acc[r][e] = 0.0f;
        }
    }
    const size_t groups = (size_t)gridDim.y * ty, per = (f.vocab + groups - 1) / groups;
    const size_t first = ((size_t)blockIdx.y * ty + g) * per, last = min(first + per, (size_t)f.vocab);
    if (in) {
        for (size_t v0 = first; v0 < last; v0 += U) {
            float w[U][VEC];
#pragma unroll
            for (int u = 0; u < U; u++) load_vec<T, VEC>(w[u], (const T*)f.w + min(v0 + u, last - 1) * d + c0);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const size_t v = v0 + u;
                if (v >= last) break;
                float p[NB];
                if constexpr (NB >= 4) {
#pragma unroll
                    for (int r = 0; r < NB; r += 4) {
                        const float4 a = *reinterpret_cast<const float4*>(f.p + v * NB + r);
                        p[r] = a.x, p[r + 1] = a.y, p[r + 2] = a.z, p[r + 3] = a.w;
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < NB; r++) p[r] = f.p[v * NB + r];
                }
                alignas(16) T o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    float q = 0.0f;
#pragma unroll
                    for (int r = 0; r < NB; r++) {
                        q = fmaf(p[r], x[r][e], q);
                        acc[r][e] = fmaf(p[r], w[u][e], acc[r][e]);
                    }
                    if constexpr (sizeof(T) == 2) o[e] = __float2bfloat16_rn(q);
                    else o[e] = q;
                }
                T* out = (T*)f.dw + v * d + c0;
                if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(o);
                else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(o);
                else out[0] = o[0];
            }
        }
    }
    // the groups' sums, in order
#pragma unroll
    for (int r = 0; r < NB; r++) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; e++) red[g * tx + t][e] = acc[r][e];
        __syncthreads();
        if (g == 0 && in && r < (int)f.n) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                float v = red[t][e];
                for (unsigned q = 1; q < ty; q++) v += red[q * tx + t][e];
                f.part[((size_t)blockIdx.y * f.n + r) * d + c0 + e] = v;
            }
        }
    }
}

// dx = dloss times the slabs' sums, added in a fixed order (32 strided sums of an
// element, then a tree).
template <typename T>
__global__ void __launch_bounds__(1024)
k_few_fold(const __grid_constant__ Few f) {
    __shared__ float t[32][33];
    const size_t all = (size_t)f.n * f.dim, i = (size_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (i < all) {
#pragma unroll 4
        for (unsigned k = threadIdx.y; k < f.parts; k += 32) s += f.part[k * all + i];
    }
    t[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = t[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const size_t q = (size_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && q < all) {
        const unsigned r = (unsigned)(q / f.dim);
        const long long l = label_at(f.labels, f.index_bytes, r);
        const float v = l >= 0 && l < f.vocab ? s * f.dloss[r] : 0.0f;
        if constexpr (sizeof(T) == 2) ((bf16*)f.dx)[q] = __float2bfloat16_rn(v);
        else ((float*)f.dx)[q] = v;
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

template <int CG, bool SIX>
int launch_work(Ctx& c, const Work& w) {
    NXV_CK(cudaFuncSetAttribute(k_xgemm<CG, SIX>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(std::min<uint32_t>(w.tiles, c.dev->sm_count / CG) * CG));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NXV_CK(cudaLaunchKernelEx(&cfg, k_xgemm<CG, SIX>, w));
    count_launch();
    return OK;
}

int run_work(Ctx& c, Work& w, int cg, bool six) {
    w.err = wait_flag(c);
    if (cg == 2) return six ? launch_work<2, true>(c, w) : launch_work<2, false>(c, w);
    return six ? launch_work<1, true>(c, w) : launch_work<1, false>(c, w);
}

// Slices of the K of an [M, N] product of few tiles, so that it does not run on a
// few SMs while the others wait: each slice is at least 16 k-blocks.
int out_slices(size_t M, size_t N, size_t K, int cg) {
    const size_t t = (size_t)BT * cg, tiles = ((M + t - 1) / t) * ((N + t - 1) / t);
    const size_t units = 148 / cg, kb = (K + BK - 1) / BK;
    if (tiles * 2 > units || kb < 32) return 1;
    return (int)std::min(units / tiles, kb / 16);
}

// The K of one of `slices` slices.
int slice_k(size_t K, int slices) { return (int)(((K + slices - 1) / slices + BK - 1) / BK * BK); }

// Adds a job; jobs with a longer K come first.  kslice: 0 for all of K.
void add_job(Work& w, Job j, const CUtensorMap& a, const CUtensorMap& b, int cg, int kslice = 0) {
    const int t = BT * cg;
    j.tm = (j.M + t - 1) / t;
    j.plane = j.tm * ((j.N + t - 1) / t);  // below 2^31: the entry points check
    j.kslice = kslice ? kslice : slice_k(j.K, 1);
    j.tiles = j.plane * ((j.K + j.kslice - 1) / j.kslice);
    int at = w.jobs;
    while (at > 0 && w.job[at - 1].kslice < j.kslice) {
        w.job[at] = w.job[at - 1];
        w.map[2 * at] = w.map[2 * at - 2];
        w.map[2 * at + 1] = w.map[2 * at - 1];
        at--;
    }
    w.job[at] = j;
    w.map[2 * at] = a;
    w.map[2 * at + 1] = b;
    w.jobs++;
    w.tiles += j.tiles;
}

size_t up(size_t v, size_t to) { return (v + to - 1) / to * to; }

// How a call uses its workspace.  The vocabulary is cut into pieces of vp
// classes (a multiple of the widest tile) so that a piece's G, and its packed
// w where w cannot be read in place, stay within a fixed budget.  The gradient
// holds two pieces: a launch makes P of one while it multiplies the other.
struct Plan {
    int planes, cg;
    size_t dp;                // packed row length
    size_t vp, pieces;
    size_t seg;               // classes of one (maximum, sum) entry
    size_t xp, sp, unit, wp[2], g[2], ldg, acc, px, pw, pm, ps, zl, total;  // byte offsets; ldg in elements
    int sx, sw, ksx, ksw;     // slices of K of dx and of dw, and their length
};

constexpr size_t kPieceBytes = (size_t)256 << 20;
constexpr size_t kTile = 2 * BT;

Plan make_plan(const XentP& p, bool grad) {
    Plan q{};
    q.planes = p.dt == F32 ? 3 : 1;
    // Pairs' tiles read half as much per product, but where the single tiles of the logits
    // fit the SMs at once these finish sooner (512 x 4000 x 768 bf16 14.4 / 38 us instead
    // of 16.5 / 43, 400 x 1000 x 1000 f32 41 / 81 and 49 / 99; not 256 x 10000 x 512 f32,
    // two rounds of single tiles, 46 / 115 and 40 / 111).
    const size_t single = (((size_t)p.n + BT - 1) / BT) * (((size_t)p.vocab + BT - 1) / BT);
    q.cg = p.n > BT && p.vocab > BT && single > 148 ? 2 : 1;
    q.seg = (size_t)BT * q.cg / 2;
    // whole 128-byte lines: a box row that straddles two costs two requests
    // (2048 x 8192 x 1000 f32: 750 instead of 510 cycles per stage)
    q.dp = up(p.dim, 64);
    const size_t per_class = (size_t)q.planes * 2 * (q.dp + (grad ? (size_t)p.n : 0));
    size_t vp = std::max<size_t>(kPieceBytes / per_class / kTile * kTile, 4 * kTile);
    const size_t all = up(p.vocab, kTile);
    vp = std::min(vp, all);
    q.pieces = (p.vocab + vp - 1) / vp;
    q.vp = up((p.vocab + q.pieces - 1) / q.pieces, kTile);
    q.pieces = (p.vocab + q.vp - 1) / q.vp;
    q.ldg = q.vp;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up(bytes, 1024);
        return o;
    };
    q.xp = take((size_t)q.planes * 2 * p.n * q.dp);
    for (int b = 0; b < 2; b++)
        q.wp[b] = b < (grad ? (int)q.pieces : 1) ? take((size_t)q.planes * 2 * q.vp * q.dp) : q.wp[0];
    if (grad) {
        q.sp = take((size_t)q.planes * 2 * p.n * q.dp);
        q.unit = take(4);
        for (int b = 0; b < 2; b++)
            q.g[b] = b < (int)q.pieces ? take((size_t)q.planes * 2 * p.n * q.ldg) : q.g[0];
        // (the last piece, if shorter, fills fewer slices of dx's sums)
        const size_t most = std::min<size_t>(q.vp, p.vocab);
        q.ksx = slice_k(most, out_slices(p.n, p.dim, most, q.cg));
        q.sx = (int)((most + q.ksx - 1) / q.ksx);
        q.ksw = slice_k(p.n, out_slices(most, p.dim, p.n, q.cg));
        q.sw = (int)((p.n + q.ksw - 1) / q.ksw);
        q.acc = take(p.dt == BF16 && q.pieces > 1 && q.sx == 1 ? (size_t)4 * p.n * p.dim : 0);
        q.px = take(q.sx > 1 ? (size_t)4 * q.sx * p.n * p.dim : 0);
        q.pw = take(q.sw > 1 ? (size_t)4 * q.sw * q.vp * p.dim : 0);
    } else {
        const size_t segs = (p.vocab + q.seg - 1) / q.seg;
        q.pm = take(4 * segs * p.n);
        q.ps = take(4 * segs * p.n);
        q.zl = take((size_t)4 * p.n);
    }
    q.total = at;
    return q;
}

// Adds a tensor to what a launch of k_pack makes; a scaled one first.
void pack_add(PackWork& w, const XentP& p, bf16* dst, const void* src, size_t rows, bool scaled = false) {
    w.job[w.jobs++] = {dst, src, (long long)rows,
                       ((uintptr_t)src & 15) == 0 && p.dim * dtype_bytes(p.dt) % 16 == 0, scaled};
}
void run_pack(Ctx& c, const XentP& p, PackWork& w, int ld) {
    if (w.jobs == 0) return;
    w.dim = (int)p.dim;
    w.ld = ld;
    w.labels = p.labels;
    w.index_bytes = p.index_bytes;
    w.vocab = p.vocab;
    w.n = p.n;
    size_t rows = 0;
    for (int i = 0; i < w.jobs; i++) rows += w.job[i].rows;
    const unsigned grid = grid_for(c, rows, 8, 16);
    if (p.dt == F32) k_pack<float, 3><<<grid, 256, 0, c.stream>>>(w);
    else k_pack<bf16, 1><<<grid, 256, 0, c.stream>>>(w);
    count_launch();
    w = PackWork{};
}

// A tensor can feed TMA where it lies when its rows start on 16-byte boundaries.
bool in_place(const XentP& p, const void* t) {
    return p.dt == BF16 && p.dim % 8 == 0 && ((uintptr_t)t & 15) == 0;
}

void join(Ctx& c, const XentP& p, void* loss, void* lse, const float* pm, const float* ps,
          const float* zl, size_t segs) {
    if (p.n <= 512)
        k_xent_join_row<<<p.n, 256, 0, c.stream>>>((float*)loss, (float*)lse, pm, ps, zl, p.labels,
                                                   p.index_bytes, p.vocab, p.n, (int)segs);
    else
        k_xent_join<<<(p.n + 31) / 32, dim3(32, 32), 0, c.stream>>>((float*)loss, (float*)lse, pm, ps,
                                                                    zl, p.labels, p.index_bytes,
                                                                    p.vocab, p.n, (int)segs);
    count_launch();
}

// ---- host: small problems --------------------------------------------------------

bool is_small(const XentP& p) {
    const unsigned long long most = p.dt == BF16 ? kSmallBf16 : p.n > BT ? kSmallF32 / 2 : kSmallF32;
    const unsigned long long n = up(p.n, 16);  // whole row tiles
    // no overflow: the entry points bound the tiles, and so n vocab, below 2^45
    return n * p.vocab <= most && n * p.vocab * p.dim <= most;
}

// The tile: 64 x 64 where that gives every SM one and is not mostly empty, else 16 x 32.
struct SmallTile {
    int m, n;
};
SmallTile small_tile(size_t M, size_t N) {
    const size_t big = ((M + 63) / 64) * ((N + 63) / 64);
    return M > 32 && N > 32 && big >= 148 ? SmallTile{64, 64} : SmallTile{16, 32};
}
// Slices of a long K where the tiles leave SMs idle: each at least 256 k.
int small_slices(size_t tiles, size_t K) {
    if (K < 512 || tiles * 2 > 148) return 1;
    return (int)std::min(K / 256, 148 / tiles);
}
size_t tiles_of(const SmallTile& t, size_t M, size_t N) {
    return ((M + t.m - 1) / t.m) * ((N + t.n - 1) / t.n);
}
int slices_of(const SmallTile& t, size_t M, size_t N, size_t K) { return small_slices(tiles_of(t, M, N), K); }

void small_add(SmallWork& w, SmallJob j, const SmallTile& t, int slices) {
    j.tm = (j.M + t.m - 1) / t.m;
    j.tn = (j.N + t.n - 1) / t.n;
    j.kslice = ((j.K + slices - 1) / slices + KSTEP - 1) / KSTEP * KSTEP;
    slices = (j.K + j.kslice - 1) / j.kslice;
    j.tiles = j.tm * j.tn * slices;
    w.job[w.jobs++] = j;
    w.tiles += j.tiles;
}

template <typename T, bool P>
void run_small_t(Ctx& c, const SmallWork& w, const SmallTile& t) {
    if (t.m == 64) k_small<T, P, 64, 64, 4, 4, 2, 64><<<w.tiles, 512, 0, c.stream>>>(w);
    else if (!P && w.job[0].K >= 512)  // a longer chunk hides more of its loads' latency
        k_small<T, P, 16, 32, 4, 2, 8, 128><<<w.tiles, 512, 0, c.stream>>>(w);
    else k_small<T, P, 16, 32, 4, 2, 8, 64><<<w.tiles, 512, 0, c.stream>>>(w);
    count_launch();
}
void run_small(Ctx& c, int dt, const SmallWork& w, const SmallTile& t) {
    const bool out = w.job[0].kind == OUT;
    if (dt == F32) out ? run_small_t<float, true>(c, w, t) : run_small_t<float, false>(c, w, t);
    else out ? run_small_t<bf16, true>(c, w, t) : run_small_t<bf16, false>(c, w, t);
}

// Workspace, in bytes: forward part_m, part_s [segments][n] and zlabel [n];
// backward P [n][vocab] and the slices' products.
struct SmallPlan {
    SmallTile z, tx, tw;  // of the logits, of dx, of dw
    size_t segs, pm, ps, zl, p, dx, dw, total;
    int sx, sw;  // slices of dx, dw
};
SmallPlan small_plan(const XentP& p, bool grad) {
    SmallPlan q{};
    q.z = small_tile(p.n, p.vocab);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up(bytes, 256);
        return o;
    };
    if (!grad) {
        q.segs = (p.vocab + q.z.n - 1) / q.z.n;
        q.pm = take(4 * q.segs * p.n);
        q.ps = take(4 * q.segs * p.n);
        q.zl = take((size_t)4 * p.n);
    } else {
        q.tx = small_tile(p.n, p.dim);
        q.tw = small_tile(p.vocab, p.dim);
        q.sx = slices_of(q.tx, p.n, p.dim, p.vocab);
        q.sw = slices_of(q.tw, p.vocab, p.dim, p.n);
        q.p = take((size_t)4 * p.n * p.vocab);
        q.dx = take(q.sx > 1 ? (size_t)4 * q.sx * p.n * p.dim : 0);
        q.dw = take(q.sw > 1 ? (size_t)4 * q.sw * p.vocab * p.dim : 0);
    }
    q.total = std::max<size_t>(at, 256);
    return q;
}

SmallJob small_logits(const XentP& p, int kind) {
    SmallJob j{};
    j.kind = kind;
    j.A = p.x;
    j.B = p.w;
    j.lda = j.ldb = p.dim;
    j.M = (int)p.n;
    j.N = (int)p.vocab;
    j.K = (int)p.dim;
    j.labels = p.labels;
    j.index_bytes = p.index_bytes;
    j.vocab = p.vocab;
    return j;
}

void run_sum(Ctx& c, const XentP& p, SumWork& s) {
    s.labels = p.labels;
    s.index_bytes = p.index_bytes;
    s.vocab = p.vocab;
    size_t n = 0;
    for (const SumJob& j : s.job) n = std::max(n, j.slices ? (size_t)(j.M * j.N) : 0);
    const dim3 grid(grid_for(c, n, 256, 8), 2);
    if (p.dt == F32) k_sum<float><<<grid, 256, 0, c.stream>>>(s);
    else k_sum<bf16><<<grid, 256, 0, c.stream>>>(s);
    count_launch();
}

int small_xent(Ctx& c, const XentP& p, void* loss, void* lse, void* ws) {
    const SmallPlan q = small_plan(p, false);
    char* base = (char*)ws;
    SmallJob j = small_logits(p, LSE);
    j.part_m = (float*)(base + q.pm);
    j.part_s = (float*)(base + q.ps);
    j.zlabel = (float*)(base + q.zl);
    SmallWork w{};
    small_add(w, j, q.z, 1);
    run_small(c, p.dt, w, q.z);
    join(c, p, loss, lse, j.part_m, j.part_s, j.zlabel, q.segs);
    pdl_record_all(c);
    return finish(c);
}

int small_xent_grad(Ctx& c, const XentP& p, void* dx, void* dw, const void* dloss, const void* lse,
                    void* ws) {
    const SmallPlan q = small_plan(p, true);
    char* base = (char*)ws;
    SmallJob z = small_logits(p, GRAD);
    z.lse = (const float*)lse;
    z.p = (float*)(base + q.p);
    SmallWork w{};
    small_add(w, z, q.z, 1);
    run_small(c, p.dt, w, q.z);
    SmallWork o{};
    // dx = dloss (P w)
    SmallJob j = small_logits(p, OUT);
    j.A = z.p;
    j.B = p.w;
    j.lda = p.vocab;
    j.ldb = p.dim;
    j.N = (int)p.dim;
    j.K = (int)p.vocab;
    j.partial = q.sx > 1;
    j.out = j.partial ? base + q.dx : dx;
    j.dloss = (const float*)dloss;
    small_add(o, j, q.tx, q.sx);
    const int sx = o.job[0].tiles / (o.job[0].tm * o.job[0].tn);
    if (q.tx.m != q.tw.m) {
        run_small(c, p.dt, o, q.tx);
        o = SmallWork{};
    }
    // dw = P^T (dloss x)
    j.a_mn = 1;
    j.B = p.x;
    j.bscale = (const float*)dloss;
    j.dloss = nullptr;
    j.M = (int)p.vocab;
    j.K = (int)p.n;
    j.partial = q.sw > 1;
    j.out = j.partial ? base + q.dw : dw;
    small_add(o, j, q.tw, q.sw);
    const SmallJob& jw = o.job[o.jobs - 1];
    const int sw = jw.tiles / (jw.tm * jw.tn);
    run_small(c, p.dt, o, q.tw);
    if (q.sx > 1 || q.sw > 1) {
        SumWork s{};
        if (q.sx > 1) s.job[0] = {(const float*)(base + q.dx), dx, (const float*)dloss, nullptr, p.n, p.dim, sx};
        if (q.sw > 1) s.job[1] = {(const float*)(base + q.dw), dw, nullptr, nullptr, p.vocab, p.dim, sw};
        run_sum(c, p, s);
    }
    pdl_record_all(c);
    return finish(c);
}

// ---- host: few rows ----------------------------------------------------------------

unsigned few_pad(unsigned n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16; }
// The rules' sides in us (this path's first), loss / gradient: f32 1 x 1000 x 1000 11 / 15
// and 19 / 45, 1 x 65536 x 2048 86 / 272 and 621 / 1143, 8 x 65536 x 2048 97 / 361 and
// 609 / 1078, 16 x 65536 x 2048 178 / 786 and 462 / 914,
// 16 x 4000 x 2000 gradient 65 and 132, forward only 24 x 2100 x 1000 17 and 19; bf16 1 x 65536 x 2048 50 / 147 and 80 / 315, 3 x 20001 x 777 17 / 69
// and 38 / 137, 8 x 65536 x 2048 93 / 320 and 79 / 298.
bool is_few(const XentP& p, bool grad) {
    if (std::min<size_t>(few_pad(p.n), 8) * p.dim > kFewX) return false;
    if (p.dt == BF16) return p.n <= (p.dim % 8 ? kFewRows : kFewRows / 2);
    // more rows of f32 read w again, which costs less than making its planes
    return p.n <= kFewRows ||
           (p.n <= (grad ? 2 : 3) * kFewRows && (size_t)p.vocab * p.dim >= (grad ? 1u << 20 : 1u << 21));
}

// Workspace, in bytes: forward part_m, part_s [CTAs][n] and zlabel; backward P and
// the slabs' sums.
struct FewPlan {
    unsigned ctas;      // of k_few_z
    unsigned tx, gx, gy;  // of k_few_out
    size_t pm, ps, zl, p, part, total;
};
// vec: columns of a thread of k_few_out
FewPlan few_plan(const XentP& p, bool grad, unsigned vec) {
    FewPlan q{};
    q.ctas = (unsigned)std::min<size_t>(((size_t)p.vocab + 8 * kFewC - 1) / (8 * kFewC), kFewCtas);
    const unsigned pieces = (p.dim + vec - 1) / vec;
    for (q.tx = 32; q.tx < pieces && q.tx < 256; q.tx *= 2) {}
    q.gx = (pieces + q.tx - 1) / q.tx;
    const size_t classes = 8 * (256 / q.tx);  // of a slab, at least
    q.gy = (unsigned)std::max<size_t>(1, std::min<size_t>((p.vocab + classes - 1) / classes, kFewCtas / q.gx));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up(bytes, 256);
        return o;
    };
    if (!grad) {
        q.pm = take((size_t)4 * q.ctas * p.n);
        q.ps = take((size_t)4 * q.ctas * p.n);
        q.zl = take((size_t)4 * p.n);
    } else {
        q.p = take((size_t)4 * p.vocab * few_pad(p.n));
        q.part = take((size_t)4 * q.gy * p.n * p.dim);
    }
    q.total = std::max<size_t>(at, 256);
    return q;
}
// Columns of a thread of k_few_out: 16 bytes (with 8 rows of bf16 and 16 of f32 8 bytes,
// for the registers) where w's and dw's rows are aligned to it, else 1.
unsigned few_vec(const XentP& p, bool aligned) {
    const unsigned nb = few_pad(p.n), most = p.dt == F32 ? (nb == 16 ? 2 : 4) : (nb == 8 ? 4 : 8);
    return aligned && p.dim % most == 0 ? most : 1;
}

template <typename T, int NB, bool GRADIENT>
int run_few_z(Ctx& c, const Few& f, unsigned ctas) {
    const dim3 grid(ctas, (f.n + NB - 1) / NB);
    constexpr int V = 16 / sizeof(T);
    const bool vec = f.dim % V == 0 && ((uintptr_t)f.w & 15) == 0;
    auto k = vec ? k_few_z<T, NB, V, GRADIENT> : k_few_z<T, NB, 1, GRADIENT>;
    const int bytes = (int)(NB * f.dim * 4);
    NXV_CK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    k<<<grid, 256, bytes, c.stream>>>(f);
    count_launch();
    return OK;
}

// NB: the rows, padded; k_few_z takes 8 of them at most.
template <typename T, int NB>
int few_t(Ctx& c, const XentP& p, Few f, bool grad, void* loss, void* lse, void* ws) {
    constexpr int NZ = NB > 8 ? 8 : NB;
    char* base = (char*)ws;
    int rc;
    if (!grad) {
        const FewPlan q = few_plan(p, false, 1);
        f.part_m = (float*)(base + q.pm);
        f.part_s = (float*)(base + q.ps);
        f.zlabel = (float*)(base + q.zl);
        if ((rc = run_few_z<T, NZ, false>(c, f, q.ctas))) return rc;
        join(c, p, loss, lse, f.part_m, f.part_s, f.zlabel, q.ctas);
        return OK;
    }
    const unsigned vec = few_vec(p, (((uintptr_t)f.w | (uintptr_t)f.dw) & 15) == 0);
    const FewPlan q = few_plan(p, true, vec);
    f.p = (float*)(base + q.p);
    f.part = (float*)(base + q.part);
    f.parts = q.gy;
    f.ldp = NB;
    if ((rc = run_few_z<T, NZ, true>(c, f, q.ctas))) return rc;
    constexpr int V = sizeof(T) == 4 ? (NB == 16 ? 2 : 4) : (NB == 8 ? 4 : 8);
    const dim3 grid(q.gx, q.gy), block(q.tx, 256 / q.tx);
    if (vec > 1) k_few_out<T, NB, V><<<grid, block, 0, c.stream>>>(f);
    else k_few_out<T, NB, 1><<<grid, block, 0, c.stream>>>(f);
    k_few_fold<T><<<(unsigned)(((size_t)p.n * p.dim + 31) / 32), dim3(32, 32), 0, c.stream>>>(f);
    count_launch(2);
    return OK;
}

// loss and lse are outputs of the forward call, lse an input of the gradient.
int few(Ctx& c, const XentP& p, bool grad, void* loss, void* lse, void* dx, void* dw, const void* dloss, void* ws) {
    Few f{};
    f.x = p.x, f.w = p.w, f.labels = p.labels, f.index_bytes = p.index_bytes;
    f.n = p.n, f.vocab = p.vocab, f.dim = p.dim;
    f.lse = (const float*)lse, f.dloss = (const float*)dloss;
    f.dx = dx, f.dw = dw;
    const unsigned nb = few_pad(p.n);
    int rc;
#define FEW(T) (nb == 1   ? few_t<T, 1>(c, p, f, grad, loss, lse, ws) \
                : nb == 2 ? few_t<T, 2>(c, p, f, grad, loss, lse, ws) \
                : nb == 4 ? few_t<T, 4>(c, p, f, grad, loss, lse, ws) \
                          : few_t<T, 8>(c, p, f, grad, loss, lse, ws))
    if (nb == 16) rc = few_t<float, 16>(c, p, f, grad, loss, lse, ws);  // f32 only: is_few
    else rc = p.dt == F32 ? FEW(float) : FEW(bf16);
#undef FEW
    if (rc) return rc;
    pdl_record_all(c);
    return finish(c);
}

}  // namespace

size_t xent_workspace(const XentP& p, bool grad) {
    if (is_few(p, grad)) return std::max(few_plan(p, grad, 1).total, few_plan(p, grad, few_vec(p, true)).total);
    return is_small(p) ? small_plan(p, grad).total : make_plan(p, grad).total;
}

int launch_xent(Ctx& c, const XentP& p, void* loss, void* lse, void* ws) {
    if (p.n == 0) return OK;
    if (is_few(p, false)) return few(c, p, false, loss, lse, nullptr, nullptr, nullptr, ws);
    if (is_small(p)) return small_xent(c, p, loss, lse, ws);
    const Plan q = make_plan(p, false);
    char* base = (char*)ws;
    const bool wip = in_place(p, p.w), xip = in_place(p, p.x);
    const bf16* xp = (const bf16*)p.x;
    PackWork packs{};
    if (!xip) {
        xp = (bf16*)(base + q.xp);
        pack_add(packs, p, (bf16*)xp, p.x, p.n);
    }
    CUtensorMap ma, mb;
    int rc;
    const size_t ldx = xip ? p.dim : q.dp, ldw = wip ? p.dim : q.dp;
    if ((rc = make_map(&ma, xp, p.dim, p.n, ldx, q.planes, p.n * ldx, BT))) return rc;
    Job g{};
    g.kind = LSE;
    g.M = (int)p.n;
    g.K = (int)p.dim;
    g.zlabel = (float*)(base + q.zl);
    g.labels = p.labels;
    g.index_bytes = p.index_bytes;
    g.vocab = p.vocab;
    const size_t vp = wip ? (size_t)p.vocab : q.vp;
    for (size_t v0 = 0; v0 < p.vocab; v0 += vp) {
        const size_t nv = std::min<size_t>(vp, p.vocab - v0);
        const bf16* wp = (const bf16*)p.w;
        if (!wip) {
            wp = (bf16*)(base + q.wp[0]);
            pack_add(packs, p, (bf16*)wp, (const char*)p.w + v0 * p.dim * dtype_bytes(p.dt), nv);
        }
        run_pack(c, p, packs, (int)q.dp);
        if ((rc = make_map(&mb, wp, p.dim, nv, ldw, q.planes, nv * ldw, BT))) return rc;
        g.N = (int)nv;
        g.col0 = (long long)v0;
        g.part_m = (float*)(base + q.pm) + v0 / q.seg * p.n;
        g.part_s = (float*)(base + q.ps) + v0 / q.seg * p.n;
        Work w{};
        add_job(w, g, ma, mb, q.cg);
        if ((rc = run_work(c, w, q.cg, q.planes == 3))) return rc;
    }
    join(c, p, loss, lse, (const float*)(base + q.pm), (const float*)(base + q.ps),
         (const float*)(base + q.zl), (p.vocab + q.seg - 1) / q.seg);
    pdl_record_all(c);
    return finish(c);
}

int launch_xent_grad(Ctx& c, const XentP& p, void* dx, void* dw, const void* dloss,
                     const void* lse, void* ws) {
    if (p.n == 0) {
        NXV_CK(cudaMemsetAsync(dw, 0, (size_t)p.vocab * p.dim * dtype_bytes(p.dt), c.stream));
        return finish(c);
    }
    if (is_few(p, true)) return few(c, p, true, nullptr, const_cast<void*>(lse), dx, dw, dloss, ws);
    if (is_small(p)) return small_xent_grad(c, p, dx, dw, dloss, lse, ws);
    const Plan q = make_plan(p, true);
    char* base = (char*)ws;
    const bool wip = in_place(p, p.w), six = q.planes == 3;
    const size_t es = dtype_bytes(p.dt);
    const bool xip = in_place(p, p.x);
    const size_t ldx = xip ? p.dim : q.dp, ldw = wip ? p.dim : q.dp;
    const bf16* xp = (const bf16*)p.x;
    bf16* sp = (bf16*)(base + q.sp);  // dloss x / unit
    float* unit = (float*)(base + q.unit);
    if (p.n > kOwnUnit) {
        k_xent_unit<<<1, 1024, 0, c.stream>>>(unit, (const float*)dloss, p.labels, p.index_bytes,
                                              p.vocab, p.n);
        count_launch();
    }
    PackWork packs{};
    packs.dloss = (const float*)dloss;
    packs.unit = unit;
    pack_add(packs, p, sp, p.x, p.n, true);
    if (!xip) {
        xp = (bf16*)(base + q.xp);
        pack_add(packs, p, (bf16*)xp, p.x, p.n);
    }
    const size_t gplane = (size_t)p.n * q.ldg;
    CUtensorMap mxk, mxn, mwk, mwn, mgk, mgm;
    int rc;
    // x: K-major A of z = x w^T; dloss x: N-major B of dw = G^T (dloss x)
    if ((rc = make_map(&mxk, xp, p.dim, p.n, ldx, q.planes, p.n * ldx, BT))) return rc;
    if ((rc = make_map(&mxn, sp, p.dim, p.n, q.dp, q.planes, p.n * q.dp, BK))) return rc;
    Job z{};
    z.kind = GRAD;
    z.M = (int)p.n;
    z.K = (int)p.dim;
    z.labels = p.labels;
    z.index_bytes = p.index_bytes;
    z.vocab = p.vocab;
    z.lse = (const float*)lse;
    z.ldg = (long long)q.ldg;
    z.gplane = six ? (long long)gplane : 0;
    // launch i: G of piece i, and the products of piece i - 1
    for (size_t i = 0; i <= q.pieces; i++) {
        Work w{};
        if (i > 0) {
            const size_t v0 = (i - 1) * q.vp, nv = std::min<size_t>(q.vp, p.vocab - v0);
            const bool first = i == 1, last = i == q.pieces;
            const bf16* gp = (const bf16*)(base + q.g[(i - 1) & 1]);
            const bf16* wp = wip ? (const bf16*)p.w + v0 * p.dim : (bf16*)(base + q.wp[(i - 1) & 1]);
            if ((rc = make_map(&mwn, wp, p.dim, nv, ldw, q.planes, nv * ldw, BK))) return rc;
            if ((rc = make_map(&mgk, gp, nv, p.n, q.ldg, q.planes, gplane, BT))) return rc;
            if ((rc = make_map(&mgm, gp, nv, p.n, q.ldg, q.planes, gplane, BK))) return rc;
            Job o{};
            o.kind = OUT;
            o.ldo = p.dim;
            o.N = (int)p.dim;
            o.b_mn = 1;
            // dx = dloss (sum of the pieces' G w): K runs over the piece's classes;
            // the sum so far is f32
            o.M = (int)p.n;
            o.K = (int)nv;
            if (q.sx > 1) {  // each slice's sum over the pieces; added up at the end
                o.out = base + q.px;
                o.acc_in = first ? nullptr : (const float*)(base + q.px);
            } else {
                o.out_bf16 = !six && last;
                o.out = six || last ? dx : base + q.acc;
                o.acc_in = first ? nullptr : six ? (const float*)dx : (const float*)(base + q.acc);
                o.dloss = last ? (const float*)dloss : nullptr;
            }
            o.labels = p.labels;
            o.index_bytes = p.index_bytes;
            o.vocab = p.vocab;
            add_job(w, o, mgk, mwn, q.cg, q.ksx);
            o.dloss = nullptr;
            o.factor = q.sw > 1 ? nullptr : unit;
            // dw = unit P^T (dloss x / unit): K runs over the tokens
            o.M = (int)nv;
            o.K = (int)p.n;
            o.a_mn = 1;
            o.out_bf16 = !six && q.sw == 1;
            o.out = q.sw > 1 ? (void*)(base + q.pw) : (char*)dw + v0 * p.dim * es;
            o.acc_in = nullptr;
            add_job(w, o, mgm, mxn, q.cg, q.ksw);
        }
        if (i < q.pieces) {
            const size_t v0 = i * q.vp, nv = std::min<size_t>(q.vp, p.vocab - v0);
            const bf16* wp = (const bf16*)p.w + (wip ? v0 * p.dim : 0);
            if (!wip) {
                wp = (bf16*)(base + q.wp[i & 1]);
                pack_add(packs, p, (bf16*)wp, (const char*)p.w + v0 * p.dim * es, nv);
            }
            run_pack(c, p, packs, (int)q.dp);
            if ((rc = make_map(&mwk, wp, p.dim, nv, ldw, q.planes, nv * ldw, BT))) return rc;
            z.N = (int)nv;
            z.col0 = (long long)v0;
            z.g = (bf16*)(base + q.g[i & 1]);
            add_job(w, z, mxk, mwk, q.cg);
        }
        if ((rc = run_work(c, w, q.cg, six))) return rc;
        SumWork s{};
        if (i > 0 && q.sw > 1) {
            const size_t v0 = (i - 1) * q.vp, nv = std::min<size_t>(q.vp, p.vocab - v0);
            s.job[0] = {(const float*)(base + q.pw), (char*)dw + v0 * p.dim * es, nullptr, unit,
                        (long long)nv, p.dim, q.sw};
        }
        if (i == q.pieces && q.sx > 1)
            s.job[1] = {(const float*)(base + q.px), dx, (const float*)dloss, nullptr, p.n, p.dim, q.sx};
        if (s.job[0].slices || s.job[1].slices) run_sum(c, p, s);
    }
    pdl_record_all(c);
    return finish(c);
}

}  // namespace nxv
