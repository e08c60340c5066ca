// k_norm.cu -- layer norm over the rows of a [rows, cols] matrix, forward and
// backward (f32, f64, bf16).
//
// forward:  mean = (1/c) sum_j x_j,  var = (1/c) sum_j (x_j - mean)^2,
//           rstd = 1 / sqrt(var + eps),
//           y_j = (x_j - mean) rstd gamma_j + beta_j
// backward: xh_j = (x_j - mean) rstd,  g_j = dy_j gamma_j,
//           dx_j = rstd (g_j - (1/c) sum g - xh_j (1/c) sum g xh),
//           dgamma_j = sum_rows dy_j xh_j,  dbeta_j = sum_rows dy_j
//
// Statistics, sums and the arithmetic are f32 for f32 and bf16 and f64 for
// f64; a bf16 result is rounded once, at its store.  The variance is taken
// from the centred values (two passes over registers, not E[x^2] - mean^2,
// which cancels for rows with a large mean).
//
// Both directions are bound by memory: a row is read once, stays in the
// registers of its CTA (or warp) and is written once.  A thread holds NV
// pieces of VEC consecutive elements (16 bytes when every row starts on a
// 16-byte boundary, else single elements); rows longer than the largest CTA
// holds go through a looping variant that reads the row again from L2.
#include "kernels.h"
#include "ops_common.cuh"

#include <cuda_bf16.h>

namespace nxv {

namespace {

using bf16 = __nv_bfloat16;

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };
template <typename T> using acc_t = typename Acc<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_acc(float& d, float v) { d = v; }
__device__ __forceinline__ void from_acc(double& d, double v) { d = v; }
__device__ __forceinline__ void from_acc(bf16& d, float v) { d = __float2bfloat16_rn(v); }

// VEC consecutive elements, as one load or store.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T e[VEC];
};

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sum of v over the threads of one row (blockDim.x of them), in a fixed
// order, to every thread.  red: 2 x 32 values per row of the block, used in
// turn so that one barrier per sum is enough.
template <typename A, int K>
__device__ __forceinline__ void row_sum(A (&v)[K], A* red, int& turn) {
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = warp_sum(v[k]);
    const int nw = blockDim.x >> 5;
    if (nw == 1) return;
    A* buf = red + (turn & 1) * (32 * K);
    turn++;
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) {
#pragma unroll
        for (int k = 0; k < K; k++) buf[k * 32 + w] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = warp_sum(l < nw ? buf[k * 32 + l] : A(0));
}

template <typename A>
__device__ __forceinline__ A rsqrt_exact(A v) {
    return div_(A(1), sqrt_(v));
}

// One row per blockDim.x threads (blockDim.y rows per block; blockDim.y > 1
// only with one warp per row).  NV = 0: the looping variant.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024)
k_norm_fwd(T* y, acc_t<T>* __restrict__ mean, acc_t<T>* __restrict__ rstd,
           const T* x, const T* __restrict__ gamma, const T* __restrict__ beta, unsigned rows,
           unsigned cols, acc_t<T> eps) {
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    __shared__ A red[64];
    int turn = 0;
    const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= rows) return;  // whole warps: blockDim.y > 1 has no barriers
    const P* xr = reinterpret_cast<const P*>(x + row * cols);
    P* yr = reinterpret_cast<P*>(y + row * cols);
    const P* gp = reinterpret_cast<const P*>(gamma);
    const P* bp = reinterpret_cast<const P*>(beta);
    const unsigned nv = cols / VEC;  // exact: VEC > 1 only for cols % VEC == 0
    const A inv = A(1) / A(cols);
    if constexpr (NV > 0) {
        P r[NV];
        A s[1] = {A(0)};
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const unsigned i = threadIdx.x + k * blockDim.x;
            if (i < nv) r[k] = xr[i];
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (threadIdx.x + k * blockDim.x < nv) {
#pragma unroll
                for (int e = 0; e < VEC; e++) s[0] += to_acc(r[k].e[e]);
            }
        }
        row_sum<A, 1>(s, red, turn);
        const A m = s[0] * inv;
        s[0] = A(0);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (threadIdx.x + k * blockDim.x < nv) {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const A d = to_acc(r[k].e[e]) - m;
                    s[0] += d * d;
                }
            }
        }
        row_sum<A, 1>(s, red, turn);
        const A rs = rsqrt_exact(s[0] * inv + eps);
        if (threadIdx.x == 0) {
            mean[row] = m;
            rstd[row] = rs;
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const unsigned i = threadIdx.x + k * blockDim.x;
            if (i < nv) {
                const P g = gp[i], b = bp[i];
                P o;
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    from_acc(o.e[e], (to_acc(r[k].e[e]) - m) * rs * to_acc(g.e[e]) + to_acc(b.e[e]));
                yr[i] = o;
            }
        }
    } else {
        A s[1] = {A(0)};
        for (unsigned i = threadIdx.x; i < nv; i += blockDim.x) {
            const P v = xr[i];
#pragma unroll
            for (int e = 0; e < VEC; e++) s[0] += to_acc(v.e[e]);
        }
        row_sum<A, 1>(s, red, turn);
        const A m = s[0] * inv;
        s[0] = A(0);
        for (unsigned i = threadIdx.x; i < nv; i += blockDim.x) {
            const P v = xr[i];
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const A d = to_acc(v.e[e]) - m;
                s[0] += d * d;
            }
        }
        row_sum<A, 1>(s, red, turn);
        const A rs = rsqrt_exact(s[0] * inv + eps);
        if (threadIdx.x == 0) {
            mean[row] = m;
            rstd[row] = rs;
        }
        for (unsigned i = threadIdx.x; i < nv; i += blockDim.x) {
            const P v = xr[i], g = gp[i], b = bp[i];
            P o;
#pragma unroll
            for (int e = 0; e < VEC; e++)
                from_acc(o.e[e], (to_acc(v.e[e]) - m) * rs * to_acc(g.e[e]) + to_acc(b.e[e]));
            yr[i] = o;
        }
    }
}

// Rows r = blockIdx.x, + gridDim.x, ...: a thread owns the same columns of
// every row, so it adds up its columns' dy xh and dy in registers and writes
// them once, as row blockIdx.x of the partial sums [2][gridDim.x][cols].
// NV = 0: the looping variant, which adds into its partial row in memory.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024)
k_norm_bwd(T* dx, acc_t<T>* __restrict__ part, const T* dy, const T* x,
           const T* __restrict__ gamma, const acc_t<T>* __restrict__ mean,
           const acc_t<T>* __restrict__ rstd, unsigned rows, unsigned cols) {
    using A = acc_t<T>;
    using P = Pack<T, VEC>;
    __shared__ A red[128];
    int turn = 0;
    const unsigned nv = cols / VEC;
    const A inv = A(1) / A(cols);
    const P* gp = reinterpret_cast<const P*>(gamma);
    A* pg = part + (size_t)blockIdx.x * cols;
    A* pb = part + (size_t)(gridDim.x + blockIdx.x) * cols;
    if constexpr (NV > 0) {
        A ag[NV][VEC], ab[NV][VEC];
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) ag[k][e] = ab[k][e] = A(0);
        for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
            const P* xr = reinterpret_cast<const P*>(x + row * cols);
            const P* dr = reinterpret_cast<const P*>(dy + row * cols);
            P* or_ = reinterpret_cast<P*>(dx + row * cols);
            P rx[NV], rd[NV];
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const unsigned i = threadIdx.x + k * blockDim.x;
                if (i < nv) {
                    rx[k] = xr[i];
                    rd[k] = dr[i];
                }
            }
            const A m = mean[row], rs = rstd[row];
            A s[2] = {A(0), A(0)};
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const unsigned i = threadIdx.x + k * blockDim.x;
                if (i < nv) {
                    const P g = gp[i];
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const A d = to_acc(rd[k].e[e]), xh = (to_acc(rx[k].e[e]) - m) * rs;
                        const A w = d * to_acc(g.e[e]);
                        s[0] += w;
                        s[1] += w * xh;
                        ag[k][e] += d * xh;
                        ab[k][e] += d;
                    }
                }
            }
            row_sum<A, 2>(s, red, turn);
            const A c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const unsigned i = threadIdx.x + k * blockDim.x;
                if (i < nv) {
                    const P g = gp[i];
                    P o;
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const A xh = (to_acc(rx[k].e[e]) - m) * rs;
                        from_acc(o.e[e], rs * (to_acc(rd[k].e[e]) * to_acc(g.e[e]) - c1 - xh * c2));
                    }
                    or_[i] = o;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const unsigned i = threadIdx.x + k * blockDim.x;
            if (i < nv) {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    pg[(size_t)i * VEC + e] = ag[k][e];
                    pb[(size_t)i * VEC + e] = ab[k][e];
                }
            }
        }
    } else {
        for (unsigned i = threadIdx.x; i < cols; i += blockDim.x) pg[i] = pb[i] = A(0);
        for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
            const T* xr = x + row * cols;
            const T* dr = dy + row * cols;
            T* or_ = dx + row * cols;
            const A m = mean[row], rs = rstd[row];
            A s[2] = {A(0), A(0)};
            // the thread that adds into column i is the same for every row
            for (unsigned i = threadIdx.x; i < cols; i += blockDim.x) {
                const A d = to_acc(dr[i]), xh = (to_acc(xr[i]) - m) * rs, w = d * to_acc(gamma[i]);
                s[0] += w;
                s[1] += w * xh;
                pg[i] += d * xh;
                pb[i] += d;
            }
            row_sum<A, 2>(s, red, turn);
            const A c1 = s[0] * inv, c2 = s[1] * inv;
            for (unsigned i = threadIdx.x; i < cols; i += blockDim.x) {
                const A xh = (to_acc(xr[i]) - m) * rs;
                from_acc(or_[i], rs * (to_acc(dr[i]) * to_acc(gamma[i]) - c1 - xh * c2));
            }
        }
    }
}

// dgamma_j, dbeta_j: the P partial rows added in a fixed order (8 strided
// sums per column, then a tree); P = 0 gives zeros.  blockIdx.y: which of the two.
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_fold(T* __restrict__ dgamma, T* __restrict__ dbeta, const acc_t<T>* __restrict__ part,
            unsigned P, unsigned cols) {
    using A = acc_t<T>;
    __shared__ A t[8][33];
    const unsigned col = blockIdx.x * 32 + threadIdx.x;
    const A* p = part + (size_t)blockIdx.y * P * cols;
    A s = A(0);
    if (col < cols)
        for (unsigned r = threadIdx.y; r < P; r += 8) s += p[(size_t)r * cols + col];
    t[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && col < cols) {
        A v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = t[k][threadIdx.x];
        const A sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        from_acc((blockIdx.y == 0 ? dgamma : dbeta)[col], sum);
    }
}

bool aligned16(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (((uintptr_t)p) & 15) return false;
    return true;
}

// Threads per row: enough warps that a thread holds at most NVMAX pieces.
unsigned row_threads(size_t pieces, unsigned per_thread, unsigned most) {
    size_t t = (pieces + per_thread - 1) / per_thread;
    t = (t + 31) / 32 * 32;
    return (unsigned)(t > most ? most : t);
}

template <typename T, int VEC>
void fwd(Ctx& c, T* y, acc_t<T>* mean, acc_t<T>* rstd, const T* x, const T* g, const T* b,
         unsigned rows, unsigned cols, double eps) {
    const size_t nv = cols / VEC;
    const auto e = (acc_t<T>)eps;
    const unsigned tx = row_threads(nv, 4, 1024);
    const unsigned ty = tx == 32 ? 4 : 1;
    const dim3 blk(tx, ty), grid((rows + ty - 1) / ty);
    const size_t k = (nv + tx - 1) / tx;
    if (k <= 1) k_norm_fwd<T, VEC, 1><<<grid, blk, 0, c.stream>>>(y, mean, rstd, x, g, b, rows, cols, e);
    else if (k <= 2) k_norm_fwd<T, VEC, 2><<<grid, blk, 0, c.stream>>>(y, mean, rstd, x, g, b, rows, cols, e);
    else if (k <= 4) k_norm_fwd<T, VEC, 4><<<grid, blk, 0, c.stream>>>(y, mean, rstd, x, g, b, rows, cols, e);
    else if (k <= 8) k_norm_fwd<T, VEC, 8><<<grid, blk, 0, c.stream>>>(y, mean, rstd, x, g, b, rows, cols, e);
    else k_norm_fwd<T, VEC, 0><<<grid, blk, 0, c.stream>>>(y, mean, rstd, x, g, b, rows, cols, e);
    count_launch();
}

template <typename T>
int fwd_t(Ctx& c, void* y, void* mean, void* rstd, const void* x, const void* g, const void* b,
          unsigned rows, unsigned cols, double eps) {
    constexpr int V = 16 / sizeof(T);
    using A = acc_t<T>;
    if (cols % V == 0 && aligned16({y, x, g, b}))
        fwd<T, V>(c, (T*)y, (A*)mean, (A*)rstd, (const T*)x, (const T*)g, (const T*)b, rows, cols, eps);
    else
        fwd<T, 1>(c, (T*)y, (A*)mean, (A*)rstd, (const T*)x, (const T*)g, (const T*)b, rows, cols, eps);
    pdl_record_all(c);
    return finish(c);
}

template <typename T, int VEC>
void bwd(Ctx& c, T* dx, acc_t<T>* part, const T* dy, const T* x, const T* g, const acc_t<T>* mean,
         const acc_t<T>* rstd, unsigned rows, unsigned cols, unsigned P) {
    const size_t nv = cols / VEC;
    const unsigned tx = row_threads(nv, 2, 512);
    const size_t k = (nv + tx - 1) / tx;
    if (k <= 1) k_norm_bwd<T, VEC, 1><<<P, tx, 0, c.stream>>>(dx, part, dy, x, g, mean, rstd, rows, cols);
    else if (k <= 2) k_norm_bwd<T, VEC, 2><<<P, tx, 0, c.stream>>>(dx, part, dy, x, g, mean, rstd, rows, cols);
    else if (k <= 4) k_norm_bwd<T, VEC, 4><<<P, tx, 0, c.stream>>>(dx, part, dy, x, g, mean, rstd, rows, cols);
    else k_norm_bwd<T, VEC, 0><<<P, 1024, 0, c.stream>>>(dx, part, dy, x, g, mean, rstd, rows, cols);
    count_launch();
}

template <typename T>
int bwd_t(Ctx& c, void* dx, void* dg, void* db, void* ws, const void* dy, const void* x,
          const void* g, const void* mean, const void* rstd, unsigned rows, unsigned cols) {
    constexpr int V = 16 / sizeof(T);
    using A = acc_t<T>;
    const unsigned P = norm_grad_blocks(rows);
    if (rows > 0) {
        if (cols % V == 0 && aligned16({dx, dy, x, g}))
            bwd<T, V>(c, (T*)dx, (A*)ws, (const T*)dy, (const T*)x, (const T*)g, (const A*)mean,
                      (const A*)rstd, rows, cols, P);
        else
            bwd<T, 1>(c, (T*)dx, (A*)ws, (const T*)dy, (const T*)x, (const T*)g, (const A*)mean,
                      (const A*)rstd, rows, cols, P);
    }
    k_norm_fold<T><<<dim3((cols + 31) / 32, 2), dim3(32, 8), 0, c.stream>>>((T*)dg, (T*)db,
                                                                           (const A*)ws, P, cols);
    count_launch();
    pdl_record_all(c);
    return finish(c);
}

}  // namespace

// Partial rows of the weight gradients: one per CTA of the backward kernel.
unsigned norm_grad_blocks(unsigned rows) { return rows < 296 ? rows : 296; }

size_t norm_grad_workspace(unsigned rows, unsigned cols, int dt) {
    return (size_t)2 * norm_grad_blocks(rows) * cols * (dt == F64 ? 8 : 4);
}

int launch_layer_norm(Ctx& c, int dt, void* y, void* mean, void* rstd, const void* x,
                      const void* gamma, const void* beta, unsigned rows, unsigned cols,
                      double eps) {
    if (rows == 0) return OK;
    if (dt == F32) return fwd_t<float>(c, y, mean, rstd, x, gamma, beta, rows, cols, eps);
    if (dt == F64) return fwd_t<double>(c, y, mean, rstd, x, gamma, beta, rows, cols, eps);
    return fwd_t<bf16>(c, y, mean, rstd, x, gamma, beta, rows, cols, eps);
}

int launch_layer_norm_grad(Ctx& c, int dt, void* dx, void* dgamma, void* dbeta, void* ws,
                           const void* dy, const void* x, const void* gamma, const void* mean,
                           const void* rstd, unsigned rows, unsigned cols) {
    if (dt == F32)
        return bwd_t<float>(c, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
    if (dt == F64)
        return bwd_t<double>(c, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
    return bwd_t<bf16>(c, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
}

}  // namespace nxv
