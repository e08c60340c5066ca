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
// f64 (the sums along rows longer than a CTA's registers f64 for all); a bf16
// result is rounded once, at its store.  The variance is taken from the centred
// values (two passes over registers, not E[x^2] - mean^2, which cancels for rows
// with a large mean).
//
// Both directions are bound by memory: a row is read once, stays in registers
// and is written once.  What counts is how many bytes are in flight: forward the
// whole row is loaded before anything waits for any of it; backward, where the
// column sums take the registers, one CTA an SM holds some rows while the next ones
// are on their way to L2.  Pairs of f32 values go through the packed two-f32
// instructions.
// Measured: [32768, 4096] bf16 forward 84 us over the same tensors (6.4 TB/s), 90 to 92
// over changing ones (5.9), [16384, 8192] bf16 backward 165 to 169 us (4.8 TB/s; next
// row in registers 216, rows again from L2 187).
//
// Pieces are 16 bytes.  A row that does not start on a 16-byte boundary is worked on in
// the aligned pieces of its memory: x, dy and what is written lie at the same place of
// theirs, so nothing is shifted but gamma and beta, once for rows that start at the
// same place.  A piece at a row's end holds elements of the rows around it, which are
// ignored and, in the result, written by their own rows; rows within 16 bytes of the
// tensor's ends are read element by element, so that nothing outside the tensor is
// touched.  (Pieces of the row's own columns, shifted at every load and store through
// shuffles: [16384, 1001] f32 37 us forward and 68 backward, instead of 27 and 52.)
// The kernels for rows beyond a CTA's registers read two aligned pieces for one.
#include "kernels.h"
#include "ops_common.cuh"

#include <cuda_bf16.h>

#include <algorithm>

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

// V consecutive columns of a row, as they lie in memory.
template <typename T> constexpr int kV = 16 / sizeof(T);
template <typename T>
union Piece {
    uint32_t w[4];
    T e[kV<T>];
    __device__ Piece() {}
};

// w[k] = the four bytes from byte 4 k + o of the 32 bytes a || b, 0 <= o < 16, a
// multiple of T's size.  w may be a or b.
template <typename T>
__device__ __forceinline__ void shift_bytes(uint32_t (&w)[4], const uint32_t (&a)[4],
                                            const uint32_t (&b)[4], unsigned o) {
    uint32_t c[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    if (o & 8) {
#pragma unroll
        for (int k = 0; k < 6; k++) c[k] = c[k + 2];
    }
    if (sizeof(T) < 8 && (o & 4)) {
#pragma unroll
        for (int k = 0; k < 5; k++) c[k] = c[k + 1];
    }
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = sizeof(T) < 4 ? __funnelshift_r(c[k], c[k + 1], (o & 3) * 8) : c[k];
}

__device__ __forceinline__ void load16(uint32_t (&w)[4], const void* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
}

// Two f32 values (or one f64) that one instruction works on.
struct F2 {
    float x, y;
};
__device__ __forceinline__ unsigned long long bits(F2 a) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ F2 from_bits(unsigned long long r) {
    F2 a;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
    return a;
}
__device__ __forceinline__ F2 vfma(F2 a, F2 b, F2 c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return from_bits(r);
}
__device__ __forceinline__ F2 vadd(F2 a, F2 b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return from_bits(r);
}
__device__ __forceinline__ F2 vmul(F2 a, F2 b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return from_bits(r);
}
__device__ __forceinline__ double vfma(double a, double b, double c) { return __fma_rn(a, b, c); }
__device__ __forceinline__ double vadd(double a, double b) { return __dadd_rn(a, b); }
__device__ __forceinline__ double vmul(double a, double b) { return __dmul_rn(a, b); }
__device__ __forceinline__ F2 vset(float v, F2*) { return F2{v, v}; }
__device__ __forceinline__ double vset(double v, double*) { return v; }
__device__ __forceinline__ float vsum(F2 a) { return a.x + a.y; }
__device__ __forceinline__ double vsum(double a) { return a; }

template <typename T> struct Vec { using type = F2; };
template <> struct Vec<double> { using type = double; };
template <typename T> using vec_t = typename Vec<T>::type;
template <typename T> constexpr int kN = sizeof(vec_t<T>) / sizeof(acc_t<T>);  // values of a vec
template <typename T> constexpr int kP = kV<T> / kN<T>;                       // vecs of a piece

__device__ __forceinline__ void unpack(F2 (&v)[4], const Piece<bf16>& p) {
#pragma unroll
    for (int k = 0; k < 4; k++)
        v[k] = F2{__uint_as_float(p.w[k] << 16), __uint_as_float(p.w[k] & 0xffff0000u)};
}
__device__ __forceinline__ void unpack(F2 (&v)[2], const Piece<float>& p) {
#pragma unroll
    for (int k = 0; k < 2; k++) v[k] = F2{p.e[2 * k], p.e[2 * k + 1]};
}
__device__ __forceinline__ void unpack(double (&v)[2], const Piece<double>& p) {
    v[0] = p.e[0], v[1] = p.e[1];
}
__device__ __forceinline__ void pack(Piece<bf16>& p, const F2 (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[k].x, v[k].y);
        p.w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ void pack(Piece<float>& p, const F2 (&v)[2]) {
#pragma unroll
    for (int k = 0; k < 2; k++) p.e[2 * k] = v[k].x, p.e[2 * k + 1] = v[k].y;
}
__device__ __forceinline__ void pack(Piece<double>& p, const double (&v)[2]) {
    p.e[0] = v[0], p.e[1] = v[1];
}
// Makes the compiler unpack p again at its next use instead of keeping the
// wider values in registers.
template <typename T>
__device__ __forceinline__ void keep_packed(Piece<T>& p) {
    asm volatile("" : "+r"(p.w[0]), "+r"(p.w[1]), "+r"(p.w[2]), "+r"(p.w[3]));
}
// v's values outside columns [0, cols) as zeros; c: its first column.
__device__ __forceinline__ void keep_inside(F2& v, int c, unsigned cols) {
    if ((unsigned)c >= cols) v.x = 0.0f;
    if ((unsigned)(c + 1) >= cols) v.y = 0.0f;
}
__device__ __forceinline__ void keep_inside(double& v, int c, unsigned cols) {
    if ((unsigned)c >= cols) v = 0.0;
}

// Less than 16 bytes of the tensor before or behind the row, or no such row.
template <typename T>
__device__ __forceinline__ bool edge_row(size_t row, size_t rows, size_t cols) {
    return row * cols < kV<T> || row >= rows || (rows - 1 - row) * cols < kV<T>;
}

// Piece i of the row of `cols` elements at p, zeros past the row.  edge: edge_row,
// or one that stands alone.  AL: every row starts on
// a 16-byte boundary and is whole pieces long.
template <typename T, bool AL>
__device__ __forceinline__ void row_load(Piece<T>& v, const T* p, unsigned i, unsigned cols, bool edge) {
    constexpr unsigned V = kV<T>;
    if constexpr (AL) {
        if (i * V < cols) load16(v.w, p + (size_t)i * V);
        else v.w[0] = v.w[1] = v.w[2] = v.w[3] = 0;
    } else {
        const unsigned s = (unsigned)((uintptr_t)p & 15);
        if (s != 0 && !edge) {
            const unsigned end = s + cols * (unsigned)sizeof(T);
            const char* base = (const char*)p - s + 16 * (size_t)i;
            uint32_t a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
            if (16 * i < end) load16(a, base);
            if (16 * i + 16 < end) load16(b, base + 16);
            shift_bytes<T>(v.w, a, b, s);
            if (i * V + V > cols) {
#pragma unroll
                for (unsigned e = 0; e < V; e++)
                    if (i * V + e >= cols) v.e[e] = T(0.0f);
            }
        } else if (s == 0 && i * V + V <= cols) {
            load16(v.w, p + (size_t)i * V);
        } else {
#pragma unroll
            for (unsigned e = 0; e < V; e++) v.e[e] = i * V + e < cols ? p[i * V + e] : T(0.0f);
        }
    }
}

// ---- rows in the pieces of their memory
//
// Piece i of a row holds the aligned 16 bytes i of the memory that the row of x lies
// in: columns i V - sh .., of which those outside [0, cols) belong to other rows
// (sh = the elements before the row in its first piece; 0 with AL).

__device__ __forceinline__ bool outside(int c, unsigned cols) { return (unsigned)c >= cols; }

// Some of the piece's columns lie in the row and some do not.
template <typename T, bool AL>
__device__ __forceinline__ bool cut(unsigned i, unsigned sh, unsigned cols) {
    constexpr unsigned V = kV<T>;
    return !AL && ((i == 0 && sh > 0) || (i * V < sh + cols && i * V + V > sh + cols));
}

// apart: element by element (an edge_row; a tensor that does not lie as x does);
// otherwise the columns outside the row are whatever is there, until clear_cut.
template <typename T, bool AL>
__device__ __forceinline__ void piece_load(Piece<T>& v, const T* p, unsigned i, unsigned sh, unsigned cols,
                                           bool apart) {
    constexpr unsigned V = kV<T>;
    if constexpr (AL) {
        row_load<T, true>(v, p, i, cols, false);
    } else if (!apart) {
        v.w[0] = v.w[1] = v.w[2] = v.w[3] = 0;
        if (i * V < sh + cols) load16(v.w, (const char*)p + 16 * (size_t)i - sh * sizeof(T));
    } else {
        const int c = (int)(i * V) - (int)sh;
#pragma unroll
        for (int e = 0; e < (int)V; e++) v.e[e] = outside(c + e, cols) ? T(0.0f) : p[c + e];
    }
}
// The columns outside the row of a piece that is cut as zeros.
template <typename T>
__device__ __forceinline__ void clear_cut(Piece<T>& v, unsigned i, unsigned sh, unsigned cols) {
    const int c = (int)(i * kV<T>) - (int)sh;
#pragma unroll
    for (int e = 0; e < kV<T>; e++)
        if (outside(c + e, cols)) v.e[e] = T(0.0f);
}
template <typename T, bool AL>
__device__ __forceinline__ void piece_store(T* p, const Piece<T>& v, unsigned i, unsigned sh, unsigned cols,
                                            bool apart) {
    constexpr unsigned V = kV<T>;
    if (AL || (!apart && !cut<T, AL>(i, sh, cols))) {
        if (i * V < sh + cols)
            *reinterpret_cast<uint4*>((char*)p + 16 * (size_t)i - sh * sizeof(T)) =
                make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    } else {
        const int c = (int)(i * V) - (int)sh;
#pragma unroll
        for (int e = 0; e < (int)V; e++)
            if (!outside(c + e, cols)) p[c + e] = v.e[e];
    }
}
// The same columns of a vector of weights, what lies outside [0, cols) as zeros.
template <typename T>
__device__ __forceinline__ void weights_load(Piece<T>& v, const T* g, unsigned i, unsigned sh, unsigned cols) {
    constexpr unsigned V = kV<T>;
    // the aligned pieces i - 1 and i of the weights' own memory
    if ((((uintptr_t)g & 15) == 0) && i * V + V <= cols && (i > 0 || sh == 0)) {
        load16(v.w, g + (size_t)i * V);
        if (sh) {
            uint32_t a[4];
            load16(a, g + (size_t)(i - 1) * V);
            shift_bytes<T>(v.w, a, v.w, (V - sh) * (unsigned)sizeof(T));
        }
    } else {
        piece_load<T, false>(v, g, i, sh, cols, true);
    }
}

// Stores piece i of the row at p; lane: the thread's place among the `width`
// (at most 32) lanes of its warp that hold the row's consecutive pieces; live:
// it has a row.  Whole warps.
template <typename T, bool AL>
__device__ __forceinline__ void row_store(T* p, const Piece<T>& v, unsigned i, unsigned cols,
                                          unsigned lane, unsigned width, bool live) {
    constexpr unsigned V = kV<T>;
    if constexpr (AL) {
        if (live && i * V < cols)
            reinterpret_cast<uint4*>(p)[i] = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    } else {
        const unsigned s = (unsigned)((uintptr_t)p & 15), bytes = cols * (unsigned)sizeof(T);
        char* base = (char*)p - s;
        uint32_t prev[4], out[4];
#pragma unroll
        for (int k = 0; k < 4; k++) prev[k] = __shfl_up_sync(0xffffffffu, v.w[k], 1);
        if (!live || i * V >= cols) return;
        if (s == 0) {
            if (16 * i + 16 <= bytes) {
                reinterpret_cast<uint4*>(p)[i] = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
            } else {
#pragma unroll
                for (unsigned e = 0; e < V; e++)
                    if (i * V + e < cols) p[i * V + e] = v.e[e];
            }
            return;
        }
        shift_bytes<T>(out, prev, v.w, 16 - s);
        // aligned piece i (the end of piece i - 1, the start of piece i): whole within the row
        const bool mine = lane > 0 && 16 * i + 16 <= s + bytes;
        const bool next = lane + 1 < width && 16 * i + 32 <= s + bytes;  // piece i + 1's lane will
        if (mine) reinterpret_cast<uint4*>(base)[i] = make_uint4(out[0], out[1], out[2], out[3]);
        if (!mine || !next) {
#pragma unroll
            for (unsigned e = 0; e < V; e++) {
                const bool head = e * sizeof(T) + s < 16;
                if (i * V + e < cols && (head ? !mine : !next)) p[i * V + e] = v.e[e];
            }
        }
    }
}

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename A>
__device__ __forceinline__ A rsqrt_exact(A v) {
    return div_(A(1), sqrt_(v));
}

// Forward: a row in the registers of a group of G = 32, 64, .. threads (blockDim.x),
// blockDim.y rows a CTA.  A thread's 4 or 8 (of the longest rows 16) pieces are loaded
// before anything waits for them.
// AL: more than one row a CTA only with one warp a row, where there is no barrier.
// Otherwise the CTA's rows are 2^lgp apart, so that they start at the same place of
// a piece, and share gamma and beta, shifted to it, in shared memory (2 `room`
// elements): [16384, 1001] f32 27 us (every thread shifting them for itself 41 us).
template <typename T, int NV, bool AL>
__global__ void __launch_bounds__(NV > 8 ? 512 : 1024)
k_norm_fwd(T* y, acc_t<T>* __restrict__ mean, acc_t<T>* __restrict__ rstd, const T* x,
           const T* __restrict__ gamma, const T* __restrict__ beta, unsigned rows, unsigned cols,
           acc_t<T> eps, unsigned lgp, unsigned room) {
    using A = acc_t<T>;
    using W = vec_t<T>;
    constexpr int V = kV<T>, N = kN<T>, NP = kP<T>;
    __shared__ A red[2][32];
    extern __shared__ __align__(16) unsigned char mem[];
    const unsigned t = threadIdx.x, G = blockDim.x, lane = t & 31, warps = G >> 5;
    const unsigned w0 = threadIdx.y * warps;  // the row's first warp
    auto total = [&](A v, int which) {
        v = warp_sum(v);
        if (warps == 1) return v;
        if (lane == 0) red[which][w0 + (t >> 5)] = v;
        __syncthreads();
        return warp_sum(lane < warps ? red[which][w0 + lane] : A(0));
    };
    const unsigned P = 1u << lgp;
    const size_t row = AL ? (size_t)blockIdx.x * blockDim.y + threadIdx.y
                          : (((size_t)(blockIdx.x >> lgp) * blockDim.y + threadIdx.y) << lgp) + (blockIdx.x & (P - 1));
    if (AL && row >= rows) return;  // whole warps: blockDim.y > 1 has no barriers
    const bool live = AL || row < rows;
    const T* xr = x + row * cols;
    Piece<T> p[NV];
    const unsigned sh = AL ? 0 : (unsigned)((uintptr_t)xr & 15) / (unsigned)sizeof(T);
    const bool edge = edge_row<T>(row, rows, cols);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        if (live) piece_load<T, AL>(p[k], xr, t + k * G, sh, cols, edge);
        else p[k].w[0] = p[k].w[1] = p[k].w[2] = p[k].w[3] = 0;
    }
    T* sg = reinterpret_cast<T*>(mem);
    if constexpr (!AL) {
        for (unsigned i = threadIdx.y * G + t; i * V < room; i += G * blockDim.y) {
            Piece<T> g, b;
            weights_load(g, gamma, i, sh, cols);
            weights_load(b, beta, i, sh, cols);
            *reinterpret_cast<uint4*>(sg + (size_t)i * V) = make_uint4(g.w[0], g.w[1], g.w[2], g.w[3]);
            *reinterpret_cast<uint4*>(sg + room + (size_t)i * V) = make_uint4(b.w[0], b.w[1], b.w[2], b.w[3]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (cut<T, AL>(t + k * G, sh, cols)) clear_cut(p[k], t + k * G, sh, cols);
    W s = vset(A(0), (W*)0);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        W v[NP];
        unpack(v, p[k]);
#pragma unroll
        for (int e = 0; e < NP; e++) s = vadd(s, v[e]);  // zeros past the row
    }
    const A m = div_(total(vsum(s), 0), A(cols));
    const W mm = vset(-m, (W*)0);
    s = vset(A(0), (W*)0);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const unsigned i = t + k * G;
        if (i * V < sh + cols) {
            W v[NP];
            keep_packed(p[k]);
            unpack(v, p[k]);
            if (cut<T, AL>(i, sh, cols)) {
#pragma unroll
                for (int e = 0; e < NP; e++) {
                    W c = vadd(v[e], mm);
                    keep_inside(c, (int)(i * V) - (int)sh + e * N, cols);
                    s = vfma(c, c, s);
                }
            } else {
#pragma unroll
                for (int e = 0; e < NP; e++) {
                    const W c = vadd(v[e], mm);
                    s = vfma(c, c, s);
                }
            }
        }
    }
    const A rs = rsqrt_exact(div_(total(vsum(s), 1), A(cols)) + eps);
    if (!live) return;
    if (t == 0) {
        mean[row] = m;
        rstd[row] = rs;
    }
    const W rr = vset(rs, (W*)0);
    const bool y_apart = !AL && (((uintptr_t)y ^ (uintptr_t)x) & 15);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const unsigned i = t + k * G;
        if (i * V < sh + cols) {
            Piece<T> g, b;
            load16(g.w, AL ? gamma + (size_t)i * V : sg + (size_t)i * V);
            load16(b.w, AL ? beta + (size_t)i * V : sg + room + (size_t)i * V);
            W v[NP], gv[NP], bv[NP];
            keep_packed(p[k]);
            unpack(v, p[k]);
            unpack(gv, g);
            unpack(bv, b);
#pragma unroll
            for (int e = 0; e < NP; e++) v[e] = vfma(vmul(vadd(v[e], mm), rr), gv[e], bv[e]);
            pack(p[k], v);
            piece_store<T, AL>(y + row * cols, p[k], i, sh, cols, y_apart);
        }
    }
}

// Rows that 512 threads, or gamma and beta that the shared memory, cannot hold: three
// passes over the row.  A thread adds up to 2^18 values one after the other, so the sums are
// f64 (in f32 the mean of 2^28 values of N(1003, 1) is 2 off, of 2^26 0.16).  Two CTAs an
// SM: 32 registers ([500, 65536] f32 99 us; 58 registers and one CTA 145).
template <typename T>
__global__ void __launch_bounds__(1024, 2)
k_norm_fwd_long(T* y, acc_t<T>* __restrict__ mean, acc_t<T>* __restrict__ rstd, const T* x,
                const T* __restrict__ gamma, const T* __restrict__ beta, unsigned rows,
                unsigned cols, acc_t<T> eps) {
    using A = acc_t<T>;
    __shared__ double red[2][32];
    const unsigned lane = threadIdx.x & 31;
    auto total = [&](double v, int which) {
        v = warp_sum(v);
        if (lane == 0) red[which][threadIdx.x >> 5] = v;
        __syncthreads();
        return warp_sum(red[which][lane]);
    };
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * cols;
        T* yr = y + row * cols;
        double s = 0.0;
        for (unsigned i = threadIdx.x; i < cols; i += 1024) s += (double)to_acc(xr[i]);
        const A m = (A)div_(total(s, 0), (double)cols);
        s = 0.0;
        for (unsigned i = threadIdx.x; i < cols; i += 1024) {
            const double d = (double)(to_acc(xr[i]) - m);
            s = __fma_rn(d, d, s);
        }
        const A rs = rsqrt_exact((A)div_(total(s, 1), (double)cols) + eps);
        if (threadIdx.x == 0) {
            mean[row] = m;
            rstd[row] = rs;
        }
        for (unsigned i = threadIdx.x; i < cols; i += 1024)
            from_acc(yr[i], (to_acc(xr[i]) - m) * rs * to_acc(gamma[i]) + to_acc(beta[i]));
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The value at p in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t peer_address(const void* p, unsigned rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_value(const float* p, unsigned rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_address(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ double peer_value(const double* p, unsigned rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(peer_address(p, rank)) : "memory");
    return v;
}

// Backward: how the rows are dealt out: G threads (a power of two, lg its logarithm)
// take R rows at a time.  Rows r and r + 2^lgp start at the same place of a 16-byte
// piece (lgp = 0 where all do), and a group takes rows of one such class only: a
// thread's pieces then hold the same columns of all of them.  units: the most R
// rows of a class.
struct Deal {
    unsigned rows, cols, G, lg, lgp, units;
};
constexpr int kBwdThreads = 512;

// Brings rows [r0, r0 + n) into L2.
template <typename T>
__device__ __forceinline__ void prefetch_rows(const T* t, size_t r0, unsigned n, unsigned cols) {
    const uintptr_t a = ((uintptr_t)(t + r0 * cols) + 15) & ~(uintptr_t)15;
    const uintptr_t b = (uintptr_t)(t + (r0 + n) * cols) & ~(uintptr_t)15;
    if (b > a)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a), "r"((uint32_t)(b - a)) : "memory");
}

// The sums of K = 2 or 4 values over the G threads of a row, in a fixed order, to
// all of them.  Whole warps reduce by halving: the lanes part the values among
// themselves first, 6 shuffles for 4 values instead of 20.  red: 16 warps' K
// sums, by turns.  The whole CTA.
template <typename A, int K>
__device__ __forceinline__ void group_sum(A (&v)[K], unsigned G, A (*red)[16]) {
    constexpr unsigned FULL = 0xffffffffu;
    if (G < 32) {
        for (unsigned o = G / 2; o > 0; o >>= 1) {
#pragma unroll
            for (int k = 0; k < K; k++) v[k] += __shfl_xor_sync(FULL, v[k], o);
        }
        return;
    }
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    A b;
    constexpr unsigned part = K == 4 ? 8 : 16;  // lanes that end up with one value
    if constexpr (K == 4) {
        const bool h = lane & 16, q = lane & 8;
        const A a0 = (h ? v[2] : v[0]) + __shfl_xor_sync(FULL, h ? v[0] : v[2], 16);
        const A a1 = (h ? v[3] : v[1]) + __shfl_xor_sync(FULL, h ? v[1] : v[3], 16);
        b = (q ? a1 : a0) + __shfl_xor_sync(FULL, q ? a0 : a1, 8);
    } else {
        const bool h = lane & 16;
        b = (h ? v[1] : v[0]) + __shfl_xor_sync(FULL, h ? v[0] : v[1], 16);
        b += __shfl_xor_sync(FULL, b, 8);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) b += __shfl_xor_sync(FULL, b, o);
    if (G > 32) {
        const unsigned nw = G >> 5, w0 = warp & ~(nw - 1), id = lane / part, j = lane % part;
        if (j == 0) red[id][warp] = b;
        __syncthreads();
        b = j < nw ? red[id][w0 + j] : A(0);
        if (part == 8 && nw == 16) b += red[id][w0 + 8 + j];
#pragma unroll
        for (unsigned o = part / 2; o > 0; o >>= 1) b += __shfl_xor_sync(FULL, b, o);
    }
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = __shfl_sync(FULL, b, k * part);
}

// Persistent; a thread holds the same columns of every row that its group takes,
// so it adds up its columns' dy xh and dy in registers.  R rows at a time (bf16:
// 2; 1 and 3: [16384, 8192] 200 and 172 us instead of 165), while the next round's come
// into L2 (of the next two: 167 us).  At the end the groups' column
// sums are added, in order, into row blockIdx.x of the partial sums
// [2][gridDim.x][cols]; or, where the grid is one cluster of up to 8 CTAs (dgamma is
// given), over the CTAs' shared memory into dgamma and dbeta, which saves the fold's
// launch.  With t = x - mean, e = dy rstd:
//   dgamma += e t,  dbeta += dy,  dx = e gamma - rstd c1 - t rstd^2 c2,
// c1 = mean(dy gamma), c2 = mean(dy gamma t) rstd (xh in place of t in both passes:
// [16384, 8192] bf16 179 us instead of 172).  rstd^2 c2 stays finite while the
// variance is a normal number.
template <typename T, int NV, int R, bool AL>
__global__ void __launch_bounds__(kBwdThreads, 1)
k_norm_bwd(T* dx, acc_t<T>* __restrict__ part, const T* dy, const T* x,
           const T* __restrict__ gamma, const acc_t<T>* __restrict__ mean,
           const acc_t<T>* __restrict__ rstd, T* dgamma, T* dbeta,
           const __grid_constant__ Deal d) {
    using A = acc_t<T>;
    using W = vec_t<T>;
    constexpr int V = kV<T>, N = kN<T>, NP = kP<T>;
    __shared__ A red[2][2 * R][16];
    extern __shared__ __align__(16) unsigned char mem[];  // the groups' column sums
    const unsigned tid = threadIdx.x, cols = d.cols, G = d.G;
    const A inv = A(1) / A(cols);
    const unsigned t = tid & (G - 1), q = tid >> d.lg, groups = kBwdThreads >> d.lg;
    // the group's class and its place among the class's groups
    const unsigned P = 1u << d.lgp, all = gridDim.x * groups, id0 = blockIdx.x * groups, id = id0 + q;
    const unsigned cls = id & (P - 1), mates = (all - cls + P - 1) >> d.lgp;
    const unsigned fewest = max(all >> d.lgp, 1u);  // groups of a class
    auto shift_of = [&](unsigned c) -> unsigned {
        return AL ? 0 : (unsigned)((uintptr_t)(x + (size_t)c * cols) & 15) / (unsigned)sizeof(T);
    };
    const unsigned sh = shift_of(cls);
    const bool dy_apart = !AL && (((uintptr_t)dy ^ (uintptr_t)x) & 15);
    const bool dx_apart = !AL && (((uintptr_t)dx ^ (uintptr_t)x) & 15);
    Piece<T> g[NV];
    W ag[NV][NP], ab[NV][NP];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        piece_load<T, AL>(g[k], gamma, t + k * G, sh, cols, true);
#pragma unroll
        for (int e = 0; e < NP; e++) ag[k][e] = ab[k][e] = vset(A(0), (W*)0);
    }
    // the first of the R rows (P apart) of the group's turn `it`
    auto first_row = [&](unsigned it) { return cls + (((size_t)(id >> d.lgp) + (size_t)it * mates) * R << d.lgp); };
    auto prefetch = [&](unsigned it) {
        if (groups >= P) {  // the CTA's rows are consecutive
            const size_t r0 = ((size_t)(id0 >> d.lgp) + (size_t)it * fewest) * R << d.lgp;
            if (tid != 0 || r0 >= d.rows) return;
            const unsigned n = (unsigned)min((size_t)groups * R, d.rows - r0);
            prefetch_rows(x, r0, n, cols);
            prefetch_rows(dy, r0, n, cols);
        } else if (t == 0) {
            for (int r = 0; r < R; r++) {
                const size_t row = first_row(it) + ((size_t)r << d.lgp);
                if (row >= d.rows) return;
                prefetch_rows(x, row, 1, cols);
                prefetch_rows(dy, row, 1, cols);
            }
        }
    };
    for (unsigned it = 0, turn = 0; (size_t)(id0 >> d.lgp) + (size_t)it * fewest < d.units; it++, turn ^= 1) {
        prefetch(it + 1);
        // this group's rows; the last ones may lie past the tensor
        const size_t row0 = first_row(it);
        Piece<T> vx[R][NV], vd[R][NV];
        A m[R], rs[R], sum[2 * R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const size_t row = row0 + ((size_t)r << d.lgp);
            const bool live = row < d.rows, edge = edge_row<T>(row, d.rows, cols);
#pragma unroll
            for (int k = 0; k < NV; k++) {
                if (live) {
                    piece_load<T, AL>(vx[r][k], x + row * cols, t + k * G, sh, cols, edge);
                    piece_load<T, AL>(vd[r][k], dy + row * cols, t + k * G, sh, cols, edge || dy_apart);
                } else {
#pragma unroll
                    for (int w = 0; w < 4; w++) vx[r][k].w[w] = vd[r][k].w[w] = 0;
                }
            }
            m[r] = live ? mean[row] : A(0);
            rs[r] = live ? rstd[row] : A(0);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const W mm = vset(-m[r], (W*)0), rr = vset(rs[r], (W*)0);
            W a0 = vset(A(0), (W*)0), a1 = a0;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                if (cut<T, AL>(t + k * G, sh, cols)) {
                    clear_cut(vx[r][k], t + k * G, sh, cols);
                    clear_cut(vd[r][k], t + k * G, sh, cols);
                }
                keep_packed(g[k]);
                W xv[NP], dv[NP], gv[NP];
                unpack(xv, vx[r][k]);
                unpack(dv, vd[r][k]);
                unpack(gv, g[k]);
#pragma unroll
                for (int e = 0; e < NP; e++) {
                    // dy is zero outside the row
                    const W tt = vadd(xv[e], mm), w = vmul(dv[e], gv[e]);
                    a0 = vadd(a0, w);
                    a1 = vfma(w, tt, a1);
                    ag[k][e] = vfma(vmul(dv[e], rr), tt, ag[k][e]);
                    ab[k][e] = vadd(ab[k][e], dv[e]);
                }
            }
            sum[2 * r] = vsum(a0), sum[2 * r + 1] = vsum(a1);
        }
        group_sum<A, 2 * R>(sum, G, red[turn]);
#pragma unroll
        for (int r = 0; r < R; r++) {
            const size_t row = row0 + ((size_t)r << d.lgp);
            const W mm = vset(-m[r], (W*)0), rr = vset(rs[r], (W*)0);
            const W c1 = vset(-rs[r] * (sum[2 * r] * inv), (W*)0);
            const W c2 = vset(-rs[r] * (rs[r] * (rs[r] * (sum[2 * r + 1] * inv))), (W*)0);
#pragma unroll
            for (int k = 0; k < NV; k++) {
                W xv[NP], dv[NP], gv[NP];
                keep_packed(vx[r][k]);
                keep_packed(vd[r][k]);
                keep_packed(g[k]);
                unpack(xv, vx[r][k]);
                unpack(dv, vd[r][k]);
                unpack(gv, g[k]);
#pragma unroll
                for (int e = 0; e < NP; e++)
                    xv[e] = vfma(vadd(xv[e], mm), c2, vfma(vmul(dv[e], rr), gv[e], c1));
                pack(vx[r][k], xv);
                if (row < d.rows) piece_store<T, AL>(dx + row * cols, vx[r][k], t + k * G, sh, cols, dx_apart);
            }
        }
    }
    const unsigned pad = (NV * V) << d.lg;  // a group's columns
    A* sums = reinterpret_cast<A*>(mem);
    A* folded = sums + (size_t)groups * pad;  // with dgamma
#pragma unroll
    for (int which = 0; which < 2; which++) {
        A* out = part + ((size_t)which * gridDim.x + blockIdx.x) * cols;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int e = 0; e < NP; e++)
                *reinterpret_cast<W*>(&sums[(size_t)q * pad + (t + k * G) * V + e * N]) = which ? ab[k][e] : ag[k][e];
        __syncthreads();
        for (unsigned c = tid; c < cols; c += kBwdThreads) {
            A v = A(0);
            for (unsigned j = 0; j < groups; j++)
                v += sums[(size_t)j * pad + c + shift_of((id0 + j) & (P - 1))];
            if (dgamma) folded[c] = v;
            else out[c] = v;
        }
        if (dgamma) {
            cluster_sync();
            for (unsigned c = blockIdx.x * kBwdThreads + tid; c < cols; c += gridDim.x * kBwdThreads) {
                A v = A(0);
                for (unsigned j = 0; j < gridDim.x; j++) v += peer_value(&folded[c], j);
                from_acc((which ? dbeta : dgamma)[c], v);
            }
            cluster_sync();  // the peers have read this CTA's sums
        }
    }
}

// A row's two sums over the 512 threads of a CTA: this warp's shares.  In f64 from turn to
// turn, as many as 2^15 for the longest rows.
template <typename T, bool AL>
__device__ __forceinline__ void row_sums(double (&sum)[2], const T* px, const T* pd, const T* gamma,
                                         acc_t<T> m, acc_t<T> rs, unsigned cols, bool edge) {
    using A = acc_t<T>;
    using W = vec_t<T>;
    constexpr int V = kV<T>, NP = kP<T>, B = 4;
    const unsigned nv = (cols + V - 1) / V;
    const W mm = vset(-m, (W*)0), rr = vset(rs, (W*)0);
    sum[0] = sum[1] = 0.0;
    for (unsigned i0 = threadIdx.x; i0 < nv; i0 += B * 512) {
        W a0 = vset(A(0), (W*)0), a1 = a0;
        Piece<T> x[B], dy[B];
#pragma unroll
        for (int k = 0; k < B; k++) {
            row_load<T, AL>(x[k], px, i0 + k * 512, cols, edge);
            row_load<T, AL>(dy[k], pd, i0 + k * 512, cols, edge);
        }
#pragma unroll
        for (int k = 0; k < B; k++) {
            Piece<T> g;
            row_load<T, AL>(g, gamma, i0 + k * 512, cols, true);
            W xv[NP], dv[NP], gv[NP];
            unpack(xv, x[k]);
            unpack(dv, dy[k]);
            unpack(gv, g);
#pragma unroll
            for (int e = 0; e < NP; e++) {
                const W w = vmul(dv[e], gv[e]);  // zero past the row
                a0 = vadd(a0, w);
                a1 = vfma(w, vmul(vadd(xv[e], mm), rr), a1);
            }
        }
        sum[0] += (double)vsum(a0), sum[1] += (double)vsum(a1);
    }
    sum[0] = warp_sum(sum[0]), sum[1] = warp_sum(sum[1]);
}

// Rows that the threads of a CTA cannot hold the column sums of (x and dy are read
// twice; blocks of rows that stay in L2 in between measured slower, the launches
// too small: [4096, 12000] f32 221 us instead of 178): the two sums of
// every row first, then a pass in which a CTA takes a strip of 256 pieces of
// columns of the rows 4 blockIdx.y .., + 4 gridDim.y, ...  The f32 sums with 32 registers
// ([4096, 12000] with both kernels 180 us; with 40 registers 196).
template <typename T, bool AL>
__global__ void __launch_bounds__(512, AL && sizeof(T) == 4 ? 4 : 1)
k_norm_bwd_sums(acc_t<T>* __restrict__ sums, const T* dy, const T* x, const T* __restrict__ gamma,
                const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd, unsigned rows,
                unsigned cols) {
    __shared__ double p[2][16];
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        double s[2];
        row_sums<T, AL>(s, x + row * cols, dy + row * cols, gamma, mean[row], rstd[row], cols,
                        edge_row<T>(row, rows, cols));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) p[0][threadIdx.x >> 5] = s[0], p[1][threadIdx.x >> 5] = s[1];
        __syncthreads();
        if (threadIdx.x < 2) {
            double v = 0.0;
            for (int k = 0; k < 16; k++) v += p[threadIdx.x][k];
            sums[2 * row + threadIdx.x] = (acc_t<T>)v;
        }
    }
}

template <typename T, bool AL>
__global__ void __launch_bounds__(256)
k_norm_bwd_strips(T* dx, acc_t<T>* __restrict__ part, const acc_t<T>* __restrict__ sums,
                  const T* dy, const T* x, const T* __restrict__ gamma,
                  const acc_t<T>* __restrict__ mean, const acc_t<T>* __restrict__ rstd,
                  unsigned rows, unsigned cols) {
    using A = acc_t<T>;
    using W = vec_t<T>;
    constexpr int V = kV<T>, NP = kP<T>;
    const A inv = A(1) / A(cols);
    const unsigned i = blockIdx.x * 256 + threadIdx.x;
    Piece<T> g;
    row_load<T, AL>(g, gamma, i, cols, true);
    W gv[NP], ag[NP], ab[NP];
    unpack(gv, g);
#pragma unroll
    for (int e = 0; e < NP; e++) ag[e] = ab[e] = vset(A(0), (W*)0);
    constexpr int R = 4;  // rows whose loads are in flight together
    for (size_t row0 = (size_t)blockIdx.y * R; row0 < rows; row0 += (size_t)gridDim.y * R) {
        Piece<T> px[R], pd[R];
#pragma unroll
        for (int r = 0; r < R; r++) {
            const size_t row = row0 + r;
            if (row >= rows) break;
            const bool edge = edge_row<T>(row, rows, cols);
            row_load<T, AL>(px[r], x + row * cols, i, cols, edge);
            row_load<T, AL>(pd[r], dy + row * cols, i, cols, edge);
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const size_t row = row0 + r;
            if (row >= rows) break;
            const W mm = vset(-mean[row], (W*)0), rr = vset(rstd[row], (W*)0);
            const W c1 = vset(-sums[2 * row] * inv, (W*)0), c2 = vset(-sums[2 * row + 1] * inv, (W*)0);
            W xv[NP], dv[NP];
            unpack(xv, px[r]);
            unpack(dv, pd[r]);
#pragma unroll
            for (int e = 0; e < NP; e++) {
                const W xh = vmul(vadd(xv[e], mm), rr);
                ag[e] = vfma(dv[e], xh, ag[e]);
                ab[e] = vadd(ab[e], dv[e]);
                xv[e] = vmul(rr, vadd(vfma(xh, c2, vmul(dv[e], gv[e])), c1));
            }
            pack(px[r], xv);
            row_store<T, AL>(dx + row * cols, px[r], i, cols, threadIdx.x & 31, 32, true);
        }
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
        const unsigned c = i * V + e;
        if (c < cols) {
            part[(size_t)blockIdx.y * cols + c] = reinterpret_cast<const A*>(ag)[e];
            part[(size_t)(gridDim.y + blockIdx.y) * cols + c] = reinterpret_cast<const A*>(ab)[e];
        }
    }
}

// dgamma_j, dbeta_j: the P partial rows added in a fixed order (32 strided
// sums per column, then a tree); P = 0 gives zeros.  blockIdx.y: which of the two.
template <typename T>
__global__ void __launch_bounds__(1024)
k_norm_fold(T* __restrict__ dgamma, T* __restrict__ dbeta, const acc_t<T>* __restrict__ part,
            unsigned P, unsigned cols) {
    using A = acc_t<T>;
    __shared__ A t[32][33];
    const unsigned col = blockIdx.x * 32 + threadIdx.x;
    const A* p = part + (size_t)blockIdx.y * P * cols;
    A s = A(0);
    if (col < cols) {
#pragma unroll 4
        for (unsigned r = threadIdx.y; r < P; r += 32) s += p[(size_t)r * cols + col];
    }
    t[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    // warp y folds column y of the block
    const A sum = warp_sum(t[threadIdx.x][threadIdx.y]);
    const unsigned c2 = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && c2 < cols) from_acc((blockIdx.y == 0 ? dgamma : dbeta)[c2], sum);
}

template <typename T>
bool all_aligned(unsigned cols, std::initializer_list<const void*> ps) {
    if (cols % kV<T>) return false;
    for (const void* p : ps)
        if ((uintptr_t)p & 15) return false;
    return true;
}

// log2 of the rows after which a row starts at the same place of a 16-byte piece.
template <typename T>
unsigned row_classes(unsigned cols) {
    unsigned lgp = 0;
    while (((size_t)cols << lgp) % kV<T>) lgp++;
    return lgp;
}

// Pieces of gamma and of beta that k_norm_fwd has room for in shared memory.
constexpr size_t kWeightPieces = 7168;
constexpr int kWeightBytes = 2 * kWeightPieces * 16;

template <typename T, bool AL>
int fwd(Ctx& c, T* y, acc_t<T>* mean, acc_t<T>* rstd, const T* x, const T* g, const T* b,
         unsigned rows, unsigned cols, acc_t<T> eps) {
    // a row that starts inside a piece may take one more
    const size_t nv = ((size_t)cols + (AL ? 1 : 2) * (kV<T> - 1)) / kV<T>;
    if (nv > (AL ? 16 * 512 : kWeightPieces)) {
        k_norm_fwd_long<T><<<std::min(rows, (unsigned)c.dev->sm_count * 2), 1024, 0, c.stream>>>(
            y, mean, rstd, x, g, b, rows, cols, eps);
        return OK;
    }
    // Pieces a thread: 8 where the rows come from memory, 4, with more threads a row,
    // where they come from L2 and latency counts ([32768, 4096] bf16 84.0 us with 8, 84.5
    // with 4, 89.2 with 16; [3000, 4096] 12.6, 10.5, 14.5).  Where gamma and beta are shifted
    // into shared memory f32 and f64 gain from 8 sooner ([3000, 2049] f32 15.3 us and 16.5,
    // [500, 4001] 10.3 and 8.4), bf16 later ([16384, 3001] 59.6 and 52.6, [8192, 8001] 72 and 78).
    const size_t mb = ((size_t)rows * cols * sizeof(T)) >> 20;
    unsigned per = (AL ? mb >= 64 : kV<T> == 8 ? nv > 768 : mb >= 16) ? 8 : 4;
    while (nv > per * 512) per *= 2;
    const unsigned tx = (unsigned)((nv + per - 1) / per + 31) / 32 * 32, k = (unsigned)((nv + tx - 1) / tx);
    auto f = k <= 1   ? k_norm_fwd<T, 1, AL>
             : k <= 2 ? k_norm_fwd<T, 2, AL>
             : k <= 4 ? k_norm_fwd<T, 4, AL>
             : k <= 8 ? k_norm_fwd<T, 8, AL>
                      : k_norm_fwd<T, 16, AL>;
    unsigned ty = tx == 32 ? 4 : 1, lgp = 0;
    const unsigned room = AL ? 0 : (unsigned)(nv * kV<T>), bytes = 2 * room * (unsigned)sizeof(T);
    if (!AL) {
        lgp = row_classes<T>(cols);
        // Rows that share gamma and beta: 256 threads (of longer rows 512), as long as two
        // CTAs an SM remain ([16384, 1001] f32 with 32, 128, 256, 512 threads 64, 29, 28, 29 us).
        const unsigned most = tx == 32 ? 256 : 512;
        for (ty = 1; 2 * ty * tx <= most && rows >= (size_t)c.dev->sm_count * 4 * ty; ty *= 2) {}
        // the same for all widths: the attribute is the kernel's, not the call's, and another
        // thread may set it between here and the launch
        NXV_CK(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kWeightBytes));
    }
    const unsigned part = AL ? 1u << 30 : 1u << 27;  // rows of a launch, within the grid's limit
    for (size_t r0 = 0; r0 < rows; r0 += part) {
        const unsigned n = (unsigned)std::min<size_t>(rows - r0, part), P = 1u << lgp;
        f<<<((n + P - 1) / P + ty - 1) / ty * P, dim3(tx, ty), bytes, c.stream>>>(
            y + r0 * cols, mean + r0, rstd + r0, x + r0 * cols, g, b, n, cols, eps, lgp, room);
    }
    return OK;
}

template <typename T>
int fwd_t(Ctx& c, void* y, void* mean, void* rstd, const void* x, const void* g, const void* b,
          unsigned rows, unsigned cols, double eps) {
    using A = acc_t<T>;
    auto f = all_aligned<T>(cols, {y, x, g, b}) ? fwd<T, true> : fwd<T, false>;
    if (int rc = f(c, (T*)y, (A*)mean, (A*)rstd, (const T*)x, (const T*)g, (const T*)b, rows, cols, (A)eps)) return rc;
    count_launch();
    pdl_record_all(c);
    return finish(c);
}

// How the backward pass runs: by rows (strips = 0) or by strips; and the
// partial rows of the weights' gradients that it leaves.
struct BwdShape {
    unsigned strips, grid, parts;
    Deal deal;
};
constexpr unsigned kBwdCtas = 148;  // of a B200; fixed, as the workspace's size must not depend on the device
template <typename T> constexpr int kPer = kV<T> == 8 ? 2 : 4;   // pieces a thread: at most 16 columns' sums
template <typename T> constexpr int kRows = kV<T> == 8 ? 2 : 1;  // rows at a time
template <typename T>
BwdShape bwd_shape_t(unsigned rows, unsigned cols, bool aligned) {
    constexpr unsigned V = kV<T>;
    // a row that starts inside a piece may take one more
    const size_t nv = ((size_t)cols + (aligned ? 1 : 2) * (V - 1)) / V;
    BwdShape q{};
    if (nv > (size_t)kBwdThreads * kPer<T>) {
        q.strips = (unsigned)(((size_t)cols + 256 * V - 1) / (256 * V));
        q.grid = q.parts = std::min((rows + 3) / 4, (kBwdCtas * 4 + q.strips - 1) / q.strips);
        return q;
    }
    Deal& d = q.deal;
    d.rows = rows;
    d.cols = cols;
    for (d.G = 4, d.lg = 2; (size_t)d.G * kPer<T> < nv; d.lg++) d.G *= 2;
    d.lgp = aligned ? 0 : row_classes<T>(cols);
    const size_t P = (size_t)1 << d.lgp, groups = kBwdThreads / d.G, per_round = groups * kRows<T>;
    d.units = (unsigned)(((rows + P - 1) / P + kRows<T> - 1) / kRows<T>);
    // and a group for every class that has a row
    const size_t rounds = std::max((rows + per_round - 1) / per_round, (std::min<size_t>(rows, P) + groups - 1) / groups);
    q.grid = q.parts = (unsigned)std::min<size_t>(rounds, kBwdCtas);
    return q;
}
BwdShape bwd_shape(unsigned rows, unsigned cols, int dt, bool aligned) {
    return dt == F32   ? bwd_shape_t<float>(rows, cols, aligned)
           : dt == F64 ? bwd_shape_t<double>(rows, cols, aligned)
                       : bwd_shape_t<bf16>(rows, cols, aligned);
}
size_t bwd_part_bytes(const BwdShape& q, unsigned cols, int dt) {
    return (size_t)2 * q.parts * cols * (dt == F64 ? 8 : 4);
}

// Few CTAs fold the weights' gradients among themselves.
bool one_cluster(const BwdShape& q) { return q.strips == 0 && q.grid > 0 && q.grid <= 8; }

template <typename T, bool AL>
int bwd(Ctx& c, const BwdShape& q, T* dx, T* dg, T* db, acc_t<T>* part, acc_t<T>* sums, const T* dy,
        const T* x, const T* g, const acc_t<T>* mean, const acc_t<T>* rstd, unsigned rows,
        unsigned cols) {
    if (q.strips) {
        k_norm_bwd_sums<T, AL><<<std::min(rows, (unsigned)c.dev->sm_count * 4), 512, 0, c.stream>>>(
            sums, dy, x, g, mean, rstd, rows, cols);
        k_norm_bwd_strips<T, AL><<<dim3(q.strips, q.grid), 256, 0, c.stream>>>(
            dx, part, sums, dy, x, g, mean, rstd, rows, cols);
        count_launch(2);
        return OK;
    }
    const bool one = ((size_t)cols + (AL ? 1 : 2) * (kV<T> - 1)) / kV<T> <= q.deal.G;
    auto f = one ? k_norm_bwd<T, 1, kRows<T>, AL> : k_norm_bwd<T, kPer<T>, kRows<T>, AL>;
    const bool fold = one_cluster(q);
    const size_t bytes = ((size_t)kBwdThreads * (one ? 1 : kPer<T>) * kV<T> + (fold ? cols : 0)) * sizeof(acc_t<T>);
    NXV_CK(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(q.grid);
    cfg.blockDim = dim3(kBwdThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = fold ? q.grid : 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NXV_CK(cudaLaunchKernelEx(&cfg, f, dx, part, dy, x, g, mean, rstd, fold ? dg : (T*)nullptr, db, q.deal));
    count_launch();
    return OK;
}

template <typename T>
int bwd_t(Ctx& c, int dt, void* dx, void* dg, void* db, void* ws, const void* dy, const void* x,
          const void* g, const void* mean, const void* rstd, unsigned rows, unsigned cols) {
    using A = acc_t<T>;
    const bool aligned = all_aligned<T>(cols, {dx, dy, x, g});
    const BwdShape q = bwd_shape(rows, cols, dt, aligned);
    if (rows > 0) {
        auto f = aligned ? bwd<T, true> : bwd<T, false>;
        const int rc = f(c, q, (T*)dx, (T*)dg, (T*)db, (A*)ws, (A*)((char*)ws + bwd_part_bytes(q, cols, dt)),
                         (const T*)dy, (const T*)x, (const T*)g, (const A*)mean, (const A*)rstd, rows,
                         cols);
        if (rc) return rc;
    }
    if (!one_cluster(q)) {
        k_norm_fold<T><<<dim3((cols + 31) / 32, 2), dim3(32, 32), 0, c.stream>>>(
            (T*)dg, (T*)db, (const A*)ws, q.parts, cols);
        count_launch();
    }
    pdl_record_all(c);
    return finish(c);
}

}  // namespace

// The backward kernel's partial rows of dgamma and dbeta, and for strips two
// sums of every row; for aligned tensors and for others.
size_t norm_grad_workspace(unsigned rows, unsigned cols, int dt) {
    size_t most = 0;
    for (bool aligned : {false, true}) {
        const BwdShape q = bwd_shape(rows, cols, dt, aligned);
        most = std::max(most, bwd_part_bytes(q, cols, dt) + (q.strips ? (size_t)2 * rows * (dt == F64 ? 8 : 4) : 0));
    }
    return most;
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
        return bwd_t<float>(c, dt, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
    if (dt == F64)
        return bwd_t<double>(c, dt, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
    return bwd_t<bf16>(c, dt, dx, dgamma, dbeta, ws, dy, x, gamma, mean, rstd, rows, cols);
}

}  // namespace nxv
