// The first half of a gated MLP, h = silu(x Wg^T) * (x Wu^T), and its gradients.
//
//   g = x Wg^T, u = x Wu^T, h = g s(g) u             s the logistic function
//   dg = dh u s (1 + g (1 - s)),  du = dh g s,        dx = [dg du] [Wg; Wu],  dW = [dg du]^T x
//
// Three matrix products, of one kind: C (M, N) = sum over k of A (m, k) B (n, k), where an operand's elements are adjacent along k (x and W of
// the forward pass, [dg du] of dx) or along its rows (W of dx, both operands of dW).  With the gate, a tile of C has as many gate columns as
// up columns, the same ones, and a wavefront holds both: g and u meet in registers, and C itself is written only for the backward pass.
#include "ckv_product.h"

#include <algorithm>
#include <initializer_list>

namespace ckv {
namespace {

// ---- any type, stride and size: float32 products on v_mfma_f32_16x16x4 -----------------------------------------------------------------
//
// Bound by that instruction: 2048 x 16384 x 4096 takes 2210 us, 124 TFLOP/s, the matrix pipe busy 78 % of the cycles (the library's product 1820 us);
// rows of an odd number of elements, which no load finds aligned, cost another tenth to quarter (509 x 5462 x 1023 85 us, x 1024 71).

// kTile 128: eight wavefronts of 32 x 64, two on a SIMD: one's loads and stores stand beside the other's products.  64: four of 32 x 32, of
// which several workgroups share a compute unit.
constexpr int kStep = 32;
template <int kTile>
constexpr int kThreads = kTile == 128 ? 512 : 256;

// A tile of kTile rows and 32 steps in LDS.  A product takes four steps, one from each quarter of a wavefront's lanes; which ones does not matter as
// long as both operands' are the same.
//
// Of an operand along k, four steps of a row are a piece of 16 bytes, which a lane reads for four products.  Rows are 16 steps long, the other 16 half
// the banks on; a row's four pieces change places from four rows to the next, so that the sixteen lanes that read at a time, of two quarters and
// eight rows each, meet in no bank.  Of one along its rows, a step's rows lie together, as they are loaded, and a step is 4 banks from the next: the
// quarters' steps, four apart, meet in no bank either.
template <bool kAlongK, int kTile>
struct Stage {
    static constexpr int kHalf = kTile * 16 + 32, kPitch = kTile + 4;
    float v[kAlongK ? 2 * kHalf : kStep * kPitch];
    __device__ static int place(int row, int piece) { return (piece >> 2) * kHalf + row * 16 + (((piece & 3) ^ (0x78 >> ((row >> 1) & 6) & 3)) << 2); }
    __device__ f32x4_t read(int row, int piece) const {
        if constexpr (kAlongK) {
            return *reinterpret_cast<const f32x4_t*>(v + place(row, piece));
        } else {
            f32x4_t r;
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = v[(4 * piece + e) * kPitch + row];
            return r;
        }
    }
};

// A thread's two pieces of a tile: four adjacent elements, along k of a row or along the rows of a step.  Inside the operand they are read at a
// time, from whatever address: rows of an odd number of elements have no better one.
template <typename T, bool kAlongK, int kTile>
struct Pieces {
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
        T v[4];
    };
    static constexpr int kAcross = kAlongK ? kStep / 4 : kTile / 4;   // pieces side by side
    const T* at[2];
    int left[2];   // rows from the first element's on
    float v[2][4];
    __device__ static int row(int i) {
        return kAlongK ? (int)(threadIdx.x / kAcross) + i * (kThreads<kTile> / kAcross) : (int)(threadIdx.x % kAcross) * 4;
    }
    __device__ static int step(int i) {
        return kAlongK ? (int)(threadIdx.x % kAcross) * 4 : (int)(threadIdx.x / kAcross) + i * (kThreads<kTile> / kAcross);
    }
    // r: the row of the operand that piece i begins with, of `rows`
    __device__ void set(int i, const T* base, int64_t stride, int64_t r, int64_t rows, int64_t k) {
        at[i] = base + (kAlongK ? r * stride + k + step(i) : (k + step(i)) * stride + r);
        left[i] = (int)max((int64_t)0, min((int64_t)kTile, rows - r));
    }
    // steps behind `more` and rows behind the last are zeros
    __device__ void load(int64_t stride, int64_t more) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (left[i] >= (kAlongK ? 1 : 4) && (more >= kStep || step(i) + (kAlongK ? 4 : 1) <= more)) {
                const Four x = *reinterpret_cast<const Four*>(at[i]);
#pragma unroll
                for (int e = 0; e < 4; e++) v[i][e] = Elem<T>::to_float(x.v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool there = kAlongK ? left[i] > 0 && step(i) + e < more : left[i] > e && step(i) < more;
                    v[i][e] = there ? Elem<T>::to_float(at[i][e]) : 0.f;
                }
            }
            at[i] += kAlongK ? kStep : kStep * stride;
        }
    }
    __device__ void store(Stage<kAlongK, kTile>& stage) const {
#pragma unroll
        for (int i = 0; i < 2; i++)
            *reinterpret_cast<f32x4_t*>(stage.v + (kAlongK ? stage.place(row(i), step(i) / 4) : step(i) * stage.kPitch + row(i))) =
                f32x4_t{v[i][0], v[i][1], v[i][2], v[i][3]};
    }
};

template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue, int kTile>
__global__ void __launch_bounds__(kThreads<kTile>) product_kernel(ProductParams p) {
    __shared__ __align__(16) Stage<kAlongKA, kTile> as[2];
    __shared__ __align__(16) Stage<kAlongKB, kTile> bs[2];
    int tm, tn, share;
    float* sums = work_of<8>(p, kTile * kTile, tm, tn, share);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1, quarter = lane >> 4, l = lane & 15;
    constexpr bool kGated = kEpilogue == kGate;
    constexpr int kAcross = kTile / 32;   // products of a wavefront side by side; gated, the second half are up columns of the first's gates
    const int64_t inter = p.N / 2;
    const int64_t m0 = (int64_t)tm * kTile, n0 = (int64_t)tn * (kGated ? kTile / 2 : kTile);
    const int64_t k0 = share * p.k_share, k1 = sums ? min(p.K, k0 + p.k_share) : p.K;
    Pieces<T, kAlongKA, kTile> pa;
    Pieces<T, kAlongKB, kTile> pb;
    const T* a = (const T*)p.a.p;
    const T* b = (const T*)p.b.p;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        pa.set(i, a, p.a.stride, m0 + pa.row(i), p.M, k0);
        // gated: the first half of the rows of B's tile are gate rows, the others up rows
        const int row = pb.row(i), up = kGated && row >= kTile / 2;
        pb.set(i, b + (up ? inter * p.b.stride : 0), p.b.stride, n0 + row - (up ? kTile / 2 : 0), kGated ? inter : p.N, k0);
    }
    auto load = [&](int64_t k) {
        pa.load(p.a.stride, k1 - k);
        pb.load(p.b.stride, k1 - k);
    };
    auto column = [&](int j) {   // of the tile's, the first of a product
        return kGated ? (j / (kAcross / 2)) * (kTile / 2) + wn * (kTile / 4) + j % (kAcross / 2) * 16 : wn * (kTile / 2) + j * 16;
    };
    const bool there = m0 + wm * 32 < p.M;   // of a few rows most of the products would be of none: 64 x 5632 x 1024, 33 -> 25 us
    f32x4_t acc[2][kAcross] = {};
    load(k0);
    pa.store(as[0]);
    pb.store(bs[0]);
    __syncthreads();
    int at = 0;
    for (int64_t k = k0; k < k1; k += kStep) {
        const bool more = k + kStep < k1;
        if (more) load(k + kStep);
        if (there)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            f32x4_t av[2], bv[kAcross];
#pragma unroll
            for (int i = 0; i < 2; i++) av[i] = as[at].read(wm * 32 + i * 16 + l, h * 4 + quarter);
#pragma unroll
            for (int j = 0; j < kAcross; j++) bv[j] = bs[at].read(column(j) + l, h * 4 + quarter);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int j = 0; j < kAcross; j++)
#pragma unroll
                    for (int i = 0; i < 2; i++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[i][e], bv[j][e], acc[i][j], 0, 0, 0);
        }
        if (more) {
            pa.store(as[at ^ 1]);
            pb.store(bs[at ^ 1]);
        }
        __syncthreads();
        at ^= 1;
    }
    // element r of a sum: row 4 quarter + r, column l
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = wm * 32 + i * 16 + 4 * quarter + r;
            const int64_t m = m0 + row;
            if (sums) {
#pragma unroll
                for (int j = 0; j < kAcross; j++) sums[row * kTile + column(j) + l] = acc[i][j][r];
                continue;
            }
            if (m >= p.M) continue;
            if constexpr (kGated) {
#pragma unroll
                for (int j = 0; j < kAcross / 2; j++) {
                    const int64_t n = n0 + column(j) + l;
                    if (n >= inter) continue;
                    const float g = acc[i][j][r], u = acc[i][j + kAcross / 2][r];
                    ((T*)p.out)[m * inter + n] = Elem<T>::from_float(gate_product(g, u));
                    if (p.both) {
                        float* to = p.both + m * p.N + n;
                        to[0] = g;
                        to[inter] = u;
                    }
                }
            } else {
                const float power = power_of<T, kAlongKA>(p, m);
#pragma unroll
                for (int j = 0; j < kAcross; j++) {
                    const int64_t n = n0 + column(j) + l;
                    if (n < p.N) ((T*)p.out)[m * p.N + n] = Elem<T>::from_float(times_power<T>(acc[i][j][r], power));
                }
            }
        }
}

// Sums of the shares of a tile, in their order, and what the product's own epilogue does.  A workgroup has some rows of a tile, a thread four
// columns.
template <typename T, Epilogue kEpilogue, bool kAlongKA>
__global__ void __launch_bounds__(256) merge_kernel(ProductParams p, int tile_m, int tile_n, int high, int rows) {
    constexpr bool kGated = kEpilogue == kGate;
    const int tile = p.whole_tiles + blockIdx.x;
    int tm, tn;
    if (high == 8) place_of<8>(p, tile, tm, tn);
    else place_of<4>(p, tile, tm, tn);
    const int width = kGated ? tile_n / 2 : tile_n;
    const int64_t cols = kGated ? p.N / 2 : p.N, n0 = (int64_t)tn * width, m0 = (int64_t)tm * tile_m, share = (int64_t)tile_m * tile_n;
    const float* from = p.partial + blockIdx.x * p.shares * share;
    const int per_row = width / 4;
    for (int i = threadIdx.x; i < rows * per_row; i += 256) {
        const int row = blockIdx.y * rows + i / per_row, col = i % per_row * 4;
        const int64_t m = m0 + row, n = n0 + col;
        if (m >= p.M || n >= cols) continue;
        const float* at = from + (int64_t)row * tile_n + col;
        const float power = kGated ? 1.f : power_of<T, kAlongKA>(p, m);
        float g[4] = {}, u[4] = {};
        for (int s = 0; s < p.shares; s++) {
            const float4 a = *reinterpret_cast<const float4*>(at + s * share);
            g[0] += a.x; g[1] += a.y; g[2] += a.z; g[3] += a.w;
            if constexpr (kGated) {
                const float4 b = *reinterpret_cast<const float4*>(at + s * share + width);
                u[0] += b.x; u[1] += b.y; u[2] += b.z; u[3] += b.w;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (n + e >= cols) break;
            if constexpr (kGated) {
                ((T*)p.out)[m * cols + n + e] = Elem<T>::from_float(gate_product(g[e], u[e]));
                if (p.both) {
                    float* to = p.both + m * p.N + n + e;
                    to[0] = g[e];
                    to[cols] = u[e];
                }
            } else {
                ((T*)p.out)[m * cols + n + e] = Elem<T>::from_float(times_power<T>(g[e], power));
            }
        }
    }
}

// ---- gradients of the projections ------------------------------------------------------------------------------------------------------

// dg and du are rounded to the tensor type, that of the operands of the two products behind: off by up to 2^-8 of each (2^-11 of float16), as
// the products' own results are by their rounding.  The projections they are made from are float32.  Bound by memory: 10 bytes read and 4 written an element
// of 16 bits, 2048 x 18944 98 us, 5.5 TB/s.
__device__ inline void gate_gradients(float g, float u, float d, float& dg, float& du) {
    const float s = 1.f / (1.f + expf(-g));
    dg = d * u * s * (1.f + g * (1.f - s));
    du = d * g * s;
}

template <typename T, int kPer>
__global__ void __launch_bounds__(256) gate_gradient_kernel(const float* gate_up, const T* dout, T* grad, int64_t rows, int64_t inter) {
    struct alignas(sizeof(T) * kPer) Piece {
        T v[kPer];
    };
    struct alignas(kPer > 1 ? 16 : 4) Wide {
        float v[kPer];
    };
    const int64_t pieces = inter / kPer, all = rows * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        int64_t c;
        const int64_t row = div_index(i, pieces, c);
        const float* from = gate_up + row * 2 * inter + c * kPer;
        const Wide gate = *reinterpret_cast<const Wide*>(from), up = *reinterpret_cast<const Wide*>(from + inter);
        const Piece dh = *reinterpret_cast<const Piece*>(dout + row * inter + c * kPer);
        Piece dg, du;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            float a, b;
            gate_gradients(gate.v[e], up.v[e], Elem<T>::to_float(dh.v[e]), a, b);
            dg.v[e] = Elem<T>::from_float(a);
            du.v[e] = Elem<T>::from_float(b);
        }
        T* to = grad + row * 2 * inter + c * kPer;
        *reinterpret_cast<Piece*>(to) = dg;
        *reinterpret_cast<Piece*>(to + inter) = du;
    }
}

template <typename T>
int gate_gradient(const float* gate_up, const void* dout, void* grad, int64_t rows, int64_t inter, hipStream_t stream) {
    constexpr int kPer = 16 / (int)sizeof(T);
    const bool pieces = inter % kPer == 0 &&
                        ((reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    const int64_t all = rows * inter / (pieces ? kPer : 1);
    const unsigned blocks = (unsigned)std::min<int64_t>((all + 255) / 256, 256 * 16);
    if (pieces) hipLaunchKernelGGL((gate_gradient_kernel<T, kPer>), dim3(blocks), dim3(256), 0, stream, gate_up, (const T*)dout, (T*)grad, rows, inter);
    else hipLaunchKernelGGL((gate_gradient_kernel<T, 1>), dim3(blocks), dim3(256), 0, stream, gate_up, (const T*)dout, (T*)grad, rows, inter);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

// float16 ends at 65504 and thins out below 2^-14, where dg and du, products of three numbers, need not stop: a dh of a scaled loss that is well inside the
// type makes a dg that is not, and so does a small one at the other end.  So a row of [dg du] is kept as numbers below 2^15 times a power of two of its own,
// 2^e, which dx's row is multiplied by in float32 (exact, until the row is rounded).  For dW, whose sums run over rows, row m of x takes 2^(e_m - T) along,
// T the largest of e_m and the exponent of x's row, so that no row is above 2^15 and the largest product of two rows is at the top of the range:
//   dx_m = 2^(e_m) ([dg du]_m 2^(-e_m)) W,   dW = 2^T sum over m of ([dg du]_m 2^(-e_m)) (x_m 2^(e_m - T)).
// Below 2^-28 of its row's largest an element of [dg du] loses digits, and one of x below 2^-28 of what its row would have at the top; it is then off by up to
// 2^-39 of those.  bfloat16 has float32's range and needs none of it.

constexpr int kNoExponent = -1000;   // of a row of zeros

// 2^e of a row whose largest number is m: m 2^-e lies in [2^14, 2^15)
__device__ inline int exponent_above(float m) { return m > 0.f ? __builtin_amdgcn_frexp_expf(m) - 15 : kNoExponent; }
__device__ inline float larger_finite(float m, float v) {
    v = fabsf(v);
    return v < __builtin_huge_valf() ? fmaxf(m, v) : m;   // infinities and NaN stay what they are at any scale
}

// A workgroup a row, or for short rows 2^lanes_log of a wavefront's lanes: the row's gradients stay in registers (kHeld pieces a thread; what is behind is worked out twice) until its largest is known.
// exponents: e of every row, then e and the exponent of x's row together.  2048 x 18944 117 us, 4.7 TB/s: a workgroup's loads and stores take turns,
// which is why it is 16 wavefronts with three pieces a thread (of 8 with five or four: 136 and 125 us).  10^6 rows of 128: 340 us (the kernel
// of the other types, which does not look at rows, 325); 870 by a wavefront a row.
constexpr int kRowThreads = 1024;
template <int kPer, int kHeld, bool kShort>
__global__ void __launch_bounds__(kRowThreads, 4) gate_gradient_rows_kernel(const float* gate_up, const __half* dout, __half* grad, const __half* x, int64_t x_stride, int* exponents,
                                                                         int64_t rows, int64_t inter, int64_t k, int lanes_log) {
    struct alignas(sizeof(__half) * kPer) Piece {
        __half v[kPer];
    };
    struct alignas(kPer > 1 ? 16 : 4) Wide {
        float v[kPer];
    };
    __shared__ float tops[2][kRowThreads / 64];
    const int64_t pieces = inter / kPer;
    const int many = kShort ? 1 << lanes_log : (int)blockDim.x, me = threadIdx.x & (kShort ? many - 1 : ~0);   // threads of a row
    const int here = kShort ? (int)blockDim.x >> lanes_log : 1;   // rows of a workgroup
    const int64_t first = (int64_t)blockIdx.x * here + (kShort ? threadIdx.x >> lanes_log : 0);
    for (int64_t row = first; row < rows; row += (int64_t)gridDim.x * here) {   // the lanes of a row go together
        const float* from = gate_up + row * 2 * inter;
        const __half* dh = dout + row * inter;
        __half* to = grad + row * 2 * inter;
        auto gradients = [&](int64_t c, float (&dg)[kPer], float (&du)[kPer]) {
            const Wide gate = *reinterpret_cast<const Wide*>(from + c * kPer), up = *reinterpret_cast<const Wide*>(from + inter + c * kPer);
            const Piece d = *reinterpret_cast<const Piece*>(dh + c * kPer);
#pragma unroll
            for (int e = 0; e < kPer; e++) gate_gradients(gate.v[e], up.v[e], __half2float(d.v[e]), dg[e], du[e]);
        };
        float dg[kHeld][kPer], du[kHeld][kPer], most = 0.f, most_x = 0.f;
        auto look = [&](const float (&a)[kPer], const float (&b)[kPer]) {
#pragma unroll
            for (int e = 0; e < kPer; e++) most = larger_finite(larger_finite(most, a[e]), b[e]);
        };
#pragma unroll
        for (int h = 0; h < kHeld; h++) {
            const int64_t c = me + h * (int64_t)many;
            if (c < pieces) {
                gradients(c, dg[h], du[h]);
                look(dg[h], du[h]);
            }
        }
        for (int64_t c = me + kHeld * (int64_t)many; c < pieces; c += many) {
            float a[kPer], b[kPer];
            gradients(c, a, b);
            look(a, b);
        }
        for (int64_t i = me; i < k; i += many) most_x = larger_finite(most_x, __half2float(x[row * x_stride + i]));
        for (int o = (kShort ? many : CKV_WAVE) >> 1; o > 0; o >>= 1) {
            most = fmaxf(most, __shfl_xor(most, o));
            most_x = fmaxf(most_x, __shfl_xor(most_x, o));
        }
        if constexpr (!kShort) {
            if ((threadIdx.x & 63) == 0) {
                tops[0][threadIdx.x >> 6] = most;
                tops[1][threadIdx.x >> 6] = most_x;
            }
            __syncthreads();
            for (int w = 0; w < (int)blockDim.x >> 6; w++) {
                most = fmaxf(most, tops[0][w]);
                most_x = fmaxf(most_x, tops[1][w]);
            }
        }
        const int e = exponent_above(most);
        if (me == 0) {
            exponents[row] = e;
            exponents[rows + row] = e + exponent_above(most_x);
        }
        auto store = [&](int64_t c, const float (&a)[kPer], const float (&b)[kPer]) {
            Piece g, u;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                g.v[i] = __float2half(__builtin_amdgcn_ldexpf(a[i], -e));
                u.v[i] = __float2half(__builtin_amdgcn_ldexpf(b[i], -e));
            }
            *reinterpret_cast<Piece*>(to + c * kPer) = g;
            *reinterpret_cast<Piece*>(to + inter + c * kPer) = u;
        };
#pragma unroll
        for (int h = 0; h < kHeld; h++) {
            const int64_t c = me + h * (int64_t)many;
            if (c < pieces) store(c, dg[h], du[h]);
        }
        for (int64_t c = me + kHeld * (int64_t)many; c < pieces; c += many) {
            float a[kPer], b[kPer];
            gradients(c, a, b);
            store(c, a, b);
        }
        if constexpr (!kShort) __syncthreads();   // the next row's largest come where this one's are
    }
}

// Rows of x times 2^(e_m - T), contiguous, and T behind the exponents.  Every workgroup looks for T by itself, so there are few of them.
// 2048 x 3584 8 us, 10^6 x 64 113.
template <int kPer>
__global__ void __launch_bounds__(1024) scale_rows_kernel(const __half* x, int64_t x_stride, __half* out, int* exponents, int64_t rows, int64_t k) {
    struct alignas(sizeof(__half) * kPer) Piece {
        __half v[kPer];
    };
    __shared__ int tops[16];
    int top = 2 * kNoExponent;
    for (int64_t i = threadIdx.x; i < rows; i += 8 * 1024)
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, exponents[rows + min(i + j * 1024, rows - 1)]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < 16; w++) top = max(top, tops[w]);
    if (blockIdx.x == 0 && threadIdx.x == 0) exponents[2 * rows] = top;
    const int64_t pieces = k / kPer, all = rows * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 1024) {
        int64_t c;
        const int64_t row = div_index(i, pieces, c);
        const int by = exponents[row] - top;
        Piece v = *reinterpret_cast<const Piece*>(x + row * x_stride + c * kPer);
#pragma unroll
        for (int e = 0; e < kPer; e++) v.v[e] = __float2half(__builtin_amdgcn_ldexpf(__half2float(v.v[e]), by));
        *reinterpret_cast<Piece*>(out + i * kPer) = v;
    }
}

// Both, for a product of every row and one of all rows.
int gate_gradient_rows(const float* gate_up, const void* dout, void* grad, const void* x, int64_t x_stride, void* scaled_x, int* exponents, int64_t rows,
                       int64_t inter, int64_t k, hipStream_t stream) {
    auto aligned = [](std::initializer_list<const void*> all) {
        uintptr_t bits = 0;
        for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
        return (bits & 15) == 0;
    };
    const bool pieces = inter % 8 == 0 && aligned({gate_up, dout, grad});
    const int64_t many = pieces ? inter / 8 : inter;
    const bool short_rows = many <= 3 * CKV_WAVE;   // what a wavefront holds of a row
    int lanes_log = 0;
    while (lanes_log < 6 && (1 << lanes_log) < many) lanes_log++;
    const unsigned threads = short_rows ? 256 : (unsigned)std::min<int64_t>(kRowThreads, align_up(many, CKV_WAVE));
    const int64_t here = short_rows ? 256 >> lanes_log : 1, groups = std::min<int64_t>((rows + here - 1) / here, 1 << 22);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(threads), 0, stream, gate_up, (const __half*)dout, (__half*)grad, (const __half*)x, x_stride, exponents, rows, inter,
                           k, lanes_log);
    };
    if (pieces && many <= CKV_WAVE) launch(gate_gradient_rows_kernel<8, 1, true>);
    else if (pieces && short_rows) launch(gate_gradient_rows_kernel<8, 3, true>);
    else if (pieces) launch(gate_gradient_rows_kernel<8, 3, false>);
    else if (short_rows) launch(gate_gradient_rows_kernel<1, 3, true>);
    else launch(gate_gradient_rows_kernel<1, 16, false>);
    CKV_HIP_TRY(hipGetLastError());
    if (!scaled_x) return CKV_OK;
    const dim3 grid((unsigned)std::min<int64_t>((rows * k + 8191) / 8192, 256));
    if (k % 8 == 0 && x_stride % 8 == 0 && aligned({x, scaled_x}))
        hipLaunchKernelGGL((scale_rows_kernel<8>), grid, dim3(1024), 0, stream, (const __half*)x, x_stride, (__half*)scaled_x, exponents, rows, k);
    else hipLaunchKernelGGL((scale_rows_kernel<1>), grid, dim3(1024), 0, stream, (const __half*)x, x_stride, (__half*)scaled_x, exponents, rows, k);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

// ---- which kernel, how many shares -----------------------------------------------------------------------------------------------------

// The kernels of 16-bit tiles take operands of whole pieces of 16 bytes: all but odd sizes, strides and addresses.
template <typename T>
bool fits_tiles(const ProductParams& p, bool along_a, bool along_b, bool gated) {
    if (sizeof(T) != 2) return false;
    auto whole = [&](const Operand& o, bool along, int64_t rows) {
        return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.stride % 8 == 0 && (along ? p.K : rows) % 8 == 0 && o.stride < (1 << 21);   // a tile of rows within 31 bits
    };
    return whole(p.a, along_a, p.M) && whole(p.b, along_b, p.N) && (gated ? p.N / 2 : p.N) % 8 == 0 &&
           ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.both)) & 15) == 0;
}

// Tiles of float32 products and the shares of their steps, by the time they are estimated to take: of the compute unit that has the most of them,
// 32 steps of r tiles at a time 0.4 + 1.95 r us of 128 x 128, two at a time, and 1.1 + 0.35 r of 64 x 64, four at a time (one has the
// unit wait for its loads); and of adding shares up 3 us, 0.25 a share and 2.5 MB/us.  509 x 5462 x 1023 in tiles of 64 and 128: 79 and 87 us;
// 2048 x 16384 x 4096: 2531 and 2209; 509 x 1023 x 5462 by 16 shares: 87 and 79, by one: 274 and 528.
TilePlan plan_float(int64_t M, int64_t N, int64_t K, bool gated, int cus) {
    TilePlan best;
    double least = 0;
    for (int tile : {128, 64}) {
        const int64_t at_a_time = tile == 128 ? 2 : 4;
        auto time_of = [&](int64_t r) { return r == 0 ? 0. : tile == 128 ? 0.4 + 1.95 * r : 1.1 + 0.35 * r; };
        TilePlan r;
        r.tile_m = r.tile_n = tile;
        r.deep = 1;
        r.tiles_m = (int)((M + tile - 1) / tile);
        r.tiles_n = (int)tiles_across(N, tile, gated);
        const int64_t tiles = (int64_t)r.tiles_m * r.tiles_n;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(K / 128, at_a_time * cus / tiles + 1));
        for (int64_t shares = 1; shares <= most; shares++) {
            r.k_share = ((K + shares - 1) / shares + kStep - 1) / kStep * kStep;
            r.shares = (int)((K + r.k_share - 1) / r.k_share);
            r.whole_tiles = r.shares > 1 ? 0 : (int)std::min<int64_t>(tiles, 0x7fffffff);
            const int64_t each = (tiles * r.shares + cus - 1) / cus;
            const double time = (r.k_share / kStep) * ((each / at_a_time) * time_of(at_a_time) + time_of(each % at_a_time)) + (r.shares > 1 ? 3 + 0.25 * r.shares + r.bytes() / 2.5e6 : 0);
            if (least == 0 || time < least) {
                least = time;
                best = r;
            }
        }
    }
    return best;
}

// Scratch of a product, whichever kernel takes it.
int64_t product_bytes(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus) {
    return std::max(plan_tiles(M, N, K, a_along_k, gated, cus).bytes(), plan_float(M, N, K, gated, cus).bytes());
}

template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int run_product(ProductParams& p, const DeviceInfo& di, void* workspace, int64_t bytes, hipStream_t stream) {
    constexpr bool kGated = kEpilogue == kGate;
    const bool tiles = fits_tiles<T>(p, kAlongKA, kAlongKB, kGated);
    const TilePlan plan = tiles ? plan_tiles(p.M, p.N, p.K, kAlongKA, kGated, di.cus)
                                : plan_float(p.M, p.N, p.K, kGated, di.cus);
    if (plan.bytes() && (!workspace || plan.bytes() > bytes || reinterpret_cast<uintptr_t>(workspace) & 15)) return CKV_ERR_WORKSPACE;
    if ((int64_t)plan.tiles_m * plan.tiles_n > 0x3fffffff || plan.blocks() > 0x7fffffff) return CKV_ERR_UNSUPPORTED;
    plan.fill(p);
    p.partial = (float*)workspace;
    if (tiles) {
        if constexpr (sizeof(T) == 2)
            if (int rc = run_tiles<T>(p, plan, kAlongKA, kEpilogue, stream)) return rc;
    } else {
        if (plan.tile_m == 128)
            hipLaunchKernelGGL((product_kernel<T, kAlongKA, kAlongKB, kEpilogue, 128>), dim3((unsigned)plan.blocks()), dim3(kThreads<128>), 0, stream, p);
        else hipLaunchKernelGGL((product_kernel<T, kAlongKA, kAlongKB, kEpilogue, 64>), dim3((unsigned)plan.blocks()), dim3(kThreads<64>), 0, stream, p);
        CKV_HIP_TRY(hipGetLastError());
    }
    if (plan.shares > 1) {
        constexpr int kRows = 8;
        hipLaunchKernelGGL((merge_kernel<T, kEpilogue, kAlongKA>), dim3(plan.tiles_m * plan.tiles_n - plan.whole_tiles, plan.tile_m / kRows), dim3(256), 0, stream, p, plan.tile_m,
                           plan.tile_n, tiles ? 4 : 8, kRows);
        CKV_HIP_TRY(hipGetLastError());
    }
    return CKV_OK;
}

constexpr int64_t kFewRows = 16, kFewBytes = 118 << 10;

int check_sizes(int64_t rows, int64_t inter, int64_t k, int64_t x_stride, int32_t dtype) {
    if (dtype != CKV_F32 && dtype != CKV_F16 && dtype != CKV_BF16) return CKV_ERR_DTYPE;
    if (rows < 0 || inter <= 0 || k <= 0 || x_stride < k) return CKV_ERR_SHAPE;
    if (rows > 0x7fffffff || inter > 0x3fffffff || k > 0x7fffffff) return CKV_ERR_UNSUPPORTED;
    return CKV_OK;
}

template <typename T>
int run_forward(const void* x, const void* w, void* out, float* gate_up, int64_t rows, int64_t inter, int64_t k, int64_t x_stride, void* workspace,
                int64_t bytes, const DeviceInfo& di, hipStream_t stream) {
    // A few rows wait for the weights, and the kernel of a decoding step's products streams them through LDS beside the rows (28672 x 4096, a
    // row: 39.3 us, tiles 52; twelve rows 43 and 53; sixteen, whose rows leave no room for the streams, 59 and 49; sixteen of 3584: 47 and 61).
    if (sizeof(T) == 2 && rows <= kFewRows && rows * (2 * k + 16) <= kFewBytes && !gate_up && inter % 8 == 0 && k % 64 == 0 && (rows == 1 || x_stride % 8 == 0) &&
        ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
        const int rc = ckv_linear_rows(x, w, nullptr, nullptr, nullptr, 0.f, out, rows, 2 * inter, k, rows == 1 ? k : x_stride, 2, 1, 1, Elem<T>::code, stream);
        if (rc != CKV_ERR_UNSUPPORTED) return rc;   // rows too long for LDS
    }
    ProductParams p = {};
    p.a = Operand{x, x_stride};
    p.b = Operand{w, k};
    p.out = out;
    p.both = gate_up;
    p.M = rows;
    p.N = 2 * inter;
    p.K = k;
    return run_product<T, true, true, kGate>(p, di, workspace, bytes, stream);
}

// Scratch of a backward pass in front of its products': [dg du], and in float16 the exponents of its rows and x by them.
struct Scratch {
    int64_t exponents, x, products;   // where they begin
    Scratch(int64_t rows, int64_t inter, int64_t k, int32_t dtype) {
        exponents = align_up(rows * 2 * inter * elem_bytes(dtype), 256);
        x = exponents + (dtype == CKV_F16 ? align_up((2 * rows + 1) * (int64_t)sizeof(int), 256) : 0);
        products = x + (dtype == CKV_F16 ? align_up(rows * k * 2, 256) : 0);
    }
};

template <typename T>
int run_backward(const void* x, const void* w, const float* gate_up, const void* dout, void* dx, void* dw, int64_t rows, int64_t inter, int64_t k,
                 int64_t x_stride, char* workspace, int64_t bytes, const DeviceInfo& di, hipStream_t stream) {
    const Scratch at(rows, inter, k, Elem<T>::code);
    void* grad = workspace;
    int* exponents = nullptr;
    if constexpr (std::is_same<T, __half>::value) {
        exponents = (int*)(workspace + at.exponents);
        if (int rc = gate_gradient_rows(gate_up, dout, grad, x, x_stride, dw ? workspace + at.x : nullptr, exponents, rows, inter, k, stream)) return rc;
        x = workspace + at.x;
        x_stride = k;
    } else {
        if (int rc = gate_gradient<T>(gate_up, dout, grad, rows, inter, stream)) return rc;
    }
    workspace += at.products;
    bytes -= at.products;
    if (dx) {
        ProductParams p = {};
        p.a = Operand{grad, 2 * inter};
        p.b = Operand{w, k};
        p.out = dx;
        p.exponents = exponents;
        p.M = rows;
        p.N = k;
        p.K = 2 * inter;
        if (int rc = run_product<T, true, false, kStore>(p, di, workspace, bytes, stream)) return rc;
    }
    if (dw) {
        ProductParams p = {};
        p.a = Operand{grad, 2 * inter};
        p.b = Operand{x, x_stride};
        p.out = dw;
        p.exponents = exponents ? exponents + 2 * rows : nullptr;
        p.M = 2 * inter;
        p.N = k;
        p.K = rows;
        if (int rc = run_product<T, false, false, kStore>(p, di, workspace, bytes, stream)) return rc;
    }
    return CKV_OK;
}

// A weight without rows to learn from: zeros, by a kernel (a recorded memset is no good).
__global__ void __launch_bounds__(256) zero_kernel(uint16_t* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace
}  // namespace ckv

extern "C" int64_t ckv_gated_linear_workspace_bytes(int64_t rows, int64_t inter, int64_t k, int32_t dtype) {
    using namespace ckv;
    DeviceInfo di;
    if (check_sizes(rows, inter, k, k, dtype) || rows == 0 || current_device_info(&di)) return 0;
    return product_bytes(rows, 2 * inter, k, true, true, di.cus);
}

extern "C" int ckv_gated_linear(const void* x, const void* w, void* out, float* gate_up, int64_t rows, int64_t inter, int64_t k, int64_t x_stride,
                                int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream_) {
    using namespace ckv;
    if (int rc = check_sizes(rows, inter, k, x_stride, dtype)) return rc;
    if (rows == 0) return CKV_OK;
    if (!x || !w || !out) return CKV_ERR_NULL;
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    switch (dtype) {
        case CKV_F32: return run_forward<float>(x, w, out, gate_up, rows, inter, k, x_stride, workspace, workspace_bytes, di, stream);
        case CKV_F16: return run_forward<__half>(x, w, out, gate_up, rows, inter, k, x_stride, workspace, workspace_bytes, di, stream);
        default: return run_forward<__hip_bfloat16>(x, w, out, gate_up, rows, inter, k, x_stride, workspace, workspace_bytes, di, stream);
    }
}

extern "C" int64_t ckv_gated_linear_bwd_workspace_bytes(int64_t rows, int64_t inter, int64_t k, int32_t dtype) {
    using namespace ckv;
    DeviceInfo di;
    if (check_sizes(rows, inter, k, k, dtype) || rows == 0 || current_device_info(&di)) return 0;
    const int64_t dx = product_bytes(rows, k, 2 * inter, true, false, di.cus), dw = product_bytes(2 * inter, k, rows, false, false, di.cus);
    return Scratch(rows, inter, k, dtype).products + std::max(dx, dw);
}

extern "C" int ckv_gated_linear_bwd(const void* x, const void* w, const float* gate_up, const void* dout, void* dx, void* dw, int64_t rows,
                                    int64_t inter, int64_t k, int64_t x_stride, int32_t dtype, void* workspace, int64_t workspace_bytes,
                                    void* stream_) {
    using namespace ckv;
    if (int rc = check_sizes(rows, inter, k, x_stride, dtype)) return rc;
    if (!dx && !dw) return CKV_OK;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (rows == 0) {
        if (!dw) return CKV_OK;
        hipLaunchKernelGGL(zero_kernel, dim3(2048), dim3(256), 0, stream, (uint16_t*)dw, 2 * inter * k * elem_bytes(dtype) / 2);
        CKV_HIP_TRY(hipGetLastError());
        return CKV_OK;
    }
    if (!x || !w || !gate_up || !dout) return CKV_ERR_NULL;
    if (dtype == CKV_F16 && (reinterpret_cast<uintptr_t>(workspace) & 3)) return CKV_ERR_WORKSPACE;   // which exponents lie in
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    if (!workspace || workspace_bytes < Scratch(rows, inter, k, dtype).products) return CKV_ERR_WORKSPACE;
    char* ws = (char*)workspace;
    switch (dtype) {
        case CKV_F32: return run_backward<float>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
        case CKV_F16: return run_backward<__half>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
        default: return run_backward<__hip_bfloat16>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
    }
}
