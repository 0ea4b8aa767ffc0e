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

namespace ckv {
namespace {

// ---- any type, stride and size: float32 products on v_mfma_f32_32x32x2 -----------------------------------------------------------------

constexpr int kTile = 128, kStep = 16, kPitch = kTile + 4;

// A thread's four elements of a tile of 128 rows and 16 steps: along k of one row, or along the rows of one step.  Inside the operand they are
// read at a time, from whatever address (an odd number of float32 a row: 1023 columns, 509 rows and 5462, 64 us by elements and 52 so).
template <typename T, bool kAlongK>
struct Piece {
    struct __attribute__((packed, aligned(sizeof(T)))) Four {
        T v[4];
    };
    int row, step;   // of the first
    float v[4];
    __device__ Piece() {
        row = kAlongK ? threadIdx.x >> 2 : (threadIdx.x & 31) * 4;
        step = kAlongK ? (threadIdx.x & 3) * 4 : threadIdx.x >> 5;
    }
    // base: the operand's row 0; `first` the tile's first row, counted from base; rows behind `rows` and steps behind `end` are zeros
    __device__ void load(const T* base, int64_t stride, int64_t first, int64_t rows, int64_t k, int64_t end) {
        const int64_t r = first + row, s = k + step;
        const T* at = base + (kAlongK ? r * stride + s : s * stride + r);
        if (kAlongK ? r < rows && s + 4 <= end : s < end && r + 4 <= rows) {
            const Four x = *reinterpret_cast<const Four*>(at);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = Elem<T>::to_float(x.v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool there = kAlongK ? r < rows && s + i < end : s < end && r + i < rows;
                v[i] = there ? Elem<T>::to_float(at[i]) : 0.f;
            }
        }
    }
    __device__ void store(float (*tile)[kPitch]) const {
        if constexpr (kAlongK) {
#pragma unroll
            for (int i = 0; i < 4; i++) tile[step + i][row] = v[i];
        } else {
            *reinterpret_cast<float4*>(&tile[step][row]) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
};

// Eight wavefronts of 32 x 64, two on a SIMD: one's loads and stores stand beside the other's products.
template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
__global__ void __launch_bounds__(512) product_kernel(ProductParams p) {
    __shared__ __align__(16) float as[2][kStep][kPitch], bs[2][kStep][kPitch];
    int tm, tn, share;
    float* sums = work_of<8>(p, kTile * kTile, tm, tn, share);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1, half = lane >> 5, l = lane & 31;
    constexpr bool kGated = kEpilogue == kGate;
    const int64_t inter = p.N / 2;
    const int64_t m0 = (int64_t)tm * kTile, n0 = (int64_t)tn * (kGated ? kTile / 2 : kTile);
    const int64_t k0 = share * p.k_share, k1 = sums ? min(p.K, k0 + p.k_share) : p.K;
    Piece<T, kAlongKA> pa;
    Piece<T, kAlongKB> pb;
    const T* a = (const T*)p.a.p;
    const T* b = (const T*)p.b.p;
    // gated: rows 0..63 of B's tile are gate rows, 64..127 up rows
    const bool up = kGated && pb.row >= kTile / 2;
    auto load = [&](int64_t k) {
        pa.load(a, p.a.stride, m0, p.M, k, k1);
        if constexpr (kGated) pb.load(b + (up ? inter * p.b.stride : 0), p.b.stride, n0 - (up ? kTile / 2 : 0), inter, k, k1);
        else pb.load(b, p.b.stride, n0, p.N, k, k1);
    };
    const bool there = m0 + wm * 32 < p.M;   // of a few rows most of the products would be of none: 64 x 5632 x 1024, 33 -> 25 us
    f32x16_t acc[2] = {};
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
        for (int s = 0; s < kStep; s += 2) {
            const float av = as[at][s + half][wm * 32 + l];
#pragma unroll
            for (int j = 0; j < 2; j++)
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(av, bs[at][s + half][kGated ? j * 64 + wn * 32 + l : wn * 64 + j * 32 + l], acc[j], 0, 0, 0);
        }
        if (more) {
            pa.store(as[at ^ 1]);
            pb.store(bs[at ^ 1]);
        }
        __syncthreads();
        at ^= 1;
    }
    // element r of an accumulator: row 8 (r / 4) + 4 half + r % 4, column l
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int row = wm * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        const int64_t m = m0 + row;
        if (sums) {
#pragma unroll
            for (int j = 0; j < 2; j++) sums[row * kTile + (kGated ? j * 64 + wn * 32 : wn * 64 + j * 32) + l] = acc[j][r];
            continue;
        }
        if (m >= p.M) continue;
        if constexpr (kGated) {
            const int64_t n = n0 + wn * 32 + l;
            if (n >= inter) continue;
            const float g = acc[0][r], u = acc[1][r];
            ((T*)p.out)[m * inter + n] = Elem<T>::from_float(gate_product(g, u));
            if (p.both) {
                T* to = (T*)p.both + m * p.N + n;
                to[0] = Elem<T>::from_float(g);
                to[inter] = Elem<T>::from_float(u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int64_t n = n0 + wn * 64 + j * 32 + l;
                if (n < p.N) ((T*)p.out)[m * p.N + n] = Elem<T>::from_float(acc[j][r]);
            }
        }
    }
}

// Sums of the shares of a tile, in their order, and what the product's own epilogue does.  A workgroup has some rows of a tile, a thread four
// columns.
template <typename T, Epilogue kEpilogue>
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
                    T* to = (T*)p.both + m * p.N + n + e;
                    to[0] = Elem<T>::from_float(g[e]);
                    to[cols] = Elem<T>::from_float(u[e]);
                }
            } else {
                ((T*)p.out)[m * cols + n + e] = Elem<T>::from_float(g[e]);
            }
        }
    }
}

// ---- gradients of the projections ------------------------------------------------------------------------------------------------------

template <typename T, int kPer>
__global__ void __launch_bounds__(256) gate_gradient_kernel(const T* gate_up, const T* dout, T* grad, int64_t rows, int64_t inter) {
    struct alignas(sizeof(T) * kPer) Piece {
        T v[kPer];
    };
    const int64_t pieces = inter / kPer, all = rows * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        int64_t c;
        const int64_t row = div_index(i, pieces, c);
        const T* from = gate_up + row * 2 * inter + c * kPer;
        const Piece gate = *reinterpret_cast<const Piece*>(from), up = *reinterpret_cast<const Piece*>(from + inter);
        const Piece dh = *reinterpret_cast<const Piece*>(dout + row * inter + c * kPer);
        Piece dg, du;
#pragma unroll
        for (int e = 0; e < kPer; e++) {
            const float g = Elem<T>::to_float(gate.v[e]), u = Elem<T>::to_float(up.v[e]), d = Elem<T>::to_float(dh.v[e]);
            const float s = 1.f / (1.f + expf(-g));
            dg.v[e] = Elem<T>::from_float(d * u * s * (1.f + g * (1.f - s)));
            du.v[e] = Elem<T>::from_float(d * g * s);
        }
        T* to = grad + row * 2 * inter + c * kPer;
        *reinterpret_cast<Piece*>(to) = dg;
        *reinterpret_cast<Piece*>(to + inter) = du;
    }
}

template <typename T>
int gate_gradient(const void* gate_up, const void* dout, void* grad, int64_t rows, int64_t inter, hipStream_t stream) {
    constexpr int kPer = 16 / (int)sizeof(T);
    const bool pieces = inter % kPer == 0 &&
                        ((reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    const int64_t all = rows * inter / (pieces ? kPer : 1);
    const unsigned blocks = (unsigned)std::min<int64_t>((all + 255) / 256, 256 * 16);
    if (pieces) hipLaunchKernelGGL((gate_gradient_kernel<T, kPer>), dim3(blocks), dim3(256), 0, stream, (const T*)gate_up, (const T*)dout, (T*)grad, rows, inter);
    else hipLaunchKernelGGL((gate_gradient_kernel<T, 1>), dim3(blocks), dim3(256), 0, stream, (const T*)gate_up, (const T*)dout, (T*)grad, rows, inter);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

// ---- which kernel, how many shares -----------------------------------------------------------------------------------------------------

// The kernels of 16-bit tiles take operands of whole pieces of 16 bytes: all but odd sizes, strides and addresses.
template <typename T>
bool fits_tiles(const ProductParams& p, bool along_a, bool along_b, bool gated) {
    if (sizeof(T) != 2) return false;
    auto whole = [&](const Operand& o, bool along, int64_t rows) {
        return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.stride % 8 == 0 && (along ? p.K : rows) % 8 == 0 && o.stride < (1 << 22);
    };
    return whole(p.a, along_a, p.M) && whole(p.b, along_b, p.N) && (gated ? p.N / 2 : p.N) % 8 == 0 &&
           ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.both)) & 15) == 0;
}

// Where the tiles of float32 products leave compute units idle, the steps are shared out over as many workgroups as come to one each, none with
// fewer than 128.
TilePlan plan_float(int64_t M, int64_t N, int64_t K, int cus) {
    TilePlan r;
    r.tile_m = r.tile_n = kTile;
    r.stages = 2;
    r.tiles_m = (int)((M + kTile - 1) / kTile);
    r.tiles_n = (int)((N + kTile - 1) / kTile);
    const int64_t tiles = (int64_t)r.tiles_m * r.tiles_n;
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(cus / tiles, K / 128));
    r.k_share = ((K + shares - 1) / shares + kStep - 1) / kStep * kStep;
    r.shares = (int)((K + r.k_share - 1) / r.k_share);
    r.whole_tiles = r.shares > 1 ? 0 : (int)std::min<int64_t>(tiles, 0x7fffffff);
    return r;
}

// Columns of B's tiles are gate and up columns by halves, so there may be tiles with few of either.
int64_t tiled_columns(int64_t N, bool gated, int tile_n) {
    return gated ? (N / 2 + tile_n / 2 - 1) / (tile_n / 2) * tile_n : N;
}

// Scratch of a product, whichever kernel takes it.
int64_t product_bytes(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus) {
    return std::max(plan_tiles(M, tiled_columns(N, gated, 128), K, a_along_k, cus).bytes(), plan_float(M, tiled_columns(N, gated, kTile), K, cus).bytes());
}

template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int run_product(ProductParams& p, const DeviceInfo& di, void* workspace, int64_t bytes, hipStream_t stream) {
    constexpr bool kGated = kEpilogue == kGate;
    const bool tiles = fits_tiles<T>(p, kAlongKA, kAlongKB, kGated);
    const TilePlan plan = tiles ? plan_tiles(p.M, tiled_columns(p.N, kGated, 128), p.K, kAlongKA, di.cus)
                                : plan_float(p.M, tiled_columns(p.N, kGated, kTile), p.K, di.cus);
    if (plan.bytes() && (!workspace || plan.bytes() > bytes || reinterpret_cast<uintptr_t>(workspace) & 15)) return CKV_ERR_WORKSPACE;
    if ((int64_t)plan.tiles_m * plan.tiles_n > 0x3fffffff || plan.blocks() > 0x7fffffff) return CKV_ERR_UNSUPPORTED;
    plan.fill(p);
    p.partial = (float*)workspace;
    if (tiles) {
        if constexpr (sizeof(T) == 2)
            if (int rc = run_tiles<T>(p, plan, kAlongKA, kEpilogue, stream)) return rc;
    } else {
        hipLaunchKernelGGL((product_kernel<T, kAlongKA, kAlongKB, kEpilogue>), dim3((unsigned)plan.blocks()), dim3(512), 0, stream, p);
        CKV_HIP_TRY(hipGetLastError());
    }
    if (plan.shares > 1) {
        constexpr int kRows = 8;
        hipLaunchKernelGGL((merge_kernel<T, kEpilogue>), dim3(plan.tiles_m * plan.tiles_n - plan.whole_tiles, plan.tile_m / kRows), dim3(256), 0, stream, p, plan.tile_m,
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
int run_forward(const void* x, const void* w, void* out, void* gate_up, int64_t rows, int64_t inter, int64_t k, int64_t x_stride, void* workspace,
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

template <typename T>
int run_backward(const void* x, const void* w, const void* gate_up, const void* dout, void* dx, void* dw, int64_t rows, int64_t inter, int64_t k,
                 int64_t x_stride, char* workspace, int64_t bytes, const DeviceInfo& di, hipStream_t stream) {
    const int64_t grad_bytes = align_up(rows * 2 * inter * (int64_t)sizeof(T), 256);
    void* grad = workspace;
    if (int rc = gate_gradient<T>(gate_up, dout, grad, rows, inter, stream)) return rc;
    workspace += grad_bytes;
    bytes -= grad_bytes;
    if (dx) {
        ProductParams p = {};
        p.a = Operand{grad, 2 * inter};
        p.b = Operand{w, k};
        p.out = dx;
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

extern "C" int ckv_gated_linear(const void* x, const void* w, void* out, void* gate_up, int64_t rows, int64_t inter, int64_t k, int64_t x_stride,
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
    return align_up(rows * 2 * inter * elem_bytes(dtype), 256) + std::max(dx, dw);
}

extern "C" int ckv_gated_linear_bwd(const void* x, const void* w, const void* gate_up, const void* dout, void* dx, void* dw, int64_t rows,
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
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    if (!workspace || workspace_bytes < align_up(rows * 2 * inter * elem_bytes(dtype), 256)) return CKV_ERR_WORKSPACE;
    char* ws = (char*)workspace;
    switch (dtype) {
        case CKV_F32: return run_backward<float>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
        case CKV_F16: return run_backward<__half>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
        default: return run_backward<__hip_bfloat16>(x, w, gate_up, dout, dx, dw, rows, inter, k, x_stride, ws, workspace_bytes, di, stream);
    }
}
