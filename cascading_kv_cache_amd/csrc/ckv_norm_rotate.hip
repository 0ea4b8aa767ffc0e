// RMSNorm of every head's query and key row and the half rotation of the rows at their tokens' positions, in one pass, and its gradients.
//
//   y = x rsqrt(mean(x^2) + eps) w,   o_j = y_j cos - y_{j+R/2} sin,   o_{j+R/2} = y_{j+R/2} cos + y_j sin,   j < R/2, angle = position f_j
//   g' = R^T g,   dw = sum over rows of g' xhat,   dx = r (g' w - xhat mean(g' w xhat)),   xhat = x r
//
// Bound by memory: rows are read once and written once (the gradients: two reads, a write).  A row is dealt out in slots, pairs of
// vectors of kVec elements that rotate with each other (j and j + R/2), or, behind the rotated part, neighbours; a lane has one slot (two
// where there are no vectors), a power of two of lanes a row, so that sums are a few exchanges between neighbours.  A lane stays with its
// token and walks over heads: the angles, whose range reduction is in double (a position times a frequency has more digits than float32),
// are worked out once for all of them.  Sums, norms and rotations are float32, rounded once at the end.  The next head's row is on its way while
// one is worked on.  bfloat16, heads of 128: 4096 tokens of 32 + 8 heads 16.4 us, 5.1 TB/s, the rate of a large copy; 4 x 2047 of 28 + 4 heads 25 us
// (5.4 TB/s), their gradients 46 (4.4) and the weights' sums 4; a single token 4.6, a launch.
#include "ckv_common.h"

#include <algorithm>

namespace ckv {
namespace {

constexpr int kMaxHeadDim = 256;
constexpr int kMostBlocks = 2048, kMostChunks = 64;   // of a backward launch

struct NormSide {
    const void* x;
    const void* weight;     // (D) or null: no norm
    const void* grad;       // backward: gradient of the output
    void* out;              // forward: output, backward: gradient of x
    int64_t x_stride[3], grad_stride[3], out_stride[3];   // batch, head, token
    int heads, chunks;      // chunks of heads_per heads
    float* partial;         // backward: (gridDim.x * chunks, D) sums of the weight's gradient, or null
};

struct NormParams {
    NormSide side[2];
    const int64_t* positions;
    int64_t pos_stride;
    const float* inv_freq;
    int64_t tokens;         // B * n
    int64_t n;
    int D, half, slots, lanes_log, heads_per;   // half: R / 2
    float eps;
};

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
    T v[kVec];
};

// sin and cos of position * frequency: quadrant and remainder in double, then Taylor series of the remainder (|r| <= pi / 4, next term below 2e-9).
__device__ inline void rotation_angle(int64_t position, float freq, float* sn, float* cs) {
    const double x = (double)position * (double)freq;
    const double n = __builtin_rint(x * 0.63661977236758134);
    double rd = __builtin_fma(-n, 1.5707963267948966, x);
    rd = __builtin_fma(-n, 6.123233995736766e-17, rd);
    const float r = (float)rd, z = r * r;
    const float s = r + r * z * fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -0.16666667f);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
    const int quadrant = (int)((int64_t)n & 3);
    const float a = quadrant & 1 ? c : s, b = quadrant & 1 ? s : c;
    *sn = quadrant & 2 ? -a : a;
    *cs = quadrant == 1 || quadrant == 2 ? -b : b;
}

template <typename T, int kVec>
__device__ inline void load_vec(const T* p, float (&v)[kVec]) {
    const Vec<T, kVec> a = *reinterpret_cast<const Vec<T, kVec>*>(p);
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] = Elem<T>::to_float(a.v[e]);
}

template <typename T, int kVec>
__device__ inline void store_vec(T* p, const float (&v)[kVec]) {
    Vec<T, kVec> a;
#pragma unroll
    for (int e = 0; e < kVec; e++) a.v[e] = Elem<T>::from_float(v[e]);
    *reinterpret_cast<Vec<T, kVec>*>(p) = a;
}

__device__ inline float sum_of_row(float s, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
    return s;
}

// A lane's share of a row: kSlots pairs of vectors.
template <typename T, int kVec, int kSlots>
struct Share {
    int at[kSlots][2];       // first element of each vector, -1: none
    bool turned[kSlots];
    __device__ Share(const NormParams& p, int lane_in_row) {
        const int lanes = 1 << p.lanes_log, rotated = p.half / kVec;
#pragma unroll
        for (int i = 0; i < kSlots; i++) {
            const int s = lane_in_row + i * lanes;
            turned[i] = s < rotated;
            if (turned[i]) {
                at[i][0] = s * kVec;
                at[i][1] = s * kVec + p.half;
            } else {
                const int from = 2 * p.half + 2 * (s - rotated) * kVec;
                at[i][0] = from < p.D ? from : -1;
                at[i][1] = from + kVec < p.D ? from + kVec : -1;
            }
        }
    }
    __device__ void load(const T* row, float (&v)[kSlots][2][kVec]) const {
#pragma unroll
        for (int i = 0; i < kSlots; i++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (at[i][u] >= 0) load_vec<T, kVec>(row + at[i][u], v[i][u]);
                else {
#pragma unroll
                    for (int e = 0; e < kVec; e++) v[i][u][e] = 0.f;
                }
            }
    }
    // The same in two steps: the loads, which the next head's work is put behind, and the conversion.
    using Raw = Vec<T, kVec>[kSlots][2];
    __device__ void fetch(const T* row, Raw& v) const {
#pragma unroll
        for (int i = 0; i < kSlots; i++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (at[i][u] >= 0) v[i][u] = *reinterpret_cast<const Vec<T, kVec>*>(row + at[i][u]);
    }
    __device__ void convert(const Raw& raw, float (&v)[kSlots][2][kVec]) const {
#pragma unroll
        for (int i = 0; i < kSlots; i++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < kVec; e++) v[i][u][e] = at[i][u] >= 0 ? Elem<T>::to_float(raw[i][u].v[e]) : 0.f;
    }
    __device__ void store(T* row, const float (&v)[kSlots][2][kVec]) const {
#pragma unroll
        for (int i = 0; i < kSlots; i++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (at[i][u] >= 0) store_vec<T, kVec>(row + at[i][u], v[i][u]);
    }
    __device__ void angles(const NormParams& p, int64_t b, int64_t t, float (&sn)[kSlots][kVec], float (&cs)[kSlots][kVec]) const {
        const int64_t position = p.half ? p.positions[b * p.pos_stride + t] : 0;
#pragma unroll
        for (int i = 0; i < kSlots; i++)
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                sn[i][e] = 0.f;
                cs[i][e] = 1.f;
                if (turned[i]) rotation_angle(position, p.inv_freq[at[i][0] + e], &sn[i][e], &cs[i][e]);
            }
    }
};

// Blocks: x takes tokens, y a chunk of the heads of one side.  Idle lanes (behind the last token or slot) go along: the exchanges meet them.
template <typename T, int kVec, int kSlots>
__global__ void __launch_bounds__(256) norm_rotate_kernel(NormParams p) {
    const bool keys = blockIdx.y >= (unsigned)p.side[0].chunks;
    const NormSide& side = p.side[keys];
    const int chunk = blockIdx.y - (keys ? p.side[0].chunks : 0);
    const int h0 = chunk * p.heads_per, h1 = min(side.heads, h0 + p.heads_per);
    const int lanes = 1 << p.lanes_log;
    const Share<T, kVec, kSlots> share(p, threadIdx.x & (lanes - 1));
    const int64_t token = (int64_t)blockIdx.x * (256 >> p.lanes_log) + (threadIdx.x >> p.lanes_log);
    const bool live = token < p.tokens;
    int64_t t;
    const int64_t b = div_index(live ? token : p.tokens - 1, p.n, t);
    float w[kSlots][2][kVec], sn[kSlots][kVec], cs[kSlots][kVec];
    if (side.weight) share.load((const T*)side.weight, w);
    share.angles(p, b, t, sn, cs);
    const T* from = (const T*)side.x + b * side.x_stride[0] + t * side.x_stride[2];
    T* to = (T*)side.out + b * side.out_stride[0] + t * side.out_stride[2];
    typename Share<T, kVec, kSlots>::Raw raw = {};
    share.fetch(from + h0 * side.x_stride[1], raw);
    for (int h = h0; h < h1; h++) {
        float x[kSlots][2][kVec];
        share.convert(raw, x);
        if (h + 1 < h1) share.fetch(from + (h + 1) * side.x_stride[1], raw);   // in flight while this head is worked on
        if (side.weight) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < kSlots; i++)
#pragma unroll
                for (int e = 0; e < kVec; e++) s = fmaf(x[i][0][e], x[i][0][e], fmaf(x[i][1][e], x[i][1][e], s));
            const float r = rsqrtf(sum_of_row(s, lanes) / (float)p.D + p.eps);
#pragma unroll
            for (int i = 0; i < kSlots; i++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int e = 0; e < kVec; e++) x[i][u][e] *= r * w[i][u][e];
        }
#pragma unroll
        for (int i = 0; i < kSlots; i++)
            if (share.turned[i]) {
#pragma unroll
                for (int e = 0; e < kVec; e++) {
                    const float a = x[i][0][e], c = x[i][1][e];
                    x[i][0][e] = a * cs[i][e] - c * sn[i][e];
                    x[i][1][e] = c * cs[i][e] + a * sn[i][e];
                }
            }
        if (live) share.store(to + h * side.out_stride[1], x);
    }
}

// The same walk backwards: 4.4 TB/s of two reads and a write, 46 us; 60 before the next head's rows were on their way, and 52 of 256 tokens' blocks had
// a second round of their own.  A lane keeps the sums of the weight's gradient for its own elements, over all tokens its block comes to (the
// grid steps over them) and all heads of the chunk; a block's sums are added up in LDS, the blocks' by weight_gradient_kernel: in a fixed
// order, no atomics.
template <typename T, int kVec, int kSlots>
__global__ void __launch_bounds__(256) norm_rotate_bwd_kernel(NormParams p) {
    __shared__ float sums[4][kMaxHeadDim];
    const bool keys = blockIdx.y >= (unsigned)p.side[0].chunks;
    const NormSide& side = p.side[keys];
    const int chunk = blockIdx.y - (keys ? p.side[0].chunks : 0);
    const int h0 = chunk * p.heads_per, h1 = min(side.heads, h0 + p.heads_per);
    const int lanes = 1 << p.lanes_log, per_block = 256 >> p.lanes_log;
    const Share<T, kVec, kSlots> share(p, threadIdx.x & (lanes - 1));
    float w[kSlots][2][kVec], dw[kSlots][2][kVec] = {};
    if (side.weight) share.load((const T*)side.weight, w);
    for (int64_t first = (int64_t)blockIdx.x * per_block; first < p.tokens; first += (int64_t)gridDim.x * per_block) {
        const int64_t token = first + (threadIdx.x >> p.lanes_log);
        const bool live = token < p.tokens;
        int64_t t;
        const int64_t b = div_index(live ? token : p.tokens - 1, p.n, t);
        float sn[kSlots][kVec], cs[kSlots][kVec];
        share.angles(p, b, t, sn, cs);
        const T* from = (const T*)side.x + b * side.x_stride[0] + t * side.x_stride[2];
        const T* grad = (const T*)side.grad + b * side.grad_stride[0] + t * side.grad_stride[2];
        T* to = (T*)side.out + b * side.out_stride[0] + t * side.out_stride[2];
        typename Share<T, kVec, kSlots>::Raw raw_x = {}, raw_g = {};
        share.fetch(grad + h0 * side.grad_stride[1], raw_g);
        if (side.weight) share.fetch(from + h0 * side.x_stride[1], raw_x);
        for (int h = h0; h < h1; h++) {
            float x[kSlots][2][kVec], g[kSlots][2][kVec];
            share.convert(raw_g, g);
            if (side.weight) share.convert(raw_x, x);
            if (h + 1 < h1) {   // in flight while this head is worked on
                share.fetch(grad + (h + 1) * side.grad_stride[1], raw_g);
                if (side.weight) share.fetch(from + (h + 1) * side.x_stride[1], raw_x);
            }
#pragma unroll
            for (int i = 0; i < kSlots; i++)
                if (share.turned[i]) {
#pragma unroll
                    for (int e = 0; e < kVec; e++) {
                        const float a = g[i][0][e], c = g[i][1][e];
                        g[i][0][e] = a * cs[i][e] + c * sn[i][e];
                        g[i][1][e] = c * cs[i][e] - a * sn[i][e];
                    }
                }
            if (side.weight) {
                float s = 0.f, along = 0.f;   // of x x and of g' w x
#pragma unroll
                for (int i = 0; i < kSlots; i++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < kVec; e++) {
                            s = fmaf(x[i][u][e], x[i][u][e], s);
                            along = fmaf(g[i][u][e] * w[i][u][e], x[i][u][e], along);
                        }
                for (int o = lanes >> 1; o > 0; o >>= 1) {
                    s += __shfl_xor(s, o);
                    along += __shfl_xor(along, o);
                }
                const float r = rsqrtf(s / (float)p.D + p.eps);
                const float mean = r * along / (float)p.D;
#pragma unroll
                for (int i = 0; i < kSlots; i++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < kVec; e++) {
                            const float unit = x[i][u][e] * r;
                            if (live) dw[i][u][e] = fmaf(g[i][u][e], unit, dw[i][u][e]);
                            g[i][u][e] = r * (g[i][u][e] * w[i][u][e] - unit * mean);
                        }
            }
            if (live) share.store(to + h * side.out_stride[1], g);
        }
    }
    if (!side.weight) return;
    float* row = side.partial + ((int64_t)blockIdx.x * side.chunks + chunk) * p.D;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < kSlots; i++)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                float s = dw[i][u][e];
                for (int o = lanes; o < CKV_WAVE; o <<= 1) s += __shfl_xor(s, o);
                if (lane < lanes && share.at[i][u] >= 0) sums[wave][share.at[i][u] + e] = s;
            }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += 256) row[d] = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
}

struct WeightGradients {
    const float* partial[2];
    void* out[2];
    int rows[2];
    int D;
};

// Column sums of the blocks' rows: 8 columns a workgroup, 128 threads a column, four rows in flight a thread.
template <typename T>
__global__ void __launch_bounds__(1024) weight_gradient_kernel(WeightGradients p) {
    __shared__ float sums[16][8];
    const int col = threadIdx.x & 7, part = threadIdx.x >> 3, side = blockIdx.y;
    const int at = blockIdx.x * 8 + col, rows = p.rows[side];
    float s[4] = {};
    if (at < p.D)
        for (int r = part; r < rows; r += 512) {
            const float* from = p.partial[side] + (int64_t)r * p.D + at;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (r + i * 128 < rows) s[i] += from[(int64_t)i * 128 * p.D];
        }
    float all = (s[0] + s[1]) + (s[2] + s[3]);
    for (int o = 8; o < CKV_WAVE; o <<= 1) all += __shfl_xor(all, o);
    if ((threadIdx.x & 63) < 8) sums[threadIdx.x >> 6][col] = all;
    __syncthreads();
    if (threadIdx.x < 8 && at < p.D) {
        all = 0.f;
        for (int i = 0; i < 16; i++) all += sums[i][col];
        ((T*)p.out[side])[at] = Elem<T>::from_float(all);
    }
}

bool vectors_fit(const ckv_norm_rotate_args* a, bool backward, int vec) {
    const int64_t bytes = vec * elem_bytes(a->dtype);
    if (a->D % vec || (a->rot / 2) % vec) return false;
    auto fits = [&](const void* p, const int64_t* stride) {
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride[0] % vec == 0 && stride[1] % vec == 0 && stride[2] % vec == 0;
    };
    const bool common = fits(a->q, a->q_stride) && fits(a->k, a->k_stride) && reinterpret_cast<uintptr_t>(a->q_weight) % bytes == 0 &&
                        reinterpret_cast<uintptr_t>(a->k_weight) % bytes == 0;
    if (!common) return false;
    if (!backward) return fits(a->q_out, a->q_out_stride) && fits(a->k_out, a->k_out_stride);
    return fits(a->q_grad, a->q_grad_stride) && fits(a->k_grad, a->k_grad_stride) && fits(a->dq, a->dq_stride) && fits(a->dk, a->dk_stride);
}

template <typename T, int kVec, int kSlots>
int launch_norm(NormParams& p, const ckv_norm_rotate_args* a, bool backward, int cus, hipStream_t stream) {
    p.slots = p.half / kVec + (int)((a->D - a->rot + 2 * kVec - 1) / (2 * kVec));
    p.lanes_log = 0;
    while ((kSlots << p.lanes_log) < p.slots) p.lanes_log++;
    const int64_t per_block = 256 >> p.lanes_log, blocks = std::max<int64_t>(1, (p.tokens + per_block - 1) / per_block);
    // Heads a block walks over: as many as leave sixteen wavefronts to a compute unit (a token's angles are worked out once a block)
    const int all = (int)(a->H + a->KVH);
    const int64_t wanted = std::max<int64_t>(1, 4 * (int64_t)cus / blocks);
    p.heads_per = (int)std::max<int64_t>((all + 32767) / 32768, all / wanted);   // chunks are a grid's y
    if (backward) p.heads_per = std::max(p.heads_per, (all + kMostChunks - 1) / kMostChunks);
    int chunks = 0;
    for (NormSide& s : p.side) chunks += s.chunks = (s.heads + p.heads_per - 1) / p.heads_per;
    if (chunks > 65535 || blocks > 0x7fffffff) return CKV_ERR_UNSUPPORTED;
    if (!backward) {
        hipLaunchKernelGGL((norm_rotate_kernel<T, kVec, kSlots>), dim3((unsigned)blocks, chunks), dim3(256), 0, stream, p);
        CKV_HIP_TRY(hipGetLastError());
        return CKV_OK;
    }
    const int64_t most = std::max(1, kMostBlocks / chunks), rounds = (blocks + most - 1) / most;
    const int gx = (int)((blocks + rounds - 1) / rounds);   // so that no block has a round more than most of the others
    p.side[0].partial = (float*)a->workspace;
    p.side[1].partial = p.side[0].partial + (int64_t)gx * p.side[0].chunks * p.D;
    hipLaunchKernelGGL((norm_rotate_bwd_kernel<T, kVec, kSlots>), dim3(gx, chunks), dim3(256), 0, stream, p);
    CKV_HIP_TRY(hipGetLastError());
    if (!a->q_weight) return CKV_OK;
    WeightGradients g;
    for (int i = 0; i < 2; i++) {
        g.partial[i] = p.side[i].partial;
        g.rows[i] = gx * p.side[i].chunks;
    }
    g.out[0] = a->dq_weight;
    g.out[1] = a->dk_weight;
    g.D = p.D;
    hipLaunchKernelGGL((weight_gradient_kernel<T>), dim3((p.D + 7) / 8, 2), dim3(1024), 0, stream, g);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

template <typename T>
int run_norm(NormParams& p, const ckv_norm_rotate_args* a, bool backward, int cus, hipStream_t stream) {
    constexpr int kMost = 16 / (int)sizeof(T);
    if (vectors_fit(a, backward, kMost)) return launch_norm<T, kMost, 1>(p, a, backward, cus, stream);
    if (vectors_fit(a, backward, 2)) return launch_norm<T, 2, 1>(p, a, backward, cus, stream);
    return launch_norm<T, 1, 2>(p, a, backward, cus, stream);
}

int norm_rotate(const ckv_norm_rotate_args* a, bool backward, hipStream_t stream) {
    if (!a) return CKV_ERR_NULL;
    if (a->dtype != CKV_F32 && a->dtype != CKV_F16 && a->dtype != CKV_BF16) return CKV_ERR_DTYPE;
    if (a->B < 0 || a->H <= 0 || a->KVH <= 0 || a->n < 0 || a->D <= 0 || a->rot < 0 || a->rot > a->D || a->rot % 2) return CKV_ERR_SHAPE;
    if (a->D > kMaxHeadDim || a->H > (1 << 20) || a->KVH > (1 << 20)) return CKV_ERR_UNSUPPORTED;
    if ((a->q_weight == nullptr) != (a->k_weight == nullptr)) return CKV_ERR_NULL;
    const bool nothing = a->B == 0 || a->n == 0;
    if (backward) {
        if (a->q_weight && (!a->dq_weight || !a->dk_weight)) return CKV_ERR_NULL;
        if (a->q_weight && (!a->workspace || a->workspace_bytes < ckv_norm_rotate_workspace_bytes(a->D))) return CKV_ERR_WORKSPACE;
    }
    if (nothing && !(backward && a->q_weight)) return CKV_OK;
    if (!nothing) {
        if (!a->q || !a->k || (a->rot && (!a->positions || !a->inv_freq))) return CKV_ERR_NULL;
        if (backward ? !a->q_grad || !a->k_grad || !a->dq || !a->dk : !a->q_out || !a->k_out) return CKV_ERR_NULL;
        if (a->q_stride[3] != 1 || a->k_stride[3] != 1) return CKV_ERR_STRIDE;
        if (backward ? a->q_grad_stride[3] != 1 || a->k_grad_stride[3] != 1 || a->dq_stride[3] != 1 || a->dk_stride[3] != 1
                     : a->q_out_stride[3] != 1 || a->k_out_stride[3] != 1)
            return CKV_ERR_STRIDE;
    }
    DeviceInfo di;
    if (int rc = current_device_info(&di)) return rc;
    NormParams p = {};
    p.tokens = a->B * a->n;
    p.n = std::max<int64_t>(1, a->n);
    p.D = (int)a->D;
    p.half = (int)(a->rot / 2);
    p.eps = a->eps;
    p.positions = a->positions;
    p.pos_stride = a->pos_stride;
    p.inv_freq = a->inv_freq;
    auto fill = [&](NormSide& s, const void* x, const int64_t* xs, const void* w, const void* g, const int64_t* gs, void* o, const int64_t* os, int64_t heads) {
        s.x = x;
        s.weight = w;
        s.grad = g;
        s.out = o;
        s.heads = (int)heads;
        for (int i = 0; i < 3; i++) {
            s.x_stride[i] = xs[i];
            s.grad_stride[i] = gs[i];
            s.out_stride[i] = os[i];
        }
    };
    fill(p.side[0], a->q, a->q_stride, a->q_weight, a->q_grad, a->q_grad_stride, backward ? a->dq : a->q_out, backward ? a->dq_stride : a->q_out_stride, a->H);
    fill(p.side[1], a->k, a->k_stride, a->k_weight, a->k_grad, a->k_grad_stride, backward ? a->dk : a->k_out, backward ? a->dk_stride : a->k_out_stride, a->KVH);
    switch (a->dtype) {
        case CKV_F32: return run_norm<float>(p, a, backward, di.cus, stream);
        case CKV_F16: return run_norm<__half>(p, a, backward, di.cus, stream);
        default: return run_norm<__hip_bfloat16>(p, a, backward, di.cus, stream);
    }
}

}  // namespace
}  // namespace ckv

extern "C" int64_t ckv_norm_rotate_workspace_bytes(int64_t D) {
    if (D <= 0 || D > ckv::kMaxHeadDim) return 0;
    return (int64_t)(ckv::kMostBlocks + 2 * ckv::kMostChunks) * D * 4;
}

extern "C" int ckv_norm_rotate(const ckv_norm_rotate_args* args, void* stream) {
    return ckv::norm_rotate(args, false, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int ckv_norm_rotate_bwd(const ckv_norm_rotate_args* args, void* stream) {
    return ckv::norm_rotate(args, true, reinterpret_cast<hipStream_t>(stream));
}
