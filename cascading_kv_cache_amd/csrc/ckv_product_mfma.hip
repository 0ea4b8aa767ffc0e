// C (M, N) = sum over k of A (m, k) B (n, k) of 16-bit operands on v_mfma_f32_32x32x16, with the gate of a gated MLP or shares of the
// sum behind it.
//
// A workgroup has a tile of C and brings 64 steps of both operands at a time into one of two stages of LDS by asynchronous copies, while
// it works on the other: one barrier a stage.  An operand whose rows are adjacent along k lies in LDS as rows of 128 bytes, and an operand read
// is 16 of them; one whose steps are adjacent along its rows lies as it is, and is turned on the way into registers (ds_read_b64_tr_b16).
// Pieces of 16 bytes are permuted within a row as they are copied, so that an operand read meets every bank once.
#include "ckv_product.h"

#include <algorithm>

namespace ckv {
namespace {

typedef __bf16 product_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 product_f16x8 __attribute__((ext_vector_type(8)));
typedef short product_s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t product_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSteps = 64;   // of a stage

template <typename T>
__device__ inline f32x16_t mma(uint4 a, uint4 b, f32x16_t c) {
    if constexpr (std::is_same<T, __hip_bfloat16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(product_bf16x8, a), __builtin_bit_cast(product_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(product_f16x8, a), __builtin_bit_cast(product_f16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ inline uint2 pack4(float a, float b, float c, float d) {
    return make_uint2(RopeWord<T>::pack2(a, b), RopeWord<T>::pack2(c, d));
}

// What steps behind the last one read: zeros of both operands (another row's number may be one times zero that is not zero).
__device__ uint4 g_zeros[1];

// One operand of a tile kRows rows high: copies of a wavefront, and where the lanes' operands lie.
template <int kRows, bool kAlongK, int kWaves>
struct Side {
    static constexpr int kCopies = kRows / 8 / kWaves;       // of 1 KiB a wavefront and stage
    static constexpr int kBytes = kRows * kSteps * 2;
    static constexpr int kRowBytes = kAlongK ? kSteps * 2 : kRows * 2;   // of LDS
    const char* base[kCopies];   // uniform; with the gate the rows of a copy are all gate or all up rows
    uint32_t voff[kCopies];
    int step[kCopies];           // of the lane's piece, counted from the stage's first
    int64_t advance;             // bytes a stage

    // `first`, `rows`: the tile's first row and how many the operand has; kGated: rows kRows / 2 and up are row `first` of the second half
    template <bool kGated>
    __device__ void init(const Operand& o, int64_t first, int64_t rows, int64_t k0, int wave, int lane) {
        const int64_t row_bytes = 2 * o.stride;
        advance = kAlongK ? 2 * kSteps : kSteps * row_bytes;
#pragma unroll
        for (int c = 0; c < kCopies; c++) {
            const int copy = wave * kCopies + c;
            if constexpr (kAlongK) {
                const bool up = kGated && 8 * copy >= kRows / 2;
                const int row = 8 * copy + (lane >> 3), in_half = row - (up ? kRows / 2 : 0);
                const int piece = (lane & 7) ^ ((row >> 1) & 7);
                const int64_t left = rows - first - 1;
                base[c] = (const char*)o.p + ((up ? rows : 0) + first) * row_bytes + 2 * k0;
                voff[c] = (uint32_t)(min((int64_t)in_half, left) * row_bytes) + 16 * piece;
                step[c] = 8 * piece;
            } else {
                constexpr int kLanes = kRows / 8;   // of a step
                const int k = copy * (64 / kLanes) + lane / kLanes;
                const int piece = (lane % kLanes) ^ ((k & 3) << 2);
                const int64_t left = rows - first - 8;
                base[c] = (const char*)o.p + k0 * row_bytes + 2 * first;
                voff[c] = (uint32_t)(k * row_bytes) + 2 * (uint32_t)min((int64_t)(8 * piece), left);
                step[c] = k;
            }
        }
    }
    __device__ void copy(int64_t stage, uint32_t lds, int wave) const {
#pragma unroll
        for (int c = 0; c < kCopies; c++) async_copy16(base[c] + stage * advance, voff[c], lds + (wave * kCopies + c) * 1024);
    }
    // the last stage, of which `left` steps are there
    __device__ void copy_some(int64_t stage, uint32_t lds, int wave, int left) const {
#pragma unroll
        for (int c = 0; c < kCopies; c++) {
            const char* from = base[c] + stage * advance + voff[c];
            async_copy16_from(step[c] < left ? (const void*)from : (const void*)g_zeros, lds + (wave * kCopies + c) * 1024);
        }
    }
};

// Operands of kFrags blocks of 32 rows.  Element e of a lane: row lane % 32 of the block, step 16 s + 8 (lane / 32) + e.
template <int kRows, bool kAlongK, int kFrags>
struct Reader {
    uint32_t at[kAlongK ? kSteps / 16 : kFrags];
    // block f's first row is f0 + 32 f, behind kSplit blocks f1 + 32 (f - kSplit)
    __device__ void init(uint32_t lds, int f0, int lane) {
        if constexpr (kAlongK) {
            const int r = lane & 31, h = lane >> 5;
#pragma unroll
            for (int s = 0; s < kSteps / 16; s++) at[s] = lds + (f0 + r) * (kSteps * 2) + (((2 * s + h) ^ ((r >> 1) & 7)) << 4);
        } else {
            const int rl = lane & 15, g = (lane >> 4) & 1, h = lane >> 5, k = 8 * h + (rl >> 2);
#pragma unroll
            for (int f = 0; f < kFrags; f++) {
                const int piece = (f0 + 32 * f) / 8 + 2 * g + ((rl & 3) >> 1);
                at[f] = lds + k * (kRows * 2) + ((piece ^ ((k & 3) << 2)) << 4) + 8 * (rl & 1);
            }
        }
    }
    // `jump`: bytes that the block lies further than 32 rows a block would put it
    __device__ uint4 read(uint32_t stage, int s, int f, int jump) const {
        if constexpr (kAlongK) {
            const product_u32x4 v = *(const __attribute__((address_space(3))) product_u32x4*)(uintptr_t)(at[s] + stage + f * 32 * (kSteps * 2) + jump);
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            uint2 u[2];
#pragma unroll
            for (int a = 0; a < 2; a++)
                u[a] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) product_s16x4*)(uintptr_t)(
                                                     at[f] + stage + (16 * s + 4 * a) * (kRows * 2))));
            return make_uint4(u[0].x, u[0].y, u[1].x, u[1].y);
        }
    }
};

template <int kTileM, int kTileN>
constexpr int kStageBytes = (kTileM + kTileN) * kSteps * 2;

template <typename T, int kTileM, int kTileN, int kWavesM, int kWavesN, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
__global__ void __launch_bounds__(64 * kWavesM * kWavesN) tile_kernel(ProductParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr bool kGated = kEpilogue == kGate;
    constexpr int kWaves = kWavesM * kWavesN, kFragsM = kTileM / kWavesM / 32, kFragsN = kTileN / kWavesN / 32;
    constexpr int kStage = kStageBytes<kTileM, kTileN>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / kWavesN, wn = wave % kWavesN;
    int tm, tn;
    tile_of<4>(p, tm, tn);
    const int64_t cols = kGated ? p.N / 2 : p.N;
    const int64_t m0 = (int64_t)tm * kTileM, n0 = (int64_t)tn * (kGated ? kTileN / 2 : kTileN);
    const int64_t k0 = blockIdx.y * p.k_share, steps = min(p.K - k0, p.k_share);
    const uint32_t lds = lds_address(smem);

    Side<kTileM, kAlongKA, kWaves> a;
    Side<kTileN, kAlongKB, kWaves> b;
    a.template init<false>(p.a, m0, p.M, k0, wave, lane);
    b.template init<kGated>(p.b, n0, cols, k0, wave, lane);
    Reader<kTileM, kAlongKA, kFragsM> ra;
    Reader<kTileN, kAlongKB, kFragsN> rb;
    ra.init(lds, wm * (kTileM / kWavesM), lane);
    rb.init(lds + Side<kTileM, kAlongKA, kWaves>::kBytes, kGated ? wn * (kTileN / kWavesN / 2) : wn * (kTileN / kWavesN), lane);
    // with the gate, a wavefront's second half of blocks are the up columns of its first
    constexpr int kJump = kGated ? (kTileN / 2 - kTileN / kWavesN / 2) * kSteps * 2 : 0;

    const int64_t whole = steps / kSteps, stages = (steps + kSteps - 1) / kSteps;
    auto copy = [&](int64_t stage) {
        const uint32_t to = lds + (uint32_t)(stage & 1) * kStage, to_b = to + Side<kTileM, kAlongKA, kWaves>::kBytes;
        if (stage < whole) {
            a.copy(stage, to, wave);
            b.copy(stage, to_b, wave);
        } else {
            const int left = (int)(steps - stage * kSteps);
            a.copy_some(stage, to, wave, left);
            b.copy_some(stage, to_b, wave, left);
        }
    };
    f32x16_t acc[kFragsM][kFragsN] = {};
    copy(0);
    for (int64_t stage = 0; stage < stages; stage++) {
        wait_copies<0>();
        __syncthreads();   // everybody's copies are there, and nobody reads the other stage any more
        if (stage + 1 < stages) copy(stage + 1);
        const uint32_t at = (uint32_t)(stage & 1) * kStage;
#pragma unroll
        for (int s = 0; s < kSteps / 16; s++) {
            uint4 av[kFragsM], bv[kFragsN];
#pragma unroll
            for (int i = 0; i < kFragsM; i++) av[i] = ra.read(at, s, i, 0);
#pragma unroll
            for (int j = 0; j < kFragsN; j++) bv[j] = rb.read(at, s, j, j >= kFragsN / 2 ? kJump : 0);
#pragma unroll
            for (int i = 0; i < kFragsM; i++)
#pragma unroll
                for (int j = 0; j < kFragsN; j++) acc[i][j] = mma<T>(bv[j], av[i], acc[i][j]);
        }
    }

    // Accumulator element r of a lane: row lane % 32 of C's block, column 8 (r / 4) + 4 (lane / 32) + r % 4.
    const int r32 = lane & 31, h = lane >> 5;
    const int64_t mw = m0 + wm * (kTileM / kWavesM), nw = n0 + wn * (kGated ? kTileN / kWavesN / 2 : kTileN / kWavesN);
    if (p.partial) {
#pragma unroll
        for (int i = 0; i < kFragsM; i++) {
            const int64_t m = mw + 32 * i + r32;
            float* row = p.partial + (blockIdx.y * p.M + m) * p.N;
#pragma unroll
            for (int j = 0; j < kFragsN; j++) {
                const bool up = kGated && j >= kFragsN / 2;
                const int64_t n = nw + 32 * (up ? j - kFragsN / 2 : j);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (m < p.M && n + 8 * q < cols)
                        *reinterpret_cast<float4*>(row + (up ? cols : 0) + n + 8 * q + 4 * h) =
                            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
            }
        }
        return;
    }
    // 32 rows at a time go through the wavefront's part of LDS, so that whole pieces of a row are written at a time.
    __syncthreads();
    constexpr int kBlocks = kGated ? kFragsN / 2 : kFragsN, kPieces = kBlocks * 4, kPitch = kBlocks * 64 + 16;
    unsigned char* mine = smem + wave * (32 * kPitch);
    auto write = [&](int i, auto value, void* out, int64_t stride, int64_t first) {
#pragma unroll
        for (int j = 0; j < kBlocks; j++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<uint2*>(mine + r32 * kPitch + (32 * j + 8 * q + 4 * h) * 2) =
                    pack4<T>(value(j, 4 * q), value(j, 4 * q + 1), value(j, 4 * q + 2), value(j, 4 * q + 3));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int piece = lane % kPieces;
#pragma unroll
        for (int x = 0; x < 32 * kPieces / 64; x++) {
            const int row = x * (64 / kPieces) + lane / kPieces;
            const int64_t m = mw + 32 * i + row, n = nw + 8 * piece;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + row * kPitch + piece * 16);
            if (m < p.M && n < cols) *reinterpret_cast<uint4*>((T*)out + m * stride + first + n) = v;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kFragsM; i++) {
        if constexpr (kGated) {
            write(i, [&](int j, int r) { return gate_product(acc[i][j][r], acc[i][j + kBlocks][r]); }, p.out, cols, 0);
            if (p.both) {
                write(i, [&](int j, int r) { return acc[i][j][r]; }, p.both, p.N, 0);
                write(i, [&](int j, int r) { return acc[i][j + kBlocks][r]; }, p.both, p.N, cols);
            }
        } else {
            write(i, [&](int j, int r) { return acc[i][j][r]; }, p.out, p.N, 0);
        }
    }
}

template <typename T, int kTileM, int kTileN, int kWavesM, int kWavesN, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int launch_tiles(const ProductParams& p, const TilePlan& plan, hipStream_t stream) {
    auto kernel = tile_kernel<T, kTileM, kTileN, kWavesM, kWavesN, kAlongKA, kAlongKB, kEpilogue>;
    constexpr int lds = 2 * kStageBytes<kTileM, kTileN>;
    if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3(plan.tiles_m * plan.tiles_n, plan.shares), dim3(64 * kWavesM * kWavesN), lds, stream, p);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int launch_tiles(const ProductParams& p, const TilePlan& plan, hipStream_t stream) {
    if (plan.tile_m == 256) return launch_tiles<T, 256, 256, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    if (plan.tile_m == 128) return launch_tiles<T, 128, 128, 2, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    if constexpr (kAlongKA) return launch_tiles<T, 64, 128, 2, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    return CKV_ERR_UNSUPPORTED;
}

}  // namespace

TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus) {
    TilePlan r;
    auto tiles = [&](int tm, int tn) { return ((M + tm - 1) / tm) * ((N + tn - 1) / tn); };
    r.tile_m = a_along_k && M <= 64 ? 64 : tiles(256, 256) < cus ? 128 : 256;
    r.tile_n = r.tile_m == 256 ? 256 : 128;
    r.tiles_m = (int)((M + r.tile_m - 1) / r.tile_m);
    r.tiles_n = (int)(((gated ? N / 2 : N) + r.tile_n / (gated ? 2 : 1) - 1) / (r.tile_n / (gated ? 2 : 1)));
    const int64_t all = (int64_t)r.tiles_m * r.tiles_n;
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(2 * cus / all, K / 512));
    r.k_share = ((K + shares - 1) / shares + kSteps - 1) / kSteps * kSteps;
    r.shares = (int)((K + r.k_share - 1) / r.k_share);
    return r;
}

template <typename T>
int run_tiles(ProductParams& p, const TilePlan& plan, bool a_along_k, bool b_along_k, Epilogue epilogue, hipStream_t stream) {
    p.tiles_m = plan.tiles_m;
    p.tiles_n = plan.tiles_n;
    p.k_share = plan.k_share;
    if (epilogue == kGate) return launch_tiles<T, true, true, kGate>(p, plan, stream);
    if (a_along_k) return launch_tiles<T, true, false, kStore>(p, plan, stream);
    return launch_tiles<T, false, false, kStore>(p, plan, stream);
}
template int run_tiles<__half>(ProductParams&, const TilePlan&, bool, bool, Epilogue, hipStream_t);
template int run_tiles<__hip_bfloat16>(ProductParams&, const TilePlan&, bool, bool, Epilogue, hipStream_t);

}  // namespace ckv
