// C (M, N) = sum over k of A (m, k) B (n, k) of 16-bit operands on v_mfma_f32_16x16x32, with the gate of a gated MLP or shares of the
// sum behind it.
//
// A workgroup has a tile of C and brings 32 or 64 steps of both operands at a time into one of three to seven stages of LDS by asynchronous copies,
// all but one of them ahead: one barrier a stage.  An operand whose rows are adjacent along k lies in LDS as rows of 64 or 128 bytes, and an operand
// read is 16 of them; one whose steps are adjacent along its rows lies as it is, and is turned on the way into registers (ds_read_b64_tr_b16).
// Pieces of 16 bytes are permuted within a row as they are copied, so that an operand read meets every bank once.
//
// Few rows wait for the bytes of B, and 64 steps of a row along k are a whole line (77 x 28672 x 4096 by halves of lines 53 us, 44 so: 5.3 TB/s).
// Many are bound by the products and the power they take: 4096 x 28672 x 4096 720 us, 1.34 PFLOP/s (the library's product alone, without the gate, 640),
// 2048 x 37888 x 3584 440 (510).  There the largest tile has room for stages of 32 steps alone, and is level with lower ones of 64.
//
// A wavefront of the large tile has 128 x 128 of it: with 64 x 128 each (eight wavefronts) the reads and copies of LDS alone take as long as the
// products (a stage of 64 steps: 1536 + 512 of 2048 cycles).  One wavefront on a SIMD hides nothing behind another, so reads of the next
// operands and copies stand between the products, one at a time.
#include "ckv_product.h"

#include <algorithm>
#include <utility>

namespace ckv {
namespace {

// f(0), f(1), ... f(kN - 1), the numbers known to the compiler
template <typename F, int... kI>
__device__ __attribute__((always_inline)) inline void each(F f, std::integer_sequence<int, kI...>) {
    (f(std::integral_constant<int, kI>{}), ...);
}
template <int kN, typename F>
__device__ __attribute__((always_inline)) inline void each(F f) {
    each(f, std::make_integer_sequence<int, kN>{});
}

typedef __bf16 product_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 product_f16x8 __attribute__((ext_vector_type(8)));
typedef short product_s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t product_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSteps = 32;   // of a matrix instruction; a stage has kDeep times as many

// Written as an instruction, its sum in place: what the compiler makes of the builtin gives a sum another register than it had, and moves it
// back, where there are as many as a wavefront of the large tile has.  Whoever reads a sum other than by the next product waits (sums_done).
template <typename T>
__device__ inline void mma(uint4 a, uint4 b, f32x4_t& c) {
    if constexpr (std::is_same<T, __hip_bfloat16>::value)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(__builtin_bit_cast(product_bf16x8, a)), "v"(__builtin_bit_cast(product_bf16x8, b)));
    else
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(__builtin_bit_cast(product_f16x8, a)), "v"(__builtin_bit_cast(product_f16x8, b)));
}
template <int kM, int kN>
__device__ inline void sums_done(f32x4_t (&c)[kM][kN]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < kM; i++)
#pragma unroll
        for (int j = 0; j < kN; j++) asm volatile("" : "+a"(c[i][j]));   // nobody reads it earlier
}

template <typename T>
__device__ inline uint2 pack4(float a, float b, float c, float d) {
    return make_uint2(RopeWord<T>::pack2(a, b), RopeWord<T>::pack2(c, d));
}

// What steps behind the last one read: zeros of both operands (another row's number may be one times zero that is not zero).
__device__ uint4 g_zeros[1];

// Which bits of the number of a piece step k flips: a read that turns 8 steps (k..k+3 and k+8..k+11) of 16 rows meets every bank once.
__device__ inline int turned_bits(int k) { return ((k & 3) << 2) | ((k >> 2) & 2); }

// The same where rows lie along k, of kPieces pieces: which bits of the number of a piece row r flips.  A read of 16 bytes a lane goes in four
// parts, of lanes 0-3, 12-15, 20-23 and 24-27 the first, of 4-11, 16-19 and 28-31 the second: rows 4 q.. of piece 0 for two q, of piece 1 for the
// two others.
template <int kPieces>
__device__ inline int first_piece(int r) {
    return kPieces == 4 ? ((r >> 2 << 1) ^ ((r >> 3 & 1) * 3)) & 3 : (r >> 1) & 7;
}

// One operand of a tile kRows rows high: copies of a wavefront, and where the lanes' pieces come from.
template <int kRows, bool kAlongK, int kWaves, int kDeep>
struct Side {
    static constexpr int kStageSteps = kSteps * kDeep, kPieces = kStageSteps / 8;   // of a row along k
    static constexpr int kCopies = kRows * kStageSteps / 512 / kWaves;   // of 1 KiB a wavefront and stage
    static constexpr int kBytes = kRows * kStageSteps * 2;
    const char* at;              // uniform: of the next stage to be copied
    int64_t advance;             // bytes a stage
    uint32_t voff[kCopies];

    // `first`, `rows`: the tile's first row and how many the operand has; kGated: rows kRows / 2 and up, copied by the second half of the
    // wavefronts, are row `first` of the operand's second half
    template <bool kGated>
    __device__ void init(const Operand& o, int64_t first, int64_t rows, int64_t k0, int wave, int lane) {
        static_assert(!kGated || (kAlongK && kWaves % 2 == 0), "a wavefront's copies are all gate or all up rows");
        const int64_t row_bytes = 2 * o.stride;
        const bool up = kGated && wave >= kWaves / 2;
        advance = kAlongK ? 2 * kStageSteps : kStageSteps * row_bytes;
        at = kAlongK ? (const char*)o.p + ((up ? rows : 0) + first) * row_bytes + 2 * k0 : (const char*)o.p + k0 * row_bytes + 2 * first;
#pragma unroll
        for (int c = 0; c < kCopies; c++) {
            const int copy = wave * kCopies + c;
            if constexpr (kAlongK) {
                const int row = 64 / kPieces * copy + lane / kPieces, in_half = row - (up ? kRows / 2 : 0);
                const int piece = lane % kPieces ^ first_piece<kPieces>(row);
                const int64_t left = rows - first - 1;
                voff[c] = (uint32_t)(min((int64_t)in_half, left) * row_bytes) + 16 * piece;
            } else {
                constexpr int kLanes = kRows / 8;   // of a step
                const int k = copy * (64 / kLanes) + lane / kLanes;
                const int piece = (lane % kLanes) ^ turned_bits(k);
                const int64_t left = rows - first - 8;
                voff[c] = (uint32_t)(k * row_bytes) + 2 * (uint32_t)min((int64_t)(8 * piece), left);
            }
        }
    }
    // lds: this wavefront's part of the stage
    __device__ void copy(int c, uint32_t lds) const { async_copy16(at, voff[c], lds + c * 1024); }
    // a stage of which only `left` steps are there
    __device__ void copy_some(int c, uint32_t lds, int left, int wave, int lane) const {
        const int copy = wave * kCopies + c;
        const int step = kAlongK ? 8 * (lane % kPieces ^ first_piece<kPieces>(64 / kPieces * copy + lane / kPieces)) : copy * (512 / kRows) + lane / (kRows / 8);
        async_copy16_from(step < left ? (const void*)(at + voff[c]) : (const void*)g_zeros, lds + c * 1024);
    }
};

// Operands of kFrags blocks of 16 rows.  Element e of a lane: row lane % 16 of the block, step 8 (lane / 16) + e.  A read's address is a
// register and a constant: with an addition in front of every one the products of the large tile waited for their turn to be issued.
template <int kRows, bool kAlongK, int kFrags, int kStage, int kStages, int kDeep>
struct Reader {
    static constexpr int kReach = std::min((kStages + 1) / 2, 65536 / kStage), kBases = (kStages + kReach - 1) / kReach;   // stages that a constant of 16 bits reaches over
    static constexpr int kRowBytes = kSteps * kDeep * 2;   // along k
    uint32_t at[kBases][kAlongK ? kDeep : kFrags];
    __device__ void init(uint32_t lds, int first, int lane) {
        const int r = lane & 15, g = lane >> 4;
        if constexpr (kAlongK) {
#pragma unroll
            for (int d = 0; d < kDeep; d++) at[0][d] = lds + (first + r) * kRowBytes + ((4 * d + g) ^ first_piece<4 * kDeep>(r)) * 16;
        } else {
            const int k = 8 * g + (r >> 2);   // and four further
#pragma unroll
            for (int f = 0; f < kFrags; f++) {
                const int piece = (first + 16 * f) / 8 + ((r & 3) >> 1);
                at[0][f] = lds + k * (kRows * 2) + ((piece ^ turned_bits(k)) << 4) + 8 * (r & 1);
            }
        }
#pragma unroll
        for (int f = 0; f < (kAlongK ? kDeep : kFrags); f++) {
            asm("" : "+v"(at[0][f]));
#pragma unroll
            for (int b = 1; b < kBases; b++) {
                at[b][f] = at[0][f] + b * kReach * kStage;
                asm("" : "+v"(at[b][f]));   // kept, not worked out again
            }
        }
    }
    // unit: which 32 steps of the stages.  `jump`: bytes that the block lies further than 16 rows a block would put it
    __device__ uint4 read(int unit, int f, int jump) const {
        const int stage = unit / kDeep, d = unit % kDeep, to = stage % kReach * kStage;
        if constexpr (kAlongK) {
            const product_u32x4 v = *(const __attribute__((address_space(3))) product_u32x4*)(uintptr_t)(at[stage / kReach][d] + (to + f * 16 * kRowBytes + jump));
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            uint2 u[2];
#pragma unroll
            for (int a = 0; a < 2; a++)
                u[a] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) product_s16x4*)(uintptr_t)(
                                                     at[stage / kReach][f] + (to + (d * kSteps + 4 * a) * (kRows * 2)))));
            return make_uint4(u[0].x, u[0].y, u[1].x, u[1].y);
        }
    }
};

template <int kTileM, int kTileN, int kDeep>
constexpr int kStageBytes = (kTileM + kTileN) * kSteps * kDeep * 2;

template <typename T, int kTileM, int kTileN, int kWavesM, int kWavesN, int kStages, int kDeep, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
__global__ void __launch_bounds__(64 * kWavesM * kWavesN, kTileM == 256 || kDeep > 1 ? 1 : 2) tile_kernel(ProductParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr bool kGated = kEpilogue == kGate;
    constexpr int kWaves = kWavesM * kWavesN, kFragsM = kTileM / kWavesM / 16, kFragsN = kTileN / kWavesN / 16;
    constexpr int kStage = kStageBytes<kTileM, kTileN, kDeep>, kStageSteps = kSteps * kDeep, kUnits = kStages * kDeep;
    static_assert(kUnits % 2 == 0, "of operands in registers, which two take turns for");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / kWavesN, wn = wave % kWavesN;
    int tm, tn, share;
    float* sums = work_of<4>(p, kTileM * kTileN, tm, tn, share);
    const int64_t cols = kGated ? p.N / 2 : p.N;
    const int64_t m0 = (int64_t)tm * kTileM, n0 = (int64_t)tn * (kGated ? kTileN / 2 : kTileN);
    const int64_t k0 = share * p.k_share, steps = sums ? min(p.K - k0, p.k_share) : p.K;
    const uint32_t lds = lds_address(smem);
    // One for all rows is asked for now and kept in a scalar register: a load in front of every 16 rows' results, of which a compute unit has eight
    // tiles (2048 x 37888 x 3584), was 25 us of 490.
    [[maybe_unused]] const float power = !kGated && !kAlongKA ? __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(power_of<T, kAlongKA>(p, 0)))) : 1.f;

    using SideA = Side<kTileM, kAlongKA, kWaves, kDeep>;
    using SideB = Side<kTileN, kAlongKB, kWaves, kDeep>;
    SideA a;
    SideB b;
    a.template init<false>(p.a, m0, p.M, k0, wave, lane);
    b.template init<kGated>(p.b, n0, cols, k0, wave, lane);
    Reader<kTileM, kAlongKA, kFragsM, kStage, kStages, kDeep> ra;
    Reader<kTileN, kAlongKB, kFragsN, kStage, kStages, kDeep> rb;
    ra.init(lds, wm * (kTileM / kWavesM), lane);
    rb.init(lds + SideA::kBytes, kGated ? wn * (kTileN / kWavesN / 2) : wn * (kTileN / kWavesN), lane);
    // with the gate, a wavefront's second half of blocks are the up columns of its first
    constexpr int kJump = kGated ? (kTileN / 2 - kTileN / kWavesN / 2) * kStageSteps * 2 : 0;

    // Stages that go through the pipeline, and steps behind them: all, where those are no more than are copied in one go.
    const int whole = steps < kStages * kStageSteps ? 0 : (int)(steps / kStageSteps), left = (int)(steps - (int64_t)whole * kStageSteps);
    constexpr int kCopiesA = SideA::kCopies, kCopies = kCopiesA + SideB::kCopies;
    const uint32_t mine_a = lds + wave * (kCopiesA * 1024), mine_b = lds + SideA::kBytes + wave * (SideB::kCopies * 1024);
    auto copy = [&](int c, uint32_t stage_at) {
        if (c < kCopiesA) a.copy(c, mine_a + stage_at);
        else b.copy(c - kCopiesA, mine_b + stage_at);
    };
    // The stage that is copied next.  Behind the last whole one comes the first again (to nobody's use, where that is where it began).  Few rows
    // wait for the bytes of B, and workgroups that go through its rows side by side ask for the same few channels of memory at a time: they begin
    // in different places (32 x 28672 x 4096: 62.7 -> 55.2 us).  Those that share rows do not: they would miss each other's in the L2 (tiles of
    // 256 x 128, 1024 x 22016 x 4096: 158 us, 290 so; where B's steps are its rows, which all share, 58 -> 67).
    int ahead = kDeep > 1 && kAlongKB && whole > 0 && p.tiles_m == 1 ? (int)(((uint32_t)tn * 2654435761u >> 8) % (uint32_t)whole) : 0;
    const int64_t back_a = (1 - whole) * a.advance, back_b = (1 - whole) * b.advance;
    a.at += ahead * a.advance;
    b.at += ahead * b.advance;
    auto next = [&] {
        const bool last = ahead + 1 >= whole;
        a.at += last ? back_a : a.advance;
        b.at += last ? back_b : b.advance;
        ahead = last ? 0 : ahead + 1;
    };
    f32x4_t acc[kFragsM][kFragsN] = {};
    asm volatile("s_nop 7" ::: "memory");
    uint4 av[2][kFragsM], bv[2][kFragsN];
    constexpr int kReads = kFragsM + kFragsN, kProducts = kFragsM * kFragsN;
    auto read = [&](int n, int buf, int unit) {   // in the order in which the products want them
        if (n == 0) bv[buf][0] = rb.read(unit, 0, 0);
        else if (n <= kFragsM) av[buf][n - 1] = ra.read(unit, n - 1, 0);
        else bv[buf][n - kFragsM] = rb.read(unit, n - kFragsM, n - kFragsM >= kFragsN / 2 ? kJump : 0);
    };
    // The products of the 32 steps whose operands are in registers, and between them the next ones' operands and, of the last of a stage, copies to
    // its place.
    auto step = [&](auto unit_) {
        constexpr int unit = decltype(unit_)::value, next_unit = (unit + 1) % kUnits;
        constexpr bool last = unit % kDeep == kDeep - 1;
        each<kProducts>([&](auto n_) {
            constexpr int n = decltype(n_)::value, j = n / kFragsM, i = n % kFragsM;
            mma<T>(bv[unit % 2][j], av[unit % 2][i], acc[i][j]);
            constexpr int kEarly = kProducts * 3 / 4;
            if constexpr (n < kEarly) {
                constexpr int first = n * kReads / kEarly, end = (n + 1) * kReads / kEarly;
                each<end - first>([&](auto x) { read(first + decltype(x)::value, next_unit % 2, next_unit); });
            }
            constexpr int from = n * kCopies / kProducts, to = last ? (n + 1) * kCopies / kProducts : from;
            each<to - from>([&](auto x) { copy(from + decltype(x)::value, unit / kDeep * kStage); });
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (last) next();
    };
    if (whole > 0) {
        each<kStages>([&](auto st) {
            each<kCopies>([&](auto c) { copy(decltype(c)::value, decltype(st)::value * kStage); });
            next();
        });
        wait_copies<(kStages - 1) * kCopies>();
        __syncthreads();
        each<kReads>([&](auto n) { read(decltype(n)::value, 0, 0); });
        for (int stage = 0; stage < whole; stage += kStages)
            each<kUnits>([&](auto unit) {
                constexpr int u = decltype(unit)::value;
                if (stage + u / kDeep >= whole) return;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if constexpr (u % kDeep == kDeep - 1) {   // everybody has the last of this stage in registers, so it may be copied over, and the next one is there
                    wait_copies<(kStages - 2) * kCopies>();
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                step(unit);
            });
        sums_done(acc);
        wait_copies<0>();
        __syncthreads();
    }
    if (left) {   // stages of which the last may not be whole
        a.at += (whole - ahead) * a.advance;
        b.at += (whole - ahead) * b.advance;
#pragma unroll
        for (int st = 0; st < kStages; st++) {
            if (st * kStageSteps < left) {
#pragma unroll
                for (int c = 0; c < kCopies; c++)
                    if (c < kCopiesA) a.copy_some(c, mine_a + st * kStage, left - st * kStageSteps, wave, lane);
                    else b.copy_some(c - kCopiesA, mine_b + st * kStage, left - st * kStageSteps, wave, lane);
                a.at += a.advance;
                b.at += b.advance;
            }
        }
        wait_copies<0>();
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            if (u * kSteps < left) {
#pragma unroll
                for (int n = 0; n < kReads; n++) read(n, 0, u);
#pragma unroll
                for (int n = 0; n < kProducts; n++) mma<T>(bv[0][n / kFragsM], av[0][n % kFragsM], acc[n % kFragsM][n / kFragsM]);
            }
        }
        sums_done(acc);
    }

    // Accumulator element r of a lane: row lane % 16 of C's block, column 4 (lane / 16) + r.
    const int r16 = lane & 15, c4 = 4 * (lane >> 4);
    const int64_t mw = m0 + wm * (kTileM / kWavesM), nw = n0 + wn * (kGated ? kTileN / kWavesN / 2 : kTileN / kWavesN);
    if (sums) {
        float* to = sums + (int64_t)(wm * (kTileM / kWavesM) + r16) * kTileN + (kGated ? wn * (kTileN / kWavesN / 2) : wn * (kTileN / kWavesN)) + c4;
#pragma unroll
        for (int i = 0; i < kFragsM; i++)
#pragma unroll
            for (int j = 0; j < kFragsN; j++)
                *reinterpret_cast<float4*>(to + 16 * i * kTileN + 16 * j + (kGated && j >= kFragsN / 2 ? kTileN / 2 - kTileN / kWavesN / 2 : 0)) =
                    make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
        return;
    }
    // 16 rows at a time go through the wavefront's part of LDS, so that whole pieces of a row are written at a time.
    __syncthreads();
    constexpr int kBlocks = kGated ? kFragsN / 2 : kFragsN, kPieces = kBlocks * 2, kPitch = kBlocks * 32 + 16;
    unsigned char* mine = smem + wave * (16 * kPitch);
    auto write = [&](int i, auto value, void* out, int64_t stride, int64_t first) {
#pragma unroll
        for (int j = 0; j < kBlocks; j++)
            *reinterpret_cast<uint2*>(mine + r16 * kPitch + (16 * j + c4) * 2) = pack4<T>(value(j, 0), value(j, 1), value(j, 2), value(j, 3));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int x = 0; x < (16 * kPieces + 63) / 64; x++) {
            const int at = x * 64 + lane, row = at / kPieces, piece = at % kPieces;
            const int64_t m = mw + 16 * i + row, n = nw + 8 * piece;
            if (row >= 16 || m >= p.M || n >= cols) continue;
            *reinterpret_cast<uint4*>((T*)out + m * stride + first + n) = *reinterpret_cast<const uint4*>(mine + row * kPitch + piece * 16);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kFragsM; i++) {
        if constexpr (kGated) {
            write(i, [&](int j, int r) { return gate_product(acc[i][j][r], acc[i][j + kBlocks][r]); }, p.out, cols, 0);
            if (p.both) {
                const int64_t m = mw + 16 * i + r16;
#pragma unroll
                for (int j = 0; j < kFragsN; j++) {
                    const int64_t n = nw + 16 * (j % kBlocks) + c4;
                    if (m < p.M && n < cols)
                        *reinterpret_cast<float4*>(p.both + m * p.N + (j < kBlocks ? 0 : cols) + n) = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
                }
            }
        } else {
            const float by = kAlongKA ? power_of<T, kAlongKA>(p, mw + 16 * i + r16) : power;
            write(i, [&](int j, int r) { return times_power<T>(acc[i][j][r], by); }, p.out, p.N, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <typename T, int kTileM, int kTileN, int kStages, int kDeep, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int launch_tiles(const ProductParams& p, const TilePlan& plan, hipStream_t stream) {
    constexpr int kWavesN = kTileN % 64 ? 1 : 2;   // gate and up columns of a wavefront are whole blocks
    auto kernel = tile_kernel<T, kTileM, kTileN, 4 / kWavesN, kWavesN, kStages, kDeep, kAlongKA, kAlongKB, kEpilogue>;
    constexpr int lds = kStages * kStageBytes<kTileM, kTileN, kDeep>;
    if (int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)plan.blocks()), dim3(256), lds, stream, p);
    CKV_HIP_TRY(hipGetLastError());
    return CKV_OK;
}

template <typename T, bool kAlongKA, bool kAlongKB, Epilogue kEpilogue>
int launch_tiles(const ProductParams& p, const TilePlan& plan, hipStream_t stream) {
    if (plan.tile_m == 256 && plan.deep == 1) return launch_tiles<T, 256, 256, 4, 1, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    if (plan.deep == 1) return launch_tiles<T, 128, 128, 4, 1, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    if constexpr (kEpilogue == kGate)
        switch (plan.tile_m * 1000 + plan.tile_n) {
            case 256096: return launch_tiles<T, 256, 96, 3, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 256160: return launch_tiles<T, 256, 160, 3, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 128096: return launch_tiles<T, 128, 96, 5, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 128160: return launch_tiles<T, 128, 160, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 128192: return launch_tiles<T, 128, 192, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 128224: return launch_tiles<T, 128, 224, 3, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 128256: return launch_tiles<T, 128, 256, 3, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 64096: return launch_tiles<T, 64, 96, 7, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 64160: return launch_tiles<T, 64, 160, 5, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 64192: return launch_tiles<T, 64, 192, 5, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 64224: return launch_tiles<T, 64, 224, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
            case 64256: return launch_tiles<T, 64, 256, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
        }
    if constexpr (kAlongKA) {
        if (plan.tile_m == 256) return launch_tiles<T, 256, 128, 3, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
        return plan.tile_m == 128 ? launch_tiles<T, 128, 128, 4, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream)
                                  : launch_tiles<T, 64, 128, 6, 2, kAlongKA, kAlongKB, kEpilogue>(p, plan, stream);
    }
    return CKV_ERR_UNSUPPORTED;
}

// A kind of tile, and microseconds that its workgroups take on a compute unit, `resident` of them at a time: 32 steps, and around the steps.  More
// the more units have one, as the clock falls; no less than the bytes of B take, 5.9 TB/s by whole lines (deep kinds) and 4.6 by halves.  Where B's rows
// lie across k, deep kinds are for rows that fit in a tile, at 0.33 (32 x 4096 x 28672 58 us in eight shares, 82 in four).
struct Kind {
    int tile_m, tile_n, deep, resident;
    double step_us, full_us, around_us, first_us;   // alone, and on all units; first_us: where others hide what is around the steps, once a launch
};
constexpr Kind kKinds[] = {{256, 256, 1, 1, 0.47, 0.74, 8.5, 0}, {128, 128, 1, 2, 0.65, 0.65, 1.0, 8.0},   // of two alike the first is taken
                           {64, 96, 2, 1, 0.10, 0.15, 4.0, 0},   {128, 96, 2, 1, 0.145, 0.20, 4.0, 0},  {256, 96, 2, 1, 0.22, 0.30, 5.0, 0},
                           {64, 128, 2, 1, 0.11, 0.16, 4.0, 0},  {128, 128, 2, 1, 0.13, 0.24, 4.0, 0},  {256, 128, 2, 1, 0.28, 0.37, 5.0, 0},
                           {64, 160, 2, 1, 0.10, 0.36, 5.0, 0},  {128, 160, 2, 1, 0.15, 0.28, 5.0, 0},  {256, 160, 2, 1, 0.36, 0.445, 6.0, 0},
                           {64, 192, 2, 1, 0.12, 0.45, 5.0, 0},  {128, 192, 2, 1, 0.20, 0.33, 5.0, 0},  {64, 256, 2, 1, 0.20, 0.60, 6.0, 0},
                           {128, 256, 2, 1, 0.42, 0.43, 6.0, 0}, {64, 224, 2, 1, 0.14, 0.50, 6.0, 0},   {128, 224, 2, 1, 0.30, 0.36, 6.0, 0}};

}  // namespace

// Tiles fill the compute units round by round; those of the last round may be shared out along k, which costs their sums a trip to memory (4
// TB/s both ways, 3 us the launch that adds them up).  What decides between the kinds is how near the tiles come to full rounds.  128
// rows, 128 high and 96, 128, 160, 192, 224 and 256 wide, each in the best number of shares: 22016 x 4096 43, 46, 51, 47, 48 and 49 us; 28672 x 4096 59, 49,
// 54, 59, 61 and 61; 37888 x 3584 75, 68, 59, 62, 64 and 68; 51200 x 5120 137, 133, 123, 113, 109 and 113.  More rows, 256 high
// and 128, 160 and (32 steps a stage) 256 wide: 256 x 28672 x 4096 62, 66 and 91; 512 x 37888 x 3584 146, 114 and 171; 1024 x 34816 x 5120 340, 307 and
// 376; 4096 x 28672 x 4096 744, 722 and 719.  Over 24 to 4096 rows of ten layers the rule is 0.7 % behind the best kind.
TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus) {
    TilePlan best = {};
    double best_us = 0;
    for (const Kind& kind : kKinds) {
        const bool deep = kind.deep > 1;
        if (deep && (!a_along_k || (!gated && (M > kind.tile_m || kind.tile_n != 128)))) continue;
        const int64_t tiles_m = (M + kind.tile_m - 1) / kind.tile_m, tiles_n = tiles_across(N, kind.tile_n, gated), all = tiles_m * tiles_n;
        const int64_t places = (int64_t)cus * kind.resident, rest = all % places;
        auto time_of = [&](int64_t workgroups, int64_t steps) {   // of that many at a time
            const double bytes_us = (double)std::min(workgroups, places) / tiles_m * kind.tile_n * kSteps * 2 / (deep ? 5.9e6 : 4.6e6);
            const double step_us = deep && !gated ? 0.33 : kind.step_us + (kind.full_us - kind.step_us) * (double)std::min<int64_t>(workgroups, cus) / cus;
            return (double)steps / kSteps * std::max(step_us, bytes_us) + kind.around_us;
        };
        for (int shares = 1; shares <= 8; shares++) {
            // Behind full rounds of products compute units may idle: the others' clock rises (2048 x 37888 x 3584, 4.6 rounds: 457 us, 485 with the
            // rest in three shares), unless it is bytes they wait for, as few rows do.
            if (shares > 1 && (rest == 0 || K / shares < 256 || (!(deep && tiles_m == 1) && all > places))) break;
            const int64_t k_share = shares == 1 ? K : ((K + shares - 1) / shares + 63) / 64 * 64;
            if ((K + k_share - 1) / k_share != shares) continue;
            double rounds = (double)((rest * shares + cus - 1) / cus);
            if (kind.resident > 1)   // they start as others end; one alone on a unit is the faster for it
                rounds = rest * shares <= cus && all < places ? 0.55 : all > places ? (double)rest / places : std::max(1.0, (double)rest * shares / places);
            double us = kind.first_us + (double)(all / places) * time_of(places, K) + rounds * time_of(rest * shares, k_share);
            if (shares > 1) us += 3.0 + (double)(rest * shares) * kind.tile_m * kind.tile_n * 8 / 4e6;
            if (best_us == 0 || us < best_us) {
                best_us = us;
                best = TilePlan{kind.tile_m, kind.tile_n, kind.deep, (int)tiles_m, (int)tiles_n, (int)(all - rest), shares, k_share};
            }
        }
    }
    return best;
}

template <typename T>
int run_tiles(const ProductParams& p, const TilePlan& plan, bool a_along_k, Epilogue epilogue, hipStream_t stream) {
    if (epilogue == kGate) return launch_tiles<T, true, true, kGate>(p, plan, stream);
    if (a_along_k) return launch_tiles<T, true, false, kStore>(p, plan, stream);
    return launch_tiles<T, false, false, kStore>(p, plan, stream);
}
template int run_tiles<__half>(const ProductParams&, const TilePlan&, bool, Epilogue, hipStream_t);
template int run_tiles<__hip_bfloat16>(const ProductParams&, const TilePlan&, bool, Epilogue, hipStream_t);

}  // namespace ckv
