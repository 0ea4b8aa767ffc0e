// What the kernels of a matrix product C (M, N) = sum over k of A (m, k) B (n, k) share: their parameters, the order of their tiles.
#pragma once

#include "ckv_common.h"

#include <type_traits>

namespace ckv {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Operand {
    const void* p;
    int64_t stride;    // elements between rows, where a row's elements are adjacent along k, else between steps of k, whose rows are adjacent
};

struct ProductParams {
    Operand a, b;
    void* out;          // (M, N) contiguous, or the gated (M, N / 2)
    float* both;        // gated, optional: (M, N), gate and up columns; of these, not of numbers rounded to the operands' type, gradients are made
    const int* exponents;    // optional, float16 and not gated: C is times 2 to that power; one for each of its rows where A lies along k, else one for all
    float* partial;     // sums of the shares, tile by tile: (tiles shared out, shares, tile rows, tile columns)
    int64_t M, N, K;
    int64_t k_share;    // steps of a share
    int tiles_m, tiles_n;
    int whole_tiles;    // tiles before the first that is shared out
    int shares;
};

enum Epilogue { kStore, kGate };

// What row m of C is times: a power of two, exact until the result is rounded to float16.  One beyond float32's normal numbers is the nearest of them:
// whatever it meets is nothing in float16 or above its end either way.  One for other types.
template <typename T, bool kAlongKA>
__device__ inline float power_of(const ProductParams& p, int64_t m) {
    if constexpr (std::is_same<T, __half>::value)
        return p.exponents && m < p.M ? __int_as_float((min(max(p.exponents[kAlongKA ? m : 0], -126), 127) + 127) << 23) : 1.f;
    else return 1.f;
}
template <typename T>
__device__ inline float times_power(float v, float power) {
    if constexpr (std::is_same<T, __half>::value) return v * power;
    else return v;
}

// Workgroups go round the eight XCDs: each gets a stretch of the tiles, and behind those one of the shares.  Tiles are numbered in bands
// kHigh tiles of M high, so that the tiles of a stretch that run at a time share operands in its L2.
__device__ inline int stretch(int block, int all) {
    const int xcd = block % 8, many = all / 8, over = all % 8;
    return xcd * many + min(xcd, over) + block / 8;
}
template <int kHigh>
__device__ inline void place_of(const ProductParams& p, int tile, int& tm, int& tn) {
    const int band = tile / (kHigh * p.tiles_n), in = tile - band * kHigh * p.tiles_n;
    const int high = min(kHigh, p.tiles_m - band * kHigh);
    tm = band * kHigh + in % high;
    tn = in / high;
}
// This workgroup's tile, its share of it, and, where there are several, where the sums of the share go.
template <int kHigh>
__device__ inline float* work_of(const ProductParams& p, int tile_size, int& tm, int& tn, int& share) {
    const int all = p.tiles_m * p.tiles_n, block = blockIdx.x;
    const bool rest = block >= p.whole_tiles;
    share = 0;
    if (!rest || p.shares == 1) {
        const int first = rest ? p.whole_tiles : 0;
        place_of<kHigh>(p, first + stretch(block - first, rest ? all - first : p.whole_tiles), tm, tn);
        return nullptr;
    }
    const int at = stretch(block - p.whole_tiles, (all - p.whole_tiles) * p.shares);
    share = at % p.shares;
    place_of<kHigh>(p, p.whole_tiles + at / p.shares, tm, tn);
    return p.partial + (int64_t)at * tile_size;
}

// ---- 16-bit operands on the matrix instructions of their type, ckv_product_mfma.hip -------------------------------------------------------
// Sizes and layouts it takes: whole pieces of 16 bytes everywhere (adjacent elements, strides, addresses; C's columns).
struct TilePlan {
    int tile_m, tile_n, deep;   // deep: 64 steps a stage instead of 32
    int tiles_m, tiles_n, whole_tiles, shares;
    int64_t k_share;
    int64_t blocks() const { return whole_tiles + ((int64_t)tiles_m * tiles_n - whole_tiles) * shares; }
    int64_t bytes() const {   // of the shares' sums
        return shares > 1 ? align_up(((int64_t)tiles_m * tiles_n - whole_tiles) * shares * tile_m * tile_n * 4, 256) : 0;
    }
    void fill(ProductParams& p) const {
        p.tiles_m = tiles_m;
        p.tiles_n = tiles_n;
        p.whole_tiles = whole_tiles;
        p.shares = shares;
        p.k_share = k_share;
    }
};
// Gated, a tile's columns are gate and up columns by halves, so there may be tiles with few of either.
inline int64_t tiles_across(int64_t N, int tile_n, bool gated) { return gated ? (N / 2 + tile_n / 2 - 1) / (tile_n / 2) : (N + tile_n - 1) / tile_n; }
TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus);
template <typename T>
int run_tiles(const ProductParams& p, const TilePlan& plan, bool a_along_k, Epilogue epilogue, hipStream_t stream);

}  // namespace ckv
