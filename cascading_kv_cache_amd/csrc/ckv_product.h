// What the kernels of a matrix product C (M, N) = sum over k of A (m, k) B (n, k) share: their parameters, the order of their tiles.
#pragma once

#include "ckv_common.h"

namespace ckv {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct Operand {
    const void* p;
    int64_t stride;    // elements between rows, where a row's elements are adjacent along k, else between steps of k, whose rows are adjacent
};

struct ProductParams {
    Operand a, b;
    void* out;          // (M, N) contiguous, or the gated (M, N / 2)
    void* both;         // gated, optional: (M, N), gate and up columns
    float* partial;     // (shares, M, N) where the sums are shared out, else null
    int64_t M, N, K;
    int64_t k_share;    // steps of a share
    int tiles_m, tiles_n;
    bool a_vectors, b_vectors;   // float32 products: operands of whole, aligned pieces of 16 bytes
};

enum Epilogue { kStore, kGate };

__device__ inline float gate_product(float g, float u) { return g / (1.f + expf(-g)) * u; }

// Tiles go round the eight XCDs: each gets a stretch of them, kHigh tiles of M high, so that the tiles of a stretch that run at a time share
// operands in its L2.
template <int kHigh>
__device__ inline void tile_of(const ProductParams& p, int& tm, int& tn) {
    const int all = p.tiles_m * p.tiles_n, xcd = blockIdx.x % 8, many = all / 8, over = all % 8;
    const int tile = xcd * many + min(xcd, over) + blockIdx.x / 8;
    const int band = tile / (kHigh * p.tiles_n), in = tile - band * kHigh * p.tiles_n;
    const int high = min(kHigh, p.tiles_m - band * kHigh);
    tm = band * kHigh + in % high;
    tn = in / high;
}

// ---- 16-bit operands on the matrix instructions of their type, ckv_product_mfma.hip -------------------------------------------------------
// Sizes and layouts it takes: whole pieces of 16 bytes everywhere (adjacent elements, strides, addresses; C's columns).
struct TilePlan {
    int tile_m, tile_n, tiles_m, tiles_n, shares;
    int64_t k_share;
};
TilePlan plan_tiles(int64_t M, int64_t N, int64_t K, bool a_along_k, bool gated, int cus);
// p.partial is set where plan.shares > 1
template <typename T>
int run_tiles(ProductParams& p, const TilePlan& plan, bool a_along_k, bool b_along_k, Epilogue epilogue, hipStream_t stream);

}  // namespace ckv
