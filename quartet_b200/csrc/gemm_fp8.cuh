// What the 8-bit products share.
#pragma once
#include "common.cuh"

namespace quartet {

struct Fp8GemmParams {
    const uint8_t* a_sf;
    const uint8_t* b_sf;
    int64_t M, N;
    int64_t ldd;
    int k_chunks;        // K / 128
    int a_e5m2, b_e5m2;
    float alpha;
    void* d;
    int d_f32;
};

// A product and its operands' codes.
struct Fp8Product {
    const uint8_t *a, *b;
    Fp8GemmParams g;
};
int product_two(const Fp8Product& x, const Fp8Product& y, cudaStream_t s);

// Up to eight rows (gemv_fp8.cu): from codes, or from values that the kernel quantizes.  gemv_fits: whether its shared memory holds them.
bool gemv_fits(int64_t M, int64_t K);
int gemv_fp8_codes(const uint8_t* a, const uint8_t* b, const Fp8GemmParams& g, cudaStream_t s);
int gemv_fp8_values(const void* x, bool f32, int64_t cols, const uint8_t* b, const Fp8GemmParams& g, cudaStream_t s);

}  // namespace quartet
