// Host-side description of the products of layers (product.hip).
#pragma once
#include <hip/hip_runtime.h>
#include "../../include/muon_hip.h"
#include "common.h"

// What becomes of the sums; the codes of include/muon_hip.h.
enum { PRODUCT_LINEAR = 0, PRODUCT_GATED = 1, PRODUCT_SUM = 2, PRODUCT_EACH = 3, PRODUCT_KINDS = 4 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SIGMOID = 2, ACT_SILU = 3, ACT_GELU = 4, ACT_GELU_TANH = 5, ACT_COUNT = 6 };

// An operand whose element (i, l) is base[i * row + l * col]; the second matrix, where the kind has one, has the same strides.
struct ProductOperand {
    const void* base[2];
    long row[2], col[2];
};
struct ProductArgs {
    int kind, dtype, act;
    int m, n, k;
    ProductOperand a, b;
    const void* bias[2];
    const void* residual;
    long res_row, res_col;
    void* out[2];  // m x n, row-major
    void* aux[2];
};

// Bytes of workspace that launch_product needs on a device of `cus` compute units; negative: the sizes are out of range.
long product_workspace(const ProductArgs& p, int cus);
// How launch_product computes it there; false where it cannot.
bool plan_product(const ProductArgs& p, int cus, muon_hip_product_route& out);
hipError_t launch_product(const ProductArgs& p, void* workspace, int cus, int xcd_shift, hipStream_t stream);

// dz0 = dy * d0 (and dz1 = dy * d1) with rows `pitch` elements apart, and the sums over the rows; no factor: dz0 = dy.
struct ActGradArgs {
    int dtype, m, n, factors;
    const void* dy;
    const void* d[2];
    void* dz[2];      // null: sums only
    long pitch;
    void* db[2];      // null: not wanted
    float* partials;  // act_grad_partials(m, n) floats for each factor
};
long act_grad_partials(long m, long n);
bool act_grad_fits(long m, long n);  // whether a launch has workgroups enough
hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t stream);
