// Products of 16-bit matrices with fp32 sums on the tensor cores (product_tc.cu) and for a few rows (product_rows.cu), as the dense layers of residual networks call them.
#pragma once
#include "residual.cuh"

namespace b200rl {

enum { EPI_FORWARD, EPI_INPUT, EPI_SUM };

// C(m, n) = sum_k A(m, k) B(n, k)
struct Operand {
    const void* p;              // k_rows: element (k, r) at p[k * ld + r] (the operand's rows are columns of the matrix); else (r, k) at p[r * ld + k]
    long long ld;
    bool k_rows;
};
struct Product {
    Operand a, b;
    int m, n, k;
    const float* bias;                          // EPI_FORWARD: out = add + scale act(C + bias), pre = C + bias (where pre is there)
    const void* add; long long ld_add;          // EPI_INPUT: out = act'(pre) (C + add)
    void* pre; long long ld_pre;
    void* out; long long ld_out;                // EPI_SUM: fp32, out (+)= C
    float scale;
    int act;
    int accumulate;
    float* row_sums;                            // EPI_SUM: (+)= sum_k A(m, k), or NULL
};

// bytes of workspace for this product on the tensor cores: partial sums where k is split, copies of operands that TMA cannot address
size_t product_tc_workspace_bytes(const Product& g, int epilogue);
int product_tc(const Product& g, int type, int epilogue, void* workspace, size_t workspace_bytes, cudaStream_t s);
// the forward product of a few rows, without a workspace
bool product_rows_takes(const Product& g);
int product_rows(const Product& g, int type, cudaStream_t s);
int product_tc_error_get(int* word);
int product_tc_error_clear();

}  // namespace b200rl
