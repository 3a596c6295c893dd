// Host-side description of the operators that work on rows: norms, embedding, dropout (rows.hip).
#pragma once
#include <hip/hip_runtime.h>
#include "../../include/muon_hip.h"
#include "common.h"

// How a norm or its gradient is computed on a device of `cus` compute units; each workgroup of a gradient leaves a row behind for each sum over the rows.
muon_hip_norm_route norm_route(int kind, int dtype, int rows, int n, bool backward, int cus);
hipError_t launch_norm(const muon_hip_norm& p, hipStream_t stream);
hipError_t launch_norm_grad(const muon_hip_norm_grad& p, float* partials, int cus, hipStream_t stream);

struct EmbeddingArgs {
    const void* ids;
    int wide;  // ids are 64-bit integers, otherwise 32-bit ones
    int tokens, vocab, n, dtype;
    float scale;
    const void* rows;  // the table, or the incoming gradient
    long pitch;        // elements between its rows
    void* out;
    int skip;  // the id that has no gradient; -1: none
};
hipError_t launch_embedding(const EmbeddingArgs& a, hipStream_t stream);
long embedding_grad_workspace(int tokens, int vocab, int n, int dtype);
hipError_t launch_embedding_grad(const EmbeddingArgs& a, void* workspace, hipStream_t stream);

struct DropoutArgs {
    const void *x, *residual;
    void* y;
    long count;
    int dtype;
    unsigned high, low;  // what is dropped: numbers below high * 2^16 + low, of 32 bits
    float scale;
    unsigned long long seed;
    const unsigned long long* seed_at;  // read instead of `seed`, where not null
    unsigned site;
};
hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream);
