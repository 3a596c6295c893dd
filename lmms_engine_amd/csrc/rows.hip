// The operators of a layer that work on rows, gfx950: layer norm and RMS norm with their gradients, embedding lookup and the table's gradient,
// dropout.  All of them are bound by memory; everything is computed in fp32 and rounded once.  Sums have a fixed order: no float atomics.
#include <algorithm>

#include "rows.h"

namespace {

constexpr long MOST_THREADS = 0xffffffffL;  // of a launch
inline long up(long v, long m) { return (v + m - 1) / m * m; }

// `count` values (8 at most) at any address; the others are zero.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[8]) {
    if (count >= 8) {
        if constexpr (sizeof(T) == 2) {
            const bf16x8 a = *(const bf16x8_any*)p;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = bf2f(a[e]);
        } else {
            const f32x4 a = *(const f32x4_any*)p, b = *(const f32x4_any*)(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < count ? (float)p[e] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[8]) {
    if (count >= 8) {
        if constexpr (sizeof(T) == 2) {
            bf16x8 a;
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = f2bf(v[e]);
            *(bf16x8_any*)p = a;
        } else {
            *(f32x4_any*)p = f32x4{v[0], v[1], v[2], v[3]};
            *(f32x4_any*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) p[e] = (T)v[e];
    }
}
__device__ __forceinline__ int left(int n, int j) { return n - j < 8 ? n - j : 8; }

// The sum over the four waves of a workgroup, in every thread.  `part` is written again by the next call but one at the earliest: calls
// alternate between two of them, and each has a barrier.
__device__ __forceinline__ float group_sum(float v, float* part) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// ---- norms ------------------------------------------------------------------------------------------
// A workgroup per row, which reads it once for each sum and once more for the result.
template <typename T, bool CENTRED>
__global__ void __launch_bounds__(256) norm_kernel(const muon_hip_norm p) {
    __shared__ float part[2][4];
    const float over = 1.f / p.n;
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T *x = (const T*)p.x + r * p.x_row, *res = p.residual ? (const T*)p.residual + r * p.res_row : nullptr;
        T *y = (T*)p.y + r * p.n, *sum = res ? (T*)p.sum + r * p.n : nullptr;
        float total = 0.f;
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            float v[8], w[8];
            load8(x + j, left(p.n, j), v);
            if (res) {
                load8(res + j, left(p.n, j), w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += w[e];
                store8(sum + j, left(p.n, j), v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) total += (float)(T)v[e];
        }
        const T* s = res ? sum : x;  // (a thread reads what it has written itself)
        const float mean = CENTRED ? group_sum(total, part[0]) * over : 0.f;
        float square = 0.f;
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            float v[8];
            load8(s + j, left(p.n, j), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) square += e < p.n - j ? (v[e] - mean) * (v[e] - mean) : 0.f;
        }
        const float rstd = 1.f / sqrtf(group_sum(square, part[1]) * over + (float)p.eps);
        if (!CENTRED) __syncthreads();  // (one sum a row: the next one writes where this one is read)
        if (p.stats && threadIdx.x == 0) {
            p.stats[r] = rstd;
            if (CENTRED) p.stats[p.rows + r] = mean;
        }
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            float v[8], w[8], b[8];
            load8(s + j, left(p.n, j), v);
            if (p.weight) load8((const T*)p.weight + j, left(p.n, j), w);
            if (p.bias) load8((const T*)p.bias + j, left(p.n, j), b);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = (v[e] - mean) * rstd;
                if (p.weight) v[e] *= w[e];
                if (p.bias) v[e] += b[e];
            }
            store8(y + j, left(p.n, j), v);
        }
    }
}

// A workgroup takes every gridDim-th row and adds to sums of its own, whose columns belong to one thread each.
template <typename T, bool CENTRED>
__global__ void __launch_bounds__(256) norm_grad_kernel(const muon_hip_norm_grad p, float* partials) {
    __shared__ float part[2][4];
    const float over = 1.f / p.n;
    float* dw = p.dweight ? partials + (long)blockIdx.x * p.n : nullptr;
    float* db = p.dbias ? partials + ((p.dweight ? (long)gridDim.x : 0L) + blockIdx.x) * p.n : nullptr;
    bool first = true;
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T *dy = (const T*)p.dy + r * p.dy_row, *s = p.s ? (const T*)p.s + r * p.s_row : dy;
        const float rstd = p.s ? p.stats[r] : 0.f, mean = CENTRED && p.s ? p.stats[p.rows + r] : 0.f;
        float c1 = 0.f, c2 = 0.f;
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            const int count = left(p.n, j);
            float g[8], v[8], w[8];
            load8(dy + j, count, g);
            load8(s + j, count, v);
            if (p.weight) load8((const T*)p.weight + j, count, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float hat = e < count ? (v[e] - mean) * rstd : 0.f;
                if (e < count) {
                    if (dw) dw[j + e] = (first ? 0.f : dw[j + e]) + g[e] * hat;
                    if (db) db[j + e] = (first ? 0.f : db[j + e]) + g[e];
                }
                const float gw = p.weight ? g[e] * w[e] : g[e];
                c1 += gw;
                c2 += gw * hat;
            }
        }
        first = false;
        if (!p.dx) continue;
        c1 = CENTRED ? group_sum(c1, part[0]) * over : 0.f;
        c2 = group_sum(c2, part[1]) * over;
        if (!CENTRED) __syncthreads();
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            const int count = left(p.n, j);
            float g[8], v[8], w[8], d[8];
            load8(dy + j, count, g);
            load8(s + j, count, v);
            if (p.weight) load8((const T*)p.weight + j, count, w);
            if (p.ds) load8((const T*)p.ds + r * p.ds_row + j, count, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gw = p.weight ? g[e] * w[e] : g[e];
                g[e] = rstd * (gw - c1 - (v[e] - mean) * rstd * c2);
                if (p.ds) g[e] += d[e];
            }
            store8((T*)p.dx + r * p.n + j, count, g);
        }
    }
}
// Sixteen rows of threads take the rows of sixteen columns in turn; their sums are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const float* partials, int groups, int n, T* out0, T* out1) {
    __shared__ float part[16][16];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    T* out = blockIdx.y ? out1 : out0;
    for (long j0 = blockIdx.x * 16L; j0 < n; j0 += gridDim.x * 16L) {
        const long j = j0 + x;
        float v = 0.f;
        if (j < n) {
#pragma unroll 4
            for (int c = y; c < groups; c += 16) v += partials[((long)blockIdx.y * groups + c) * n + j];
        }
        part[y][x] = v;
        __syncthreads();
        if (y == 0 && j < n) {
#pragma unroll
            for (int r = 1; r < 16; ++r) v += part[r][x];
            out[j] = (T)v;
        }
        __syncthreads();
    }
}

// ---- embedding --------------------------------------------------------------------------------------
__device__ __forceinline__ long id_at(const void* ids, int wide, long t) { return wide ? ((const long*)ids)[t] : ((const int*)ids)[t]; }

// A workgroup per token.  An id that is none of the table's has a row of NaN: the host cannot be told without waiting for the device.
template <typename T>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbeddingArgs a) {
    for (long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const long id = id_at(a.ids, a.wide, t);
        const bool known = id >= 0 && id < a.vocab;
        for (int j = threadIdx.x * 8; j < a.n; j += 2048) {
            float v[8];
            if (known) load8((const T*)a.rows + id * a.pitch + j, left(a.n, j), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = known ? v[e] * a.scale : __builtin_nanf("");
            store8((T*)a.out + t * a.n + j, left(a.n, j), v);
        }
    }
}
// A workgroup per row of the table, which looks for its tokens among all of them.
template <typename T>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const EmbeddingArgs a) {
    __shared__ int found[256];
    for (long row = blockIdx.x; row < a.vocab; row += gridDim.x) {
        for (int j0 = 0; j0 < a.n; j0 += 2048) {
            const int j = j0 + threadIdx.x * 8;
            float sum[8] = {};
            for (long t0 = 0; t0 < a.tokens && row != a.skip; t0 += 256) {
                const long t = t0 + threadIdx.x;
                __syncthreads();
                found[threadIdx.x] = t < a.tokens && id_at(a.ids, a.wide, t) == row;
                if (!__syncthreads_or(found[threadIdx.x])) continue;
                for (int i = 0; i < 256; ++i) {
                    if (!found[i] || j >= a.n) continue;
                    float v[8];
                    load8((const T*)a.rows + (t0 + i) * a.pitch + j, left(a.n, j), v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[e] += v[e];
                }
            }
            if (j < a.n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] *= a.scale;
                store8((T*)a.out + row * a.n + j, left(a.n, j), sum);
            }
        }
    }
}

// ---- dropout ----------------------------------------------------------------------------------------
// Philox4x32-10: Salmon, Moraes, Dror and Shaw, Parallel random numbers: as easy as 1, 2, 3 (2011).
__device__ __forceinline__ u32x4 philox(u32x4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c[0], b = (uint64_t)0xCD9E8D57u * c[2];
        c = u32x4{(uint32_t)(b >> 32) ^ c[1] ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c[3] ^ k1, (uint32_t)a};
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

// The number of a value is of 32 bits: its upper half is one of the eight of a block of the generator, its lower half, in another block, is
// looked at where the upper one alone does not decide, once in 2^16.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutArgs a) {
    const uint64_t seed = a.seed_at ? *a.seed_at : a.seed;
    const uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    const long blocks = (a.count + 7) / 8;
    for (long b = (long)blockIdx.x * 256 + threadIdx.x; b < blocks; b += (long)gridDim.x * 256) {
        const int count = a.count - b * 8 < 8 ? (int)(a.count - b * 8) : 8;
        float v[8], r[8];
        load8((const T*)a.x + b * 8, count, v);
        if (a.residual) load8((const T*)a.residual + b * 8, count, r);
        u32x4 c{(uint32_t)b, (uint32_t)((uint64_t)b >> 32), a.site, 0};
        const u32x4 upper = philox(c, k0, k1);
        bool keep[8], tie = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = e & 1 ? upper[e / 2] >> 16 : upper[e / 2] & 0xffff;
            keep[e] = h >= a.high;
            tie |= h == a.high;
        }
        if (tie && a.low > 0) {
            c[3] = 1;
            const u32x4 lower = philox(c, k0, k1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t h = e & 1 ? upper[e / 2] >> 16 : upper[e / 2] & 0xffff, l = e & 1 ? lower[e / 2] >> 16 : lower[e / 2] & 0xffff;
                keep[e] = h > a.high || (h == a.high && l >= a.low);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = keep[e] ? v[e] * a.scale : 0.f;
            if (a.residual) v[e] += r[e];
        }
        store8((T*)a.y + b * 8, count, v);
    }
}

inline unsigned grid_of(long groups) { return (unsigned)std::min(groups, MOST_THREADS / 256); }

}  // namespace

hipError_t launch_norm(const muon_hip_norm& p, hipStream_t stream) {
    if (p.rows == 0 || p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    void (*kern)(const muon_hip_norm);
    if (bf) kern = centred ? norm_kernel<bf16_t, true> : norm_kernel<bf16_t, false>;
    else kern = centred ? norm_kernel<float, true> : norm_kernel<float, false>;
    hipLaunchKernelGGL(kern, dim3(grid_of(p.rows)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

long norm_grad_groups(const muon_hip_norm_grad& p, int cus) { return std::min((long)p.rows, 2L * cus); }

hipError_t launch_norm_grad(const muon_hip_norm_grad& p, float* partials, int cus, hipStream_t stream) {
    if (p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    const long groups = norm_grad_groups(p, cus);
    if (groups > 0) {
        void (*kern)(const muon_hip_norm_grad, float*);
        if (bf) kern = centred ? norm_grad_kernel<bf16_t, true> : norm_grad_kernel<bf16_t, false>;
        else kern = centred ? norm_grad_kernel<float, true> : norm_grad_kernel<float, false>;
        hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, stream, p, partials);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    void* out[2] = {p.dweight ? p.dweight : p.dbias, p.dweight ? p.dbias : nullptr};
    if (!out[0]) return hipSuccess;
    const dim3 grid((unsigned)std::min(up(p.n, 16) / 16, 65536L), out[1] ? 2 : 1);
    if (bf) hipLaunchKernelGGL(column_sum_kernel<bf16_t>, grid, dim3(256), 0, stream, partials, (int)groups, p.n, (bf16_t*)out[0], (bf16_t*)out[1]);
    else hipLaunchKernelGGL(column_sum_kernel<float>, grid, dim3(256), 0, stream, partials, (int)groups, p.n, (float*)out[0], (float*)out[1]);
    return hipGetLastError();
}

hipError_t launch_embedding(const EmbeddingArgs& a, hipStream_t stream) {
    if (a.tokens == 0 || a.n == 0) return hipSuccess;
    const unsigned grid = grid_of(a.tokens);
    if (a.dtype == MUON_HIP_BF16) hipLaunchKernelGGL(embedding_kernel<bf16_t>, dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(embedding_kernel<float>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}

long embedding_grad_workspace(int, int, int, int) { return 0; }

hipError_t launch_embedding_grad(const EmbeddingArgs& a, void*, hipStream_t stream) {
    if (a.vocab == 0 || a.n == 0) return hipSuccess;
    const unsigned grid = grid_of(a.vocab);
    if (a.dtype == MUON_HIP_BF16) hipLaunchKernelGGL(embedding_grad_kernel<bf16_t>, dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(embedding_grad_kernel<float>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream) {
    if (a.count == 0) return hipSuccess;
    const unsigned grid = grid_of(up(a.count, 2048) / 2048);
    if (a.dtype == MUON_HIP_BF16) hipLaunchKernelGGL(dropout_kernel<bf16_t>, dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(dropout_kernel<float>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}
