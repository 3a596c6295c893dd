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
// A row is held in the registers of its lanes, 8 to 512 of them: it is read once, its mean is taken before the squares of what is left are
// summed, and no sum of squares cancels.  A lane has CH pieces of 16 bytes, neighbouring lanes neighbouring pieces.  Where a row is no whole number of
// pieces (RAGGED), its last one begins a piece before the row's end: it overlaps the one before, and what it has twice counts once.  Rows at any address.
constexpr int MOST_LANES = 512;  // of a row, and threads of a workgroup: 256 registers each
template <typename T> struct Piece;
template <> struct Piece<bf16_t> {
    static constexpr int V = 8;
    u32x4 raw;
    __device__ __forceinline__ void load(const void* p, unsigned bytes) { raw = __builtin_bit_cast(u32x4, (bf16x8) * (const bf16x8_any*)((const char*)p + bytes)); }
    __device__ __forceinline__ void store(void* p, unsigned bytes) const { *(bf16x8_any*)((char*)p + bytes) = __builtin_bit_cast(bf16x8, raw); }
    __device__ __forceinline__ float operator[](int e) const { return e & 1 ? high_bf16(raw[e / 2]) : low_bf16(raw[e / 2]); }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) raw[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
    }
};
template <> struct Piece<float> {
    static constexpr int V = 4;
    f32x4 raw;
    __device__ __forceinline__ void load(const void* p, unsigned bytes) { raw = *(const f32x4_any*)((const char*)p + bytes); }
    __device__ __forceinline__ void store(void* p, unsigned bytes) const { *(f32x4_any*)((char*)p + bytes) = raw; }
    __device__ __forceinline__ float operator[](int e) const { return raw[e]; }
    __device__ __forceinline__ void set(const float (&v)[4]) { raw = f32x4{v[0], v[1], v[2], v[3]}; }
};

template <int CTRL> __device__ __forceinline__ float moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// v and what lies in the other of two rows (S = 16) or halves (32) of lanes, added.
template <int S> __device__ __forceinline__ float across(float v) {
    const unsigned own = __builtin_bit_cast(unsigned, v);
    const auto r = S == 16 ? __builtin_amdgcn_permlane16_swap(own, own, false, false) : __builtin_amdgcn_permlane32_swap(own, own, false, false);
    const unsigned a = r[0], b = r[1];  // (a cast of a vector's element is one of its first element)
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
// The sum over `lanes` neighbouring lanes (8, 16, 32 or 64), in each of them: exchanges within rows of 16 lanes, then of rows and halves.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    v += moved<0xb1>(v);   // lane ^ 1
    v += moved<0x4e>(v);   // lane ^ 2
    v += moved<0x141>(v);  // the other four of eight
    if (lanes > 8) v += moved<0x140>(v);  // the other eight of sixteen
    if (lanes > 16) v = across<16>(v);
    if (lanes > 32) v = across<32>(v);
    return v;
}
// The same where a row has several waves, of K values at once: waves 0 to lanes / 64 - 1 of each row in `part`.  Calls alternate between two arrays.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], int lanes, float (*part)[8]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lanes_sum(v[k], lanes);
    if (lanes <= 64) return;
    const int wave = threadIdx.x >> 6, waves = lanes >> 6, first = wave & ~(waves - 1);
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) part[k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float t = part[k][first];
        for (int w = 1; w < waves; ++w) t += part[k][first + w];
        v[k] = t;
    }
}

// Where the pieces of a lane are.
template <typename T, int CH, bool RAGGED>
struct Place {
    static constexpr int V = Piece<T>::V;
    int lane, lanes, n;
    __device__ __forceinline__ int begin(int c) const { return (c * lanes + lane) * V; }
    __device__ __forceinline__ bool in(int c) const { return begin(c) < n; }
    __device__ __forceinline__ int at(int c) const { return RAGGED && begin(c) > n - V ? n - V : begin(c); }
    __device__ __forceinline__ unsigned bytes(int c) const { return (unsigned)at(c) * (unsigned)sizeof(T); }
    __device__ __forceinline__ bool counts(int c, int e) const { return in(c) && (!RAGGED || at(c) + e >= begin(c)); }
};

// Which of a workgroup's rows a thread works on.  WIDE rows have whole waves: their addresses are in scalar registers, of which all streams share
// the offsets of the pieces.
template <bool WIDE>
__device__ __forceinline__ int row_of(int shift) {
    const int r = (int)threadIdx.x >> shift;
    return WIDE ? __builtin_amdgcn_readfirstlane(r) : r;
}

template <typename T, bool CENTRED, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(MOST_LANES) norm_kernel(const muon_hip_norm p, int shift) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][1][8];
    const int lanes = 1 << shift;
    const Place<T, CH, RAGGED> at{(int)threadIdx.x & (lanes - 1), lanes, p.n};
    const int each = blockDim.x >> shift;
    for (long r0 = (long)blockIdx.x * each; r0 < p.rows; r0 += (long)gridDim.x * each) {
        const long r = r0 + row_of<WIDE>(shift);
        const bool row = r < p.rows;
        Piece<T> x[CH], res[CH];
        float s[CH][V];
        const T* const px = (const T*)p.x + r * p.x_row;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            x[c].raw = {};
            if (row && at.in(c)) x[c].load(px, at.bytes(c));
        }
        if (p.residual) {
            const T* const pr = (const T*)p.residual + r * p.res_row;
            T* const ps = (T*)p.sum + r * p.n;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                res[c].raw = {};
                if (row && at.in(c)) res[c].load(pr, at.bytes(c));
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = x[c][e] + res[c][e];
                x[c].set(v);
                if (row && at.in(c)) x[c].store(ps, at.bytes(c));
            }
        }
        float mean = 0.f, total[1] = {0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s[c][e] = x[c][e];
                if (CENTRED) total[0] += !RAGGED || at.counts(c, e) ? s[c][e] : 0.f;
            }
        }
        if (CENTRED) {
            row_sum(total, lanes, part[0]);
            mean = total[0] / (float)p.n;  // (a quotient: a row of one value has that one for its mean)
        }
        total[0] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                s[c][e] -= mean;
                if (CENTRED) total[0] += at.counts(c, e) ? s[c][e] * s[c][e] : 0.f;
                else total[0] += !RAGGED || at.counts(c, e) ? s[c][e] * s[c][e] : 0.f;  // (what is not there is zero)
            }
        }
        row_sum(total, lanes, part[1]);
        const float rstd = 1.f / sqrtf(total[0] / (float)p.n + (float)p.eps);
        if (!CENTRED && lanes > 64) __syncthreads();  // (one sum a row: the next one writes where this one is read)
        if (!row) continue;
        if (p.stats && at.lane == 0) {
            p.stats[r] = rstd;
            if (CENTRED) p.stats[p.rows + r] = mean;
        }
        T* const py = (T*)p.y + r * p.n;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!at.in(c)) continue;
            Piece<T> w, b, y;
            float v[V];
            if (p.weight) w.load(p.weight, at.bytes(c));
            if (p.bias) b.load(p.bias, at.bytes(c));
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = s[c][e] * rstd;
                if (p.weight) v[e] *= w[e];
                if (p.bias) v[e] += b[e];
            }
            y.set(v);
            y.store(py, at.bytes(c));
        }
    }
}

// The sums over the rows stay in the registers of a workgroup's lanes until its rows are through, are added up in LDS where several rows were worked on at
// once, and written as one row of `partials`.
template <typename T, bool CENTRED, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(MOST_LANES, CH * Piece<T>::V <= (CENTRED ? 8 : 16) ? 4 : CH * Piece<T>::V <= 16 ? 3 : 2) norm_grad_kernel(const muon_hip_norm_grad p, float* partials, int shift) {
    constexpr int V = Piece<T>::V;
    __shared__ float part[2][2][8];
    extern __shared__ float columns[];
    const int lanes = 1 << shift;
    const Place<T, CH, RAGGED> at{(int)threadIdx.x & (lanes - 1), lanes, p.n};
    const int each = blockDim.x >> shift;
    const float over = 1.f / p.n;
    Piece<T> w[CH];
    float dw[CH][V], db[CH][V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float one[V];
#pragma unroll
        for (int e = 0; e < V; ++e) dw[c][e] = db[c][e] = 0.f, one[e] = 1.f;
        w[c].set(one);
        if (p.weight && at.in(c)) w[c].load(p.weight, at.bytes(c));
    }
    int turn = 0;
    for (long r0 = (long)blockIdx.x * each; r0 < p.rows; r0 += (long)gridDim.x * each) {
        const long r = r0 + row_of<WIDE>(shift);
        const bool row = r < p.rows;
        Piece<T> dy[CH], s[CH], ds[CH];
        const T *const pdy = (const T*)p.dy + r * p.dy_row, *const ps = (const T*)p.s + r * p.s_row, *const pds = (const T*)p.ds + r * p.ds_row;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            dy[c].raw = {};
            s[c].raw = {};
            if (row && at.in(c)) {
                dy[c].load(pdy, at.bytes(c));
                if (p.s) s[c].load(ps, at.bytes(c));
                if (p.ds) ds[c].load(pds, at.bytes(c));
            }
        }
        const float rstd = p.s && row ? p.stats[r] : 0.f, mean = CENTRED && p.s && row ? p.stats[p.rows + r] : 0.f;
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float g = !RAGGED || at.counts(c, e) ? dy[c][e] : 0.f, hat = (s[c][e] - mean) * rstd;
                const float product = !RAGGED || at.counts(c, e) ? g * hat : 0.f;
                dw[c][e] += product;
                if (CENTRED) {
                    db[c][e] += g;
                    sums[0] += g * w[c][e];
                }
                sums[1] += product * w[c][e];
            }
        }
        if (!p.dx) continue;
        if constexpr (CENTRED) row_sum(sums, lanes, part[turn]);
        else {
            float one[1] = {sums[1]};
            row_sum(one, lanes, part[turn]);
            sums[1] = one[0];
        }
        turn ^= 1;
        if (!row) continue;
#pragma unroll
        for (int c = 0; c < CH && sizeof(T) == 2; ++c) {  // unpacked again below, not kept as twice the registers
            asm volatile("" : "+v"(dy[c].raw));
            asm volatile("" : "+v"(s[c].raw));
            asm volatile("" : "+v"(w[c].raw));
        }
        const float c1 = sums[0] * over, c2 = sums[1] * over;
        T* const pdx = (T*)p.dx + r * p.n;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!at.in(c)) continue;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float hat = (s[c][e] - mean) * rstd;
                v[e] = rstd * ((CENTRED ? dy[c][e] * w[c][e] - c1 : dy[c][e] * w[c][e]) - hat * c2);
                if (p.ds) v[e] += ds[c][e];
            }
            dy[c].set(v);
            dy[c].store(pdx, at.bytes(c));
        }
    }
    // what this workgroup has summed: columns of dweight, then those of dbias
    const int waves = lanes < 64 ? 1 : lanes / 64, turns = (blockDim.x >> 6) / waves, mine = (threadIdx.x >> 6) / waves;
    const auto finish = [&](float (&sum)[CH][V], float* out) {
        for (int off = lanes; off < 64; off <<= 1) {  // rows of one wave
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) sum[c][e] += __shfl_xor(sum[c][e], off, 64);
        }
        float* to = turns > 1 ? columns : out;
        for (int t = 0; t < turns; ++t) {
            if (t == mine && (int)(threadIdx.x & 63) < lanes) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (at.counts(c, e)) to[at.at(c) + e] = t ? to[at.at(c) + e] + sum[c][e] : sum[c][e];
            }
            if (turns > 1) __syncthreads();
        }
        if (turns > 1) {
            for (int j = threadIdx.x; j < p.n; j += blockDim.x) out[j] = columns[j];
            __syncthreads();
        }
    };
    if (p.dweight) finish(dw, partials + (long)blockIdx.x * p.n);
    if (CENTRED && p.dbias) finish(db, partials + ((p.dweight ? (long)gridDim.x : 0L) + blockIdx.x) * p.n);
}

// Rows of less than a piece, or longer than the registers of 512 lanes: a workgroup per row, which reads it once for each sum and once more
// for the result.
template <typename T, bool CENTRED>
__global__ void __launch_bounds__(256) norm_streamed_kernel(const muon_hip_norm p) {
    __shared__ float part[2][4];
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
        const float mean = CENTRED ? group_sum(total, part[0]) / (float)p.n : 0.f;
        float square = 0.f;
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            float v[8];
            load8(s + j, left(p.n, j), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) square += e < p.n - j ? (v[e] - mean) * (v[e] - mean) : 0.f;
        }
        const float rstd = 1.f / sqrtf(group_sum(square, part[1]) / (float)p.n + (float)p.eps);
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
__global__ void __launch_bounds__(256) norm_grad_streamed_kernel(const muon_hip_norm_grad p, float* partials) {
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
// Sixty-four rows of threads take the rows of sixteen columns in turn, all of a thread's loads at once where there are 512 rows; their sums are
// added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partials, int groups, int n, T* out0, T* out1) {
    __shared__ float part[64][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    T* out = blockIdx.y ? out1 : out0;
    for (long j0 = blockIdx.x * 16L; j0 < n; j0 += gridDim.x * 16L) {
        const long j = j0 + x;
        float v = 0.f;
        if (j < n) {
#pragma unroll 8
            for (int c = y; c < groups; c += 64) v += partials[((long)blockIdx.y * groups + c) * n + j];
        }
        part[y][x] = v;
        __syncthreads();
        if (y < 4) {
#pragma unroll
            for (int r = 1; r < 16; ++r) v += part[y + 4 * r][x];
            v += __shfl_xor(v, 16, 64);
            v += __shfl_xor(v, 32, 64);
            if (y == 0 && j < n) out[j] = (T)v;
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
// The table's gradient.  The tokens are sorted by id, keeping their order among equal ones, and the sorted tokens cut into chunks of equal length,
// whatever ids are in them: one id may have most of the tokens, as the placeholders of an image do.
//   sort_and_clear  one launch: a workgroup sorts up to 8192 tokens in LDS, the others clear the table meanwhile (151936 x 4096 in bf16 is 1.2 GB, which
//                   takes longer than any of the rest)
//   merge           joins up to 16 sorted lists, where there are more tokens than that: a token's place is its place in its own list and
//                   what binary searches in the other ones say
//   add             a chunk's lanes walk over its tokens: the sum of a run of equal ids is the table's row, or, where the run goes on in a neighbouring
//                   chunk, one of two rows of fp32 that a chunk has for that
//   join            adds those up, in their order.
constexpr int SORT_TOKENS = 8192, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_ROUNDS = SORT_TOKENS / SORT_THREADS;
constexpr int DIGIT_BITS = 7;  // at most; histograms of 128 digits for each of 16 waves
constexpr int MERGE_LISTS = 16;
constexpr int CLEAR_BYTES = SORT_THREADS * 64;  // of a workgroup

struct Sorted {
    int *key, *at;  // ids (vocab: none that counts) in order, and the tokens they are of
};

// A number for each token, among those with its digit, in the order of tokens; LDS arrays of the workgroup.
struct SortSpace {
    uint32_t key[SORT_TOKENS];
    uint16_t at[SORT_TOKENS];
    uint32_t count[(1 << DIGIT_BITS) * SORT_WAVES];  // by digit, then by wave
    uint32_t total[SORT_WAVES];
};
static_assert(sizeof(SortSpace) <= 64 * 1024, "two workgroups to a compute unit");

__device__ void sort_block(const EmbeddingArgs& a, int bits, Sorted out, SortSpace& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = blockIdx.x * SORT_TOKENS, count = a.tokens - first < SORT_TOKENS ? a.tokens - first : SORT_TOKENS;
    const int rounds = (count + SORT_THREADS - 1) / SORT_THREADS;  // of each wave, whose tokens are back to back
    const int passes = (bits + DIGIT_BITS - 1) / DIGIT_BITS, digit_bits = (bits + passes - 1) / passes;
    uint32_t key[SORT_ROUNDS], rank[SORT_ROUNDS];
    uint16_t at[SORT_ROUNDS];
    for (int r = 0; r < rounds; ++r) {
        const int i = (wave * rounds + r) * 64 + lane;
        if (i < count) {
            const long id = id_at(a.ids, a.wide, (long)first + i);
            s.key[i] = id >= 0 && id < a.vocab && id != a.skip ? (uint32_t)id : (uint32_t)a.vocab;
            s.at[i] = (uint16_t)i;
        }
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * digit_bits, digits = 1 << digit_bits;
        for (int i = threadIdx.x; i < digits * SORT_WAVES; i += SORT_THREADS) s.count[i] = 0;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ROUNDS; ++r) {
            const int i = (wave * rounds + r) * 64 + lane;
            const bool in = r < rounds && i < count;
            const uint64_t here = __ballot(in);
            if (here == 0) continue;
            key[r] = in ? s.key[i] : 0;
            at[r] = in ? s.at[i] : (uint16_t)0;
            const uint32_t d = key[r] >> shift & (digits - 1);
            uint64_t same = here;
            for (int b = 0; b < digit_bits; ++b) {
                const uint64_t set = __ballot(d >> b & 1);
                same &= d >> b & 1 ? set : ~set;
            }
            const uint64_t before = same & ((1ull << lane) - 1);
            uint32_t base = 0;
            if (in && before == 0) base = atomicAdd(&s.count[d * SORT_WAVES + wave], (uint32_t)__popcll(same));  // the first of them, for all
            base = __shfl(base, in ? __ffsll((unsigned long long)same) - 1 : lane, 64);
            rank[r] = base + __popcll(before);
        }
        __syncthreads();
        // places of digits and, within a digit, of waves: sums of what stands before, of as many counts in a row by each thread as there are
        const int each = (digits * SORT_WAVES + SORT_THREADS - 1) / SORT_THREADS;
        uint32_t mine = 0;
        for (int e = 0; e < each; ++e) {
            const int i = threadIdx.x * each + e;
            if (i < digits * SORT_WAVES) mine += s.count[i];
        }
        uint32_t upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(upto, off, 64);
            if (lane >= off) upto += o;
        }
        if (lane == 63) s.total[wave] = upto;
        __syncthreads();
        uint32_t place = upto - mine;
        for (int w = 0; w < wave; ++w) place += s.total[w];
        for (int e = 0; e < each; ++e) {
            const int i = threadIdx.x * each + e;
            if (i < digits * SORT_WAVES) {
                const uint32_t c = s.count[i];
                s.count[i] = place;
                place += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < SORT_ROUNDS; ++r) {
            const int i = (wave * rounds + r) * 64 + lane;
            if (r < rounds && i < count) {
                const uint32_t to = s.count[(key[r] >> shift & (digits - 1)) * SORT_WAVES + wave] + rank[r];
                s.key[to] = key[r];
                s.at[to] = at[r];
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < count; i += SORT_THREADS) {
        out.key[first + i] = (int)s.key[i];
        out.at[first + i] = first + s.at[i];
    }
}
template <typename T>
__global__ void __launch_bounds__(SORT_THREADS) embedding_sort_kernel(const EmbeddingArgs a, int sorters, int bits, Sorted out) {
    __shared__ SortSpace space;
    if ((int)blockIdx.x < sorters) {
        sort_block(a, bits, out, space);
        return;
    }
    constexpr int PIECE = 16 / sizeof(T);
    const long values = (long)a.vocab * a.n;
    for (long b = blockIdx.x - sorters; b * (long)(CLEAR_BYTES / sizeof(T)) < values; b += gridDim.x - sorters) {
#pragma unroll
        for (int e = 0; e < CLEAR_BYTES / (SORT_THREADS * 16); ++e) {
            const long i = b * (long)(CLEAR_BYTES / sizeof(T)) + ((long)e * SORT_THREADS + threadIdx.x) * PIECE;
            T* p = (T*)a.out + i;
            if (i + PIECE <= values) *(f32x4_any __attribute__((aligned(2)))*)p = f32x4{0.f, 0.f, 0.f, 0.f};
            else
                for (long k = i; k < values; ++k) ((T*)a.out)[k] = (T)0.f;
        }
    }
}

// Lists of `length` sorted tokens, the last one shorter: every 16 of them become one.
__global__ void __launch_bounds__(256) embedding_merge_kernel(Sorted in, Sorted out, int tokens, int length) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= tokens) return;
    const int key = in.key[i], own = (int)(i / length);
    const int group = own / MERGE_LISTS * MERGE_LISTS;
    const long start = (long)group * length;
    int lo[MERGE_LISTS], size[MERGE_LISTS];
#pragma unroll
    for (int l = 0; l < MERGE_LISTS; ++l) {
        const long rest = tokens - (start + (long)l * length);
        lo[l] = 0;
        size[l] = group + l == own || rest <= 0 ? 0 : rest < length ? (int)rest : length;
    }
    // how many of a list stand before: those with a smaller id, and with the same one where the list stands before the own one
    for (int left = length; left > 0; left >>= 1) {  // more halvings than any list needs
#pragma unroll
        for (int l = 0; l < MERGE_LISTS; ++l) {
            if (size[l] > 0) {
                const int half = size[l] >> 1;
                const int probe = in.key[start + (long)l * length + lo[l] + half];
                const bool below = group + l < own ? probe <= key : probe < key;
                lo[l] = below ? lo[l] + half + 1 : lo[l];
                size[l] = below ? size[l] - half - 1 : half;
            }
        }
    }
    long to = start + (i - (long)own * length);
#pragma unroll
    for (int l = 0; l < MERGE_LISTS; ++l) to += lo[l];
    out.key[to] = key;
    out.at[to] = in.at[i];
}

// How the sorted tokens are cut: `chunk` of them to a group of `lanes` lanes, which takes lanes * 8 columns; `slabs` such pieces make a row.
struct Cut {
    int chunk, chunks, lanes, slabs;
};
template <typename T>
__global__ void __launch_bounds__(256) embedding_add_kernel(const EmbeddingArgs a, Sorted s, Cut c, float* parts) {
    constexpr int AHEAD = 8;
    const int lane = threadIdx.x & (c.lanes - 1);
    const long g = ((long)blockIdx.x * 256 + threadIdx.x) / c.lanes;
    const int slab = (int)(g % c.slabs);
    const long chunk = g / c.slabs;
    const int j = (slab * c.lanes + lane) * 8;
    if (chunk >= c.chunks || j >= a.n) return;
    const int count = left(a.n, j);
    const int first = (int)(chunk * c.chunk), last = a.tokens - first < c.chunk ? a.tokens : first + c.chunk;
    int key = s.key[first];
    const bool goes_on = first > 0 && s.key[first - 1] == key;  // from the chunk before
    bool head = goes_on;
    float sum[8] = {};
    const T* rows = (const T*)a.rows + j;
    for (int t0 = first; t0 < last && key < a.vocab; t0 += AHEAD) {
        float v[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (t0 + u < last) load8(rows + s.at[t0 + u] * a.pitch, count, v[u]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (t0 + u >= last) break;
            const int k = s.key[t0 + u];
            if (k != key) {
                if (key < a.vocab) {
                    if (head) {
                        float* p = parts + (chunk * 2) * a.n + j;
                        store8(p, count, sum);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum[e] *= a.scale;
                        store8((T*)a.out + (long)key * a.n + j, count, sum);
                    }
                }
                head = false;
                key = k;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[u][e];
        }
    }
    if (key >= a.vocab) return;
    const bool tail = last < a.tokens && s.key[last] == key;
    if (head || tail) {
        store8(parts + (chunk * 2 + (head ? 0 : 1)) * a.n + j, count, sum);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] *= a.scale;
        store8((T*)a.out + (long)key * a.n + j, count, sum);
    }
}
// A workgroup for each chunk and slab: where a run begins in the chunk and goes on behind it, its waves take the parts in turn.
constexpr int JOIN_WAVES = 8;
template <typename T>
__global__ void __launch_bounds__(JOIN_WAVES * 64) embedding_join_kernel(const EmbeddingArgs a, Sorted s, Cut c, const float* parts) {
    __shared__ float sums[JOIN_WAVES][64][9];
    const int slabs = (a.n + 511) / 512;
    const int chunk = blockIdx.x / slabs, slab = blockIdx.x % slabs;
    const int first = chunk * c.chunk, next = first + c.chunk;  // (the last chunk has no workgroup)
    const int key = s.key[next - 1];
    if (key >= a.vocab || s.key[next] != key || (s.key[first] == key && first > 0 && s.key[first - 1] == key)) return;
    int lo = next, size = a.tokens - next;  // the end of the run
    while (size > 0) {
        const int half = size >> 1;
        if (s.key[lo + half] <= key) lo += half + 1, size -= half + 1;
        else size = half;
    }
    const int end = (lo - 1) / c.chunk;  // the chunk that it ends in
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = slab * 512 + lane * 8;
    const int count = left(a.n, j);
    float sum[8] = {};
    if (j < a.n) {
        if (wave == 0) load8(parts + (chunk * 2L + 1) * a.n + j, count, sum);
#pragma unroll 4
        for (int p = chunk + 1 + wave; p <= end; p += JOIN_WAVES) {
            float v[8];
            load8(parts + p * 2L * a.n + j, count, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave][lane][e] = sum[e];
    __syncthreads();
    if (wave > 0 || j >= a.n) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        for (int w = 1; w < JOIN_WAVES; ++w) sum[e] += sums[w][lane][e];
        sum[e] *= a.scale;
    }
    store8((T*)a.out + (long)key * a.n + j, count, sum);
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

namespace {
// How rows are laid over lanes: 2^shift of them to a row, `pieces` of 16 bytes to a lane (0: the streamed kernels), `threads` of a workgroup.
struct Layout {
    int shift, pieces, threads;
    bool ragged;
    int rows() const { return pieces ? threads >> shift : 1; }  // that a workgroup works on at once
};
// `best` pieces to a lane at most, unless there are no lanes left, and then `most`.
Layout lay_rows(int dtype, long rows, int n, int threads, int best, int most) {
    const int v = dtype == MUON_HIP_BF16 ? 8 : 4;
    const long count = up(n, v) / v;
    if (n < v || count > (long)MOST_LANES * most) return {8, 0, 256, false};
    Layout l{3, 1, threads, n % v != 0};
    auto lanes = [&] { return 1L << l.shift; };
    // A wave's lanes have one piece each before any has two; more lanes than that where the pieces are too many, or the rows alone too few to
    // fill the machine with waves.
    while (lanes() < count && (lanes() < 64 || (lanes() < MOST_LANES && (lanes() * best < count || rows * lanes() < 256 * 1024)))) ++l.shift;
    while (l.pieces * lanes() < count) l.pieces *= 2;
    l.threads = std::max(threads, (int)lanes());
    return l;
}
template <typename T, bool CENTRED, int CH, bool RAGGED>
auto norm_of(const Layout& l) {
    if constexpr (CH == 1)
        if (l.shift < 6) return norm_kernel<T, CENTRED, CH, RAGGED, false>;
    return norm_kernel<T, CENTRED, CH, RAGGED, true>;
}
template <typename T, bool CENTRED, bool RAGGED>
auto norm_of(const Layout& l) {
    return l.pieces == 1 ? norm_of<T, CENTRED, 1, RAGGED>(l) : l.pieces == 2 ? norm_of<T, CENTRED, 2, RAGGED>(l)
         : l.pieces == 4 ? norm_of<T, CENTRED, 4, RAGGED>(l) : norm_of<T, CENTRED, 8, RAGGED>(l);
}
template <typename T>
auto norm_of(const Layout& l, bool centred) {
    if (centred) return l.ragged ? norm_of<T, true, true>(l) : norm_of<T, true, false>(l);
    return l.ragged ? norm_of<T, false, true>(l) : norm_of<T, false, false>(l);
}
template <typename T, bool CENTRED, int CH, bool RAGGED>
auto norm_grad_of(const Layout& l) {
    if constexpr (CH == 1)
        if (l.shift < 6) return norm_grad_kernel<T, CENTRED, CH, RAGGED, false>;
    return norm_grad_kernel<T, CENTRED, CH, RAGGED, true>;
}
template <typename T, bool CENTRED, bool RAGGED>
auto norm_grad_of(const Layout& l) {
    if constexpr (sizeof(T) == 4 && !CENTRED)
        if (l.pieces == 8) return norm_grad_of<T, CENTRED, 8, RAGGED>(l);
    return l.pieces == 1 ? norm_grad_of<T, CENTRED, 1, RAGGED>(l) : l.pieces == 2 ? norm_grad_of<T, CENTRED, 2, RAGGED>(l) : norm_grad_of<T, CENTRED, 4, RAGGED>(l);
}
template <typename T>
auto norm_grad_of(const Layout& l, bool centred) {
    if (centred) return l.ragged ? norm_grad_of<T, true, true>(l) : norm_grad_of<T, true, false>(l);
    return l.ragged ? norm_grad_of<T, false, true>(l) : norm_grad_of<T, false, false>(l);
}
#ifndef FWD_BEST
#define FWD_BEST 4
#endif
#ifndef BWD_BEST
#define BWD_BEST (p.kind == MUON_HIP_NORM_LAYER ? 8 : 16)
#endif
#ifndef BWD_THREADS
#define BWD_THREADS 512
#endif
#ifndef BWD_PER_CU
#define BWD_PER_CU 2
#endif
Layout lay_grad(const muon_hip_norm_grad& p) {
    const int v = p.dtype == MUON_HIP_BF16 ? 8 : 4;
    return lay_rows(p.dtype, p.rows, p.n, BWD_THREADS, BWD_BEST / v, (p.dtype == MUON_HIP_F32 && p.kind == MUON_HIP_NORM_LAYER ? 16 : 32) / v);
}
long grad_groups_per_cu(const muon_hip_norm_grad& p, const Layout& l) {
    const int values = l.pieces * (p.dtype == MUON_HIP_BF16 ? 8 : 4);
    const int waves = values <= (p.kind == MUON_HIP_NORM_LAYER ? 8 : 16) ? 16 : values <= 16 ? 12 : 8;
    return std::max(1, std::min(BWD_PER_CU * 8, waves) * 64 / l.threads);
}
}  // namespace

hipError_t launch_norm(const muon_hip_norm& p, hipStream_t stream) {
    if (p.rows == 0 || p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    const Layout l = lay_rows(p.dtype, p.rows, p.n, 256, FWD_BEST, 8);
    if (l.pieces == 0) {
        void (*kern)(const muon_hip_norm);
        if (bf) kern = centred ? norm_streamed_kernel<bf16_t, true> : norm_streamed_kernel<bf16_t, false>;
        else kern = centred ? norm_streamed_kernel<float, true> : norm_streamed_kernel<float, false>;
        hipLaunchKernelGGL(kern, dim3(grid_of(p.rows)), dim3(256), 0, stream, p);
        return hipGetLastError();
    }
    const auto kern = bf ? norm_of<bf16_t>(l, centred) : norm_of<float>(l, centred);
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min(up(p.rows, l.rows()) / l.rows(), MOST_THREADS / l.threads)), dim3(l.threads), 0, stream, p, l.shift);
    return hipGetLastError();
}

long norm_grad_groups(const muon_hip_norm_grad& p, int cus) {
    const Layout l = lay_grad(p);
    return std::min(up(p.rows, l.rows()) / l.rows(), grad_groups_per_cu(p, l) * cus);
}

hipError_t launch_norm_grad(const muon_hip_norm_grad& p, float* partials, int cus, hipStream_t stream) {
    if (p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    const long groups = norm_grad_groups(p, cus);
    const Layout l = lay_grad(p);
    if (groups > 0) {
        if (l.pieces == 0) {
            void (*kern)(const muon_hip_norm_grad, float*);
            if (bf) kern = centred ? norm_grad_streamed_kernel<bf16_t, true> : norm_grad_streamed_kernel<bf16_t, false>;
            else kern = centred ? norm_grad_streamed_kernel<float, true> : norm_grad_streamed_kernel<float, false>;
            hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(256), 0, stream, p, partials);
        } else {
            const auto kern = bf ? norm_grad_of<bf16_t>(l, centred) : norm_grad_of<float>(l, centred);
            const size_t lds = l.threads > std::max(1 << l.shift, 64) && (p.dweight || p.dbias) ? (size_t)p.n * 4 : 0;
            hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(l.threads), lds, stream, p, partials, l.shift);
        }
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    void* out[2] = {p.dweight ? p.dweight : p.dbias, p.dweight ? p.dbias : nullptr};
    if (!out[0]) return hipSuccess;
    const dim3 grid((unsigned)std::min(up(p.n, 16) / 16, 65536L), out[1] ? 2 : 1);
    if (bf) hipLaunchKernelGGL(column_sum_kernel<bf16_t>, grid, dim3(1024), 0, stream, partials, (int)groups, p.n, (bf16_t*)out[0], (bf16_t*)out[1]);
    else hipLaunchKernelGGL(column_sum_kernel<float>, grid, dim3(1024), 0, stream, partials, (int)groups, p.n, (float*)out[0], (float*)out[1]);
    return hipGetLastError();
}

hipError_t launch_embedding(const EmbeddingArgs& a, hipStream_t stream) {
    if (a.tokens == 0 || a.n == 0) return hipSuccess;
    const unsigned grid = grid_of(a.tokens);
    if (a.dtype == MUON_HIP_BF16) hipLaunchKernelGGL(embedding_kernel<bf16_t>, dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(embedding_kernel<float>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}

namespace {
// Chunks are as many as fill the machine four waves deep on each of its 1024 SIMDs, and at most 2048, so that the parts of a run over all
// of them are few; at least 8 tokens, which are loaded at once.
Cut cut(int tokens, int n) {
    Cut c;
    for (c.lanes = 8; c.lanes < 64 && c.lanes * 8 < n; c.lanes *= 2) {}
    c.slabs = (int)(up(n, c.lanes * 8) / (c.lanes * 8));
    const long chunks = std::max(1L, std::min(2048L, 4096L * 64 / ((long)c.lanes * c.slabs)));
    c.chunk = (int)std::max(8L, (tokens + chunks - 1) / chunks);
    c.chunks = (tokens + c.chunk - 1) / c.chunk;
    return c;
}
struct Lists {
    Sorted sorted, other;
    float* parts;
    long bytes;
};
Lists lay_out(void* workspace, int tokens, int n) {
    const long list = up(tokens, 64);
    int* p = (int*)workspace;
    Lists l{{p, p + list}, {}, nullptr, 0};
    p += 2 * list;
    if (tokens > SORT_TOKENS) {
        l.other = Sorted{p, p + list};
        p += 2 * list;
    }
    l.parts = (float*)p;
    l.bytes = ((char*)p - (char*)workspace) + 2L * cut(tokens, n).chunks * n * 4;
    return l;
}
}  // namespace

long embedding_grad_workspace(int tokens, int vocab, int n, int) { return tokens == 0 || vocab == 0 || n == 0 ? 0 : lay_out(nullptr, tokens, n).bytes; }

template <typename T>
static hipError_t run_embedding_grad(const EmbeddingArgs& a, void* workspace, hipStream_t stream) {
    const long bytes = (long)a.vocab * a.n * (long)sizeof(T);
    const int sorters = (int)(up(a.tokens, SORT_TOKENS) / SORT_TOKENS);
    int bits = 1;
    while (a.vocab >> bits) ++bits;  // ids and `vocab` itself
    Lists l = lay_out(workspace, a.tokens, a.n);
    const long clear = std::min(up(bytes, CLEAR_BYTES) / CLEAR_BYTES, MOST_THREADS / SORT_THREADS - sorters);
    hipLaunchKernelGGL(embedding_sort_kernel<T>, dim3((unsigned)(sorters + clear)), dim3(SORT_THREADS), 0, stream, a, sorters, bits, l.sorted);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || a.tokens == 0) return e;
    for (long length = SORT_TOKENS; length < a.tokens; length *= MERGE_LISTS) {
        hipLaunchKernelGGL(embedding_merge_kernel, dim3((unsigned)(up(a.tokens, 256) / 256)), dim3(256), 0, stream, l.sorted, l.other, a.tokens, (int)length);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        std::swap(l.sorted, l.other);
    }
    const Cut c = cut(a.tokens, a.n);
    const long lanes = (long)c.chunks * c.slabs * c.lanes;
    hipLaunchKernelGGL(embedding_add_kernel<T>, dim3((unsigned)(up(lanes, 256) / 256)), dim3(256), 0, stream, a, l.sorted, c, l.parts);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || c.chunks == 1) return e;
    hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((unsigned)((c.chunks - 1) * (up(a.n, 512) / 512))), dim3(JOIN_WAVES * 64), 0, stream, a, l.sorted, c, l.parts);
    return hipGetLastError();
}
hipError_t launch_embedding_grad(const EmbeddingArgs& a, void* workspace, hipStream_t stream) {
    if (a.vocab == 0 || a.n == 0) return hipSuccess;
    return a.dtype == MUON_HIP_BF16 ? run_embedding_grad<bf16_t>(a, workspace, stream) : run_embedding_grad<float>(a, workspace, stream);
}

hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream) {
    if (a.count == 0) return hipSuccess;
    const unsigned grid = grid_of(up(a.count, 2048) / 2048);
    if (a.dtype == MUON_HIP_BF16) hipLaunchKernelGGL(dropout_kernel<bf16_t>, dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(dropout_kernel<float>, dim3(grid), dim3(256), 0, stream, a);
    return hipGetLastError();
}
