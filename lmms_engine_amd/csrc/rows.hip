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
// A row is held in the registers of its lanes, 8 to 1024 of them: it is read once, its mean is taken before the squares of what is left are
// summed, and no sum of squares cancels.  A lane has CH pieces of 16 bytes, neighbouring lanes neighbouring pieces.  Where a row is no whole number of
// pieces (RAGGED), its last one begins a piece before the row's end: it overlaps the one before, and what it has twice counts once.  Rows at any address.
//
// Bound by memory.  8192 x 4096 bf16 values: the RMS norm of x + residual, four streams of them, takes 46 us (5.8 TB/s), its gradient, four streams
// too, 46 (5.8 TB/s) and 4 for the last sums of the weight's; a layer norm's 48, 54 and 7.  The same in fp32: 87 (6.2), 112 (4.8) and 5.  262144 rows of 128 bf16
// values (16 lanes each): 27 us (4.9) and 34 (5.9).  Rows of 4090, which begin at any address: an RMS norm 50 and 48, a layer norm 54 and 60.  One row of
// 4096: 3 us.  A large copy reaches 4.9 on the same card.  Asking for the next row before the present one is through changed none of these by more than
// 2 %: there are waves enough to take turns.
constexpr int MOST_LANES = 1024, MOST_WAVES = MOST_LANES / 64;  // of a row
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

// One value, of rows that are shorter than a piece.
template <typename T> struct Single {
    static constexpr int V = 1;
    T raw;
    __device__ __forceinline__ void load(const void* p, unsigned bytes) { raw = *(const T*)((const char*)p + bytes); }
    __device__ __forceinline__ void store(void* p, unsigned bytes) const { *(T*)((char*)p + bytes) = raw; }
    __device__ __forceinline__ float operator[](int) const { return (float)raw; }
    __device__ __forceinline__ void set(const float (&v)[1]) { raw = (T)v[0]; }
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
// Which of a workgroup's rows a thread works on, and as which of the row's lanes.  WIDE rows have whole waves: their addresses are in scalar registers, of
// which all streams share the offsets of the pieces.  Other rows have 8, 16 or 32 lanes.
struct Spot {
    int row, lane;
};
template <bool WIDE> __device__ __forceinline__ Spot spot_of(int lanes) {
    const int t = threadIdx.x;
    if (!WIDE) return {t >> __builtin_ctz(lanes), t & (lanes - 1)};
    const int row = __builtin_amdgcn_readfirstlane(t >> 6) / (lanes >> 6);
    return {row, t - row * lanes};
}
// The same where a row has several waves, of K values at once, by way of LDS.  Calls alternate between two arrays.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], int lanes, int row, float (*part)[MOST_WAVES]) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lanes_sum(v[k], lanes);
    if (lanes <= 64) return;
    const int waves = lanes >> 6, first = row * waves;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) part[k][threadIdx.x >> 6] = v[k];
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
template <typename T, typename P, bool RAGGED>
struct Place {
    static constexpr int V = P::V;
    int lane, lanes, n;
    __device__ __forceinline__ int begin(int c) const { return (c * lanes + lane) * V; }
    __device__ __forceinline__ bool in(int c) const { return begin(c) < n; }
    __device__ __forceinline__ int at(int c) const { return RAGGED && begin(c) > n - V ? n - V : begin(c); }
    __device__ __forceinline__ unsigned bytes(int c) const { return (unsigned)at(c) * (unsigned)sizeof(T); }
    __device__ __forceinline__ bool counts(int c, int e) const { return in(c) && (!RAGGED || at(c) + e >= begin(c)); }
};

template <typename T, typename P, bool CENTRED, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(MOST_LANES / 2) norm_kernel(const muon_hip_norm p, int lanes) {
    constexpr int V = P::V;
    __shared__ float part[2][1][MOST_WAVES];
    const Spot spot = spot_of<WIDE>(lanes);
    const Place<T, P, RAGGED> at{spot.lane, lanes, p.n};
    const int each = blockDim.x / lanes;
    for (long r0 = (long)blockIdx.x * each; r0 < p.rows; r0 += (long)gridDim.x * each) {
        const long r = r0 + spot.row;
        const bool row = r < p.rows;
        constexpr int EARLY = CH <= 2 ? CH : 0;
        P x[CH], res[CH], w[EARLY + 1], b[EARLY + 1];
        float s[CH][V];
        const T* const px = (const T*)p.x + r * p.x_row;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            x[c].raw = {};
            if (row && at.in(c)) x[c].load(px, at.bytes(c));
        }
        // weights are asked for with the row where there is room for them (262144 rows of 128: 10 % less, 4096 x 1024 3 %)
        const auto weights = [&](int c, P& wc, P& bc) {
            if (!row || !at.in(c)) return;
            if (p.weight) wc.load(p.weight, at.bytes(c));
            if (p.bias) bc.load(p.bias, at.bytes(c));
        };
#pragma unroll
        for (int c = 0; c < EARLY; ++c) weights(c, w[c], b[c]);
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
            row_sum(total, lanes, spot.row, part[0]);
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
        row_sum(total, lanes, spot.row, part[1]);
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
            constexpr bool LATE = EARLY == 0;
            P y, &wc = w[LATE ? 0 : c], &bc = b[LATE ? 0 : c];
            float v[V];
            if (LATE) weights(c, wc, bc);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = s[c][e] * rstd;
                if (p.weight) v[e] *= wc[e];
                if (p.bias) v[e] += bc[e];
            }
            y.set(v);
            y.store(py, at.bytes(c));
        }
    }
}

// Waves that a SIMD holds of a gradient with so many values of a row in a lane, by the registers that their sums, one of each value or two, leave; and the
// lanes that a row can have with all of a compute unit's.
constexpr int grad_waves(int values, bool centred) { return values <= 8 && centred ? 5 : values <= 16 && !centred ? 4 : values <= 16 ? 3 : 2; }
constexpr int grad_lanes(int values, bool centred) { return grad_waves(values, centred) >= 4 ? MOST_LANES : 256 * grad_waves(values, centred); }
// The sums over the rows stay in the registers of a workgroup's lanes until its rows are through, are added up in LDS where several rows were worked on at
// once, and written as one row of `partials`.
template <typename T, typename P, bool CENTRED, int CH, bool RAGGED, bool WIDE>
__global__ void __launch_bounds__(grad_lanes(CH * P::V, CENTRED), grad_waves(CH * P::V, CENTRED))
    norm_grad_kernel(const muon_hip_norm_grad p, float* partials, int lanes) {
    constexpr int V = P::V;
    __shared__ float part[2][2][MOST_WAVES];
    extern __shared__ float columns[];
    const Spot spot = spot_of<WIDE>(lanes);
    const Place<T, P, RAGGED> at{spot.lane, lanes, p.n};
    const int each = blockDim.x / lanes;
    const float over = 1.f / p.n;
    P w[CH];
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
        const long r = r0 + spot.row;
        const bool row = r < p.rows;
        P dy[CH], s[CH], ds[CH];
        const T *const pdy = (const T*)p.dy + r * p.dy_row, *const ps = (const T*)p.s + r * p.s_row, *const pds = (const T*)p.ds + r * p.ds_row;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            dy[c].raw = {};
            s[c].raw = {};
            if (row && at.in(c)) {
                dy[c].load(pdy, at.bytes(c));
                s[c].load(ps, at.bytes(c));
                if (p.ds) ds[c].load(pds, at.bytes(c));
            }
        }
        const float rstd = row ? p.stats[r] : 0.f, mean = CENTRED && row ? p.stats[p.rows + r] : 0.f;
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
        if constexpr (CENTRED) row_sum(sums, lanes, spot.row, part[turn]);
        else {
            float one[1] = {sums[1]};
            row_sum(one, lanes, spot.row, part[turn]);
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

// Rows longer than the registers of their lanes hold: a workgroup per row, which reads it once for each sum and once more
// for the result, and, for the sums over rows, a workgroup per block of columns.  Most of what is read again comes from the caches: an RMS norm of
// 1024 x 40000 bf16 values with a residual takes 93 us (3.5 TB/s of four streams), its gradient 101, the sums over rows 25 and 7 more.
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

template <typename T, bool CENTRED>
__global__ void __launch_bounds__(256) norm_grad_streamed_kernel(const muon_hip_norm_grad p) {
    __shared__ float part[2][4];
    const float over = 1.f / p.n;
    for (long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T *dy = (const T*)p.dy + r * p.dy_row, *s = (const T*)p.s + r * p.s_row;
        const float rstd = p.stats[r], mean = CENTRED ? p.stats[p.rows + r] : 0.f;
        float c1 = 0.f, c2 = 0.f;
        for (int j = threadIdx.x * 8; j < p.n; j += 2048) {
            const int count = left(p.n, j);
            float g[8], v[8], w[8];
            load8(dy + j, count, g);
            load8(s + j, count, v);
            if (p.weight) load8((const T*)p.weight + j, count, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gw = p.weight ? g[e] * w[e] : g[e];
                c1 += gw;
                c2 += e < count ? gw * ((v[e] - mean) * rstd) : 0.f;
            }
        }
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
// The sums over the rows of such: a workgroup takes 256 columns (32 threads, eight each) of every `parts`-th eight rows, and leaves its sums in row `part` of
// the partial ones.
template <typename T, bool CENTRED>
__global__ void __launch_bounds__(256) norm_columns_kernel(const muon_hip_norm_grad p, float* partials, int parts) {
    __shared__ float sums[8][32][9];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, slabs = (p.n + 255) / 256;
    const int part = blockIdx.x / slabs, j0 = (blockIdx.x - part * slabs) * 256, j = j0 + tx * 8, count = left(p.n, j);
    float dw[8] = {}, db[8] = {};
    if (j < p.n) {
#pragma unroll 2
        for (long r = part * 8L + ty; r < p.rows; r += parts * 8L) {
            float g[8], v[8];
            load8((const T*)p.dy + r * p.dy_row + j, count, g);
            if (p.dweight) {
                load8((const T*)p.s + r * p.s_row + j, count, v);
                const float rstd = p.stats[r], mean = CENTRED ? p.stats[p.rows + r] : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) dw[e] += e < count ? g[e] * ((v[e] - mean) * rstd) : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) db[e] += g[e];
        }
    }
    const auto finish = [&](const float (&mine)[8], float* out) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[ty][tx][e] = mine[e];
        __syncthreads();
        const int c = threadIdx.x;
        if (j0 + c < p.n) {
            float v = 0.f;
#pragma unroll
            for (int y = 0; y < 8; ++y) v += sums[y][c >> 3][c & 7];
            out[(long)part * p.n + j0 + c] = v;
        }
    };
    if (p.dweight) finish(dw, partials);
    if (p.dbias) finish(db, partials + (p.dweight ? (long)parts * p.n : 0L));
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

// How rows of n values, in pieces of V, are cut: groups of 2^shift lanes with CH pieces each take a segment; `segments` of them make a row.
struct Cut {
    int shift, segments;
};
// A group of lanes for each segment of each token, all of whose loads are under way before the first store: 8192 rows of 4096 bf16 values from a table of
// 151936 take 27 us where a third of them are one id and the others go by rank, 41 where hardly two are alike (3.3 TB/s of results and rows).  The last
// piece of a ragged row overlaps the one before it: what it has twice is written twice.  An id that is none of the table's has a row of NaN: the host
// cannot be told without waiting for the device.
template <typename T, typename P, int CH>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbeddingArgs a, Cut cut) {
    constexpr int V = P::V;
    const int lanes = 1 << cut.shift, lane = threadIdx.x & (lanes - 1);
    const long all = (long)a.tokens * cut.segments, step = (long)gridDim.x * (256 >> cut.shift);
    for (long g = (long)blockIdx.x * (256 >> cut.shift) + (threadIdx.x >> cut.shift); g < all; g += step) {
        const long t = cut.segments == 1 ? g : g / cut.segments;
        const int first = (int)(g - t * cut.segments) * (lanes * CH * V) + lane * V;
        const long id = id_at(a.ids, a.wide, t);
        const bool known = id >= 0 && id < a.vocab;
        const T* const from = (const T*)a.rows + (known ? id : 0L) * a.pitch;
        T* const to = (T*)a.out + t * a.n;
        P v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int j = first + c * lanes * V, at = j > a.n - V ? a.n - V : j;
            if (j < a.n && known) v[c].load(from + at, 0);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int j = first + c * lanes * V, at = j > a.n - V ? a.n - V : j;
            if (j >= a.n) continue;
            if (a.scale != 1.f || !known) {
                float f[V];
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] = known ? v[c][e] * a.scale : __builtin_nanf("");
                v[c].set(f);
            }
            v[c].store(to + at, 0);
        }
    }
}

// The table's gradient.  The tokens are sorted by id, keeping their order among equal ones, and the sorted tokens cut into chunks of equal length,
// whatever ids are in them: one id may have most of the tokens, as the placeholders of an image do.
//   sort    one launch: a workgroup sorts up to 8192 tokens in LDS (27 us: a digit of up to 7 bits at a time, bound by the vector instructions of 16 waves
//           on one compute unit), the others clear the table meanwhile, which for large tables takes longer than any of the rest
//   merge   joins up to 16 sorted lists, where there are more tokens than that: a token's place is its place in its own list and what binary
//           searches in the other ones say (16384 tokens 10 us, 131072 33)
//   add     a chunk's lanes walk over its tokens: the sum of a run of equal ids is the table's row, or, where the run goes on in a neighbouring
//           chunk, one of two rows of fp32 that a chunk has for that
//   join    adds those up, in their order.
// Bound by memory: 8192 tokens into 151936 x 4096 bf16 values take 197 us to clear 1.24 GB (6.3 TB/s; a fill alone 6.9), 35 to add up 67 MB, while the
// memory-side cache still writes back what was cleared (41 where hardly two ids are alike; 268 MB into 32768 rows of a table as large: 108, in whatever order
// and by however many waves), and 6 to join.
constexpr int SORT_TOKENS = 8192, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_ROUNDS = SORT_TOKENS / SORT_THREADS;
constexpr int DIGIT_BITS = 7;  // at most; histograms of 128 digits for each of 16 waves
constexpr int MERGE_LISTS = 16;
constexpr int CLEAR_BYTES = SORT_THREADS * 128;  // of a workgroup

struct Sorted {
    int *key, *at;  // ids (vocab: none that counts) in order, and the tokens they are of
};

struct SortSpace {
    uint32_t key[SORT_TOKENS];
    uint16_t at[SORT_TOKENS];
    uint32_t count[(1 << DIGIT_BITS) * SORT_WAVES];  // by digit, then by wave
    uint32_t total[SORT_WAVES];
};
static_assert(sizeof(SortSpace) <= 64 * 1024, "two workgroups to a compute unit");

// A digit at a time, from the lowest: a wave's tokens are back to back, each counts the ones before it that have its digit, by ballots, and the sums of
// all counts say where each digit's tokens of each wave go.
__device__ void sort_block(const EmbeddingArgs& a, int bits, Sorted out, SortSpace& s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = blockIdx.x * SORT_TOKENS, count = a.tokens - first < SORT_TOKENS ? a.tokens - first : SORT_TOKENS;
    const int rounds = (count + SORT_THREADS - 1) / SORT_THREADS;  // of each wave, whose tokens are back to back
    const int passes = (bits + DIGIT_BITS - 1) / DIGIT_BITS, digit_bits = (bits + passes - 1) / passes;
    uint32_t key[SORT_ROUNDS], moved[SORT_ROUNDS];  // the token in the upper half, its place among those of its digit and wave in the lower one
    long id[SORT_ROUNDS];
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {  // all asked for at once
        const int i = (wave * rounds + r) * 64 + lane;
        id[r] = r < rounds && i < count ? id_at(a.ids, a.wide, (long)first + i) : -1;
    }
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
        const int i = (wave * rounds + r) * 64 + lane;
        if (r >= rounds || i >= count) continue;
        s.key[i] = id[r] >= 0 && id[r] < a.vocab && id[r] != a.skip ? (uint32_t)id[r] : (uint32_t)a.vocab;
        s.at[i] = (uint16_t)i;
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
            const uint32_t token = in ? s.at[i] : 0;
            const uint32_t d = key[r] >> shift & (digits - 1);
            uint32_t low = (uint32_t)here, high = (uint32_t)(here >> 32);  // the lanes with this digit
#pragma unroll
            for (int b = 0; b < DIGIT_BITS; ++b) {
                if (b >= digit_bits) break;
                const uint32_t bit = (uint32_t)((int32_t)(d << (31 - b)) >> 31);  // of all lanes, where this one's is set
                const uint64_t set = __ballot(bit != 0);
                low &= ~((uint32_t)set ^ bit);
                high &= ~((uint32_t)(set >> 32) ^ bit);
            }
            const uint64_t same = (uint64_t)high << 32 | low;
            const uint64_t before = same & ((1ull << lane) - 1);
            uint32_t base = 0;
            if (in && before == 0) base = atomicAdd(&s.count[d * SORT_WAVES + wave], (uint32_t)__popcll(same));  // the first of them, for all
            base = __shfl(base, in ? __ffsll((unsigned long long)same) - 1 : lane, 64);
            moved[r] = token << 16 | (base + __popcll(before));
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
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) place += w < wave ? s.total[w] : 0;
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
                const uint32_t to = s.count[(key[r] >> shift & (digits - 1)) * SORT_WAVES + wave] + (moved[r] & 0xffff);
                s.key[to] = key[r];
                s.at[to] = (uint16_t)(moved[r] >> 16);
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
__global__ void __launch_bounds__(SORT_THREADS, 8) embedding_sort_kernel(const EmbeddingArgs a, int sorters, int bits, Sorted out) {
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

// Lists of `length` sorted tokens, the last one shorter: every 16 of them become one.  A search begins among samples of a list in LDS, so that a
// few of its steps only go to memory, those of all lists at once.
constexpr int MERGE_THREADS = 512, SAMPLES = 256;
static_assert(SORT_TOKENS % SAMPLES == 0, "samples at equal distances");
__global__ void __launch_bounds__(MERGE_THREADS) embedding_merge_kernel(Sorted in, Sorted out, int tokens, int length) {
    __shared__ int sample[MERGE_LISTS][SAMPLES];
    const int first = blockIdx.x * MERGE_THREADS, own = first / length;  // (lists are whole numbers of workgroups long)
    const int group = own / MERGE_LISTS * MERGE_LISTS, step = length / SAMPLES;
    const long start = (long)group * length;
    int size[MERGE_LISTS];
#pragma unroll
    for (int l = 0; l < MERGE_LISTS; ++l) {
        const long rest = tokens - (start + (long)l * length);
        size[l] = group + l == own || rest <= 0 ? 0 : rest < length ? (int)rest : length;
        for (int i = threadIdx.x; i * (long)step < size[l]; i += MERGE_THREADS) sample[l][i] = in.key[start + (long)l * length + i * (long)step];
    }
    __syncthreads();
    const long i = (long)first + threadIdx.x;
    if (i >= tokens) return;
    const int key = in.key[i];
    // how many of a list stand before: those with a smaller id, and with the same one where the list stands before the own one
    const auto below = [&](int l, int other) { return group + l < own ? other <= key : other < key; };
    int lo[MERGE_LISTS];
#pragma unroll
    for (int l = 0; l < MERGE_LISTS; ++l) {
        int at = 0, left = (size[l] + step - 1) / step;
        while (left > 0) {
            const int half = left >> 1;
            if (below(l, sample[l][at + half])) at += half + 1, left -= half + 1;
            else left = half;
        }
        // sample at - 1 stands before, sample `at` does not
        lo[l] = at == 0 ? 0 : (at - 1) * step + 1;
        size[l] = at == 0 ? 0 : (size[l] < at * step ? size[l] : at * step) - lo[l];
    }
    for (int left = step - 1; left > 0; left >>= 1) {
#pragma unroll
        for (int l = 0; l < MERGE_LISTS; ++l) {
            if (size[l] > 0) {
                const int half = size[l] >> 1;
                const bool b = below(l, in.key[start + (long)l * length + lo[l] + half]);
                lo[l] = b ? lo[l] + half + 1 : lo[l];
                size[l] = b ? size[l] - half - 1 : half;
            }
        }
    }
    long to = start + (i - (long)own * length);
#pragma unroll
    for (int l = 0; l < MERGE_LISTS; ++l) to += lo[l];
    out.key[to] = key;
    out.at[to] = in.at[i];
}

// The sorted tokens in `count` chunks of `length`, the last one shorter.
struct Chunks {
    int length, count;
};
// A value of another lane of the group, whose lanes are a whole wave's where it is WIDE.
template <bool WIDE> __device__ __forceinline__ int from_lane(int v, int i) { return WIDE ? __builtin_amdgcn_readlane(v, i) : __shfl(v, i, 64); }
// A group of lanes takes a segment of a chunk's rows.  Ids and places of its next tokens are in the lanes, a token each; AHEAD rows are asked for at once.
template <typename T, typename P, bool WIDE>
__global__ void __launch_bounds__(256) embedding_add_kernel(const EmbeddingArgs a, Sorted s, Chunks c, Cut cut, float* parts) {
    constexpr int V = P::V, AHEAD = 8;
    const int shift = WIDE ? 6 : cut.shift, lanes = 1 << shift, lane = threadIdx.x & (lanes - 1), base = (threadIdx.x & 63) - lane;
    long g = ((long)blockIdx.x * 256 + threadIdx.x) >> shift;
    if (WIDE) g = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long chunk = g / cut.segments;
    if (chunk >= c.count) return;
    const int j = ((int)(g - chunk * cut.segments) * lanes + lane) * V, at = j > a.n - V ? a.n - V : j;
    const bool in = j < a.n;
    const int first = (int)(chunk * c.length), last = a.tokens - first < c.length ? a.tokens : first + c.length;
    const int before = first > 0 ? s.key[first - 1] : -1, behind = last < a.tokens ? s.key[last] : -1;
    int key = s.key[first];
    bool head = before == key;  // the run goes on from the chunk before
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    const auto leave = [&](bool part, int which) {
        if (!in) return;
        if (part) {
            float* const p = parts + (chunk * 2 + which) * a.n + at;
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = sum[e];
        } else {
            P out;
#pragma unroll
            for (int e = 0; e < V; ++e) sum[e] *= a.scale;
            out.set(sum);
            out.store((T*)a.out + (long)key * a.n + at, 0);
        }
    };
    for (int t0 = first; t0 < last && key < a.vocab; t0 += lanes) {
        const int here = last - t0 < lanes ? last - t0 : lanes;  // tokens that the lanes hold
        const int my_key = lane < here ? s.key[t0 + lane] : -1, my_place = lane < here ? s.at[t0 + lane] : 0;
        for (int u0 = 0; u0 < here && key < a.vocab; u0 += AHEAD) {  // (there are 8 lanes at least)
            P row[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const long place = from_lane<WIDE>(my_place, base + u0 + u);
                if (u0 + u < here && in) row[u].load((const T*)a.rows + place * a.pitch + at, 0);
            }
            // all of them are here before the first sum leaves: waits count loads and stores alike, and one behind a store would wait for that too
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) asm volatile("" : "+v"(row[u].raw));
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int k = from_lane<WIDE>(my_key, base + u0 + u);
                if (u0 + u >= here) continue;
                if (k != key) {
                    if (key < a.vocab) leave(head, 0);
                    head = false;
                    key = k;
#pragma unroll
                    for (int e = 0; e < V; ++e) sum[e] = 0.f;
                }
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += row[u][e];
            }
        }
    }
    if (key < a.vocab) leave(head || behind == key, head ? 0 : 1);
}
// A wave for each of eight chunks and 512 columns: where a run begins in the chunk and goes on behind it, its parts are added up, by the wave alone where
// they are few, and by all eight, in turn, where they are many.
constexpr int JOIN_WAVES = 8, JOIN_FEW = 16;
template <typename T>
__global__ void __launch_bounds__(JOIN_WAVES * 64) embedding_join_kernel(const EmbeddingArgs a, Sorted s, Chunks c, const float* parts) {
    __shared__ float sums[JOIN_WAVES][64][9];
    __shared__ int ends[JOIN_WAVES], keys[JOIN_WAVES];
    const int slabs = (a.n + 511) / 512, slab = blockIdx.x % slabs, chunk0 = blockIdx.x / slabs * JOIN_WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = slab * 512 + lane * 8;
    const int count = left(a.n, j), chunk = chunk0 + wave;
    int end = 0, key = 0;  // the chunk that the run ends in, 0: none
    if (chunk + 1 < c.count) {
        const int first = chunk * c.length, next = first + c.length;
        key = s.key[next - 1];
        const int behind = s.key[next], begin = s.key[first], before = first > 0 ? s.key[first - 1] : -1;
        if (key < a.vocab && behind == key && !(begin == key && before == key)) {
            // the last chunk that begins with the id: 64 of them are looked at in one go
            int lo = chunk + 1, size = c.count - lo;
            while (size > 1) {
                const int step = (size + 63) / 64, at = lane * step;
                const uint64_t with = __ballot(at < size && s.key[(long)(lo + at < c.count ? lo + at : lo) * c.length] == key);
                const int most = 63 - __clzll((long long)with);  // (lane 0 looks at one that does)
                lo += most * step;
                size = size - most * step < step ? size - most * step : step;
            }
            end = lo;
        }
    }
    const bool few = end > 0 && end - chunk < JOIN_FEW;
    if (lane == 0) {
        ends[wave] = few ? 0 : end;
        keys[wave] = key;
    }
    float sum[8] = {};
    const auto leave = [&](int id) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] *= a.scale;
        store8((T*)a.out + (long)id * a.n + j, count, sum);
    };
    if (few && j < a.n) {
        load8(parts + (chunk * 2L + 1) * a.n + j, count, sum);
#pragma unroll 4
        for (int p = chunk + 1; p <= end; ++p) {
            float v[8];
            load8(parts + p * 2L * a.n + j, count, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
        leave(key);
    }
    __syncthreads();
    for (int w = 0; w < JOIN_WAVES; ++w) {
        const int upto = ends[w];
        if (upto == 0) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = 0.f;
        if (j < a.n) {
            if (wave == 0) load8(parts + ((chunk0 + w) * 2L + 1) * a.n + j, count, sum);
#pragma unroll 8
            for (int p = chunk0 + w + 1 + wave; p <= upto; p += JOIN_WAVES) {
                float v[8];
                load8(parts + p * 2L * a.n + j, count, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[wave][lane][e] = sum[e];
        __syncthreads();
        if (wave == 0 && j < a.n) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                for (int i = 1; i < JOIN_WAVES; ++i) sum[e] += sums[i][lane][e];
            leave(keys[w]);
        }
        __syncthreads();
    }
}

// ---- dropout ----------------------------------------------------------------------------------------
// Bound by memory: 8192 x 12288 bf16 values take 70 us, 75 behind another pass over them (5.7 and 5.4 TB/s), with a residual 106 (5.7), fp32 values 136
// (5.9).  With one block to a thread three rounds of the generator in place of ten took 9 % less.  Sixteen random bits a value instead of 32 are
// what keeps it bound by memory: a thread draws one block for its eight values.
//
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

// ---- host side ----------------------------------------------------------------------------------------
inline unsigned grid_of(long groups) { return (unsigned)std::min(groups, MOST_THREADS / 256); }

// How rows are laid over lanes: `lanes` of them to a row, `pieces` of 16 bytes to a lane (0: the streamed kernels), `threads` of a workgroup.
struct Layout {
    int lanes, pieces, threads;
    bool ragged;
    int rows() const { return pieces ? threads / lanes : 1; }  // that a workgroup works on at once
};
// Up to `best` pieces to a lane, fewer where the rows alone are too few to fill the machine with waves, more, up to `most`, where there are no lanes left
// of the `limit` for so many pieces.  A row has 8, 16 or 32 lanes, or whole waves, whose number is a power of two where `doubled`.
template <typename Limit>
Layout lay_rows(int dtype, long rows, int n, int threads, int best, int most, bool doubled, const Limit& limit) {
    const int v = dtype == MUON_HIP_BF16 ? 8 : 4;
    const long count = up(n, v) / v;
    const auto lanes_for = [&](int pieces) {
        const long need = up((count + pieces - 1) / pieces, 64);
        long lanes = 64;
        while (doubled && lanes < need) lanes *= 2;
        return std::max(need, lanes);
    };
    const auto fits = [&](int pieces) { return lanes_for(pieces) <= limit(pieces); };
    if (!fits(most)) return {256, 0, 256, false};
    Layout l{8, 1, threads, n > v && n % v != 0};
    if (n < v) return l;  // a value to a lane: 262144 rows of 4 bf16 values take 8.6 us and their gradient 11.3, a workgroup per row 400 and 475
    if (count <= 32) {
        while (l.lanes < count) l.lanes *= 2;
        return l;
    }
    while (l.pieces < best && count > 64L * l.pieces) l.pieces *= 2;
    while (l.pieces > 1 && rows * lanes_for(l.pieces) < 256 * 1024 && fits(l.pieces / 2)) l.pieces /= 2;
    while (!fits(l.pieces)) l.pieces *= 2;
    l.lanes = (int)lanes_for(l.pieces);
    l.threads = l.lanes * std::max(1, threads / l.lanes);
    return l;
}
// Up to four pieces of each row are under way in a lane: 8192 x 4096 bf16 with a residual takes 7 % longer with up to eight, 1 to 2 with two, 6 with one.
// Numbers of waves that are no powers of two, by which gradients gain, lose here: 8192 x 12288 4 %, 8192 x 6144 3 %.
Layout lay_norm(int dtype, long rows, int n) { return lay_rows(dtype, rows, n, 256, 4, 8, true, [](int) { return MOST_LANES / 2; }); }
// A lane of a gradient holds the sums of its columns besides: 16 values of a row at most, of a layer norm, which has two sums, 8, or there are too few waves
// (8192 x 4096 bf16 with a residual: an RMS norm's with 32 values takes 19 % longer, a layer norm's with 16 or 32 22 %).  Rows have as many waves as they need and
// up to all of a compute unit's: layer norms of 8192 x 5120 take 33 % less than with 512 lanes of two pieces, 8192 x 6144 9 %, 8192 x 12288 5 %.
Layout lay_grad(int kind, int dtype, long rows, int n) {
    const int v = dtype == MUON_HIP_BF16 ? 8 : 4;
    const bool layer = kind == MUON_HIP_NORM_LAYER;
    return lay_rows(dtype, rows, n, 512, (layer ? 8 : 16) / v, (layer && dtype == MUON_HIP_BF16 ? 32 : 16) / v, false, [&](int pieces) { return grad_lanes(pieces * v, layer); });
}
// As many workgroups as are at work at once, each of which takes rows until there are none left.  (8192 x 4096 RMS: half as many take 15 % longer,
// twice as many 13 %.)
long grad_groups(int kind, int dtype, long rows, int n, const Layout& l, int cus) {
    // (streamed rows: parts of the sums over columns, of 32 rows at least, and as many as make 2048 workgroups)
    if (l.pieces == 0) return std::min(up(rows, 32) / 32, std::max(1L, std::min(1024L, 2048 / (up(n, 256) / 256))));
    const int waves = 4 * grad_waves(l.pieces * (dtype == MUON_HIP_BF16 ? 8 : 4), kind == MUON_HIP_NORM_LAYER);
    return std::min(up(rows, l.rows()) / l.rows(), (long)std::max(1, waves * 64 / l.threads) * cus);
}
template <typename T, bool CENTRED, int CH, bool RAGGED>
auto norm_of(const Layout& l) {
    if constexpr (CH == 1)
        if (l.lanes < 64) return norm_kernel<T, Piece<T>, CENTRED, CH, RAGGED, false>;
    return norm_kernel<T, Piece<T>, CENTRED, CH, RAGGED, true>;
}
template <typename T, bool CENTRED, bool RAGGED>
auto norm_of(const Layout& l) {
    return l.pieces == 1 ? norm_of<T, CENTRED, 1, RAGGED>(l) : l.pieces == 2 ? norm_of<T, CENTRED, 2, RAGGED>(l)
         : l.pieces == 4 ? norm_of<T, CENTRED, 4, RAGGED>(l) : norm_of<T, CENTRED, 8, RAGGED>(l);
}
template <typename T>
auto norm_of(const Layout& l, int n, bool centred) {
    if (n < Piece<T>::V) return centred ? norm_kernel<T, Single<T>, true, 1, false, false> : norm_kernel<T, Single<T>, false, 1, false, false>;
    if (centred) return l.ragged ? norm_of<T, true, true>(l) : norm_of<T, true, false>(l);
    return l.ragged ? norm_of<T, false, true>(l) : norm_of<T, false, false>(l);
}
template <typename T, bool CENTRED, int CH, bool RAGGED>
auto norm_grad_of(const Layout& l) {
    if constexpr (CH == 1)
        if (l.lanes < 64) return norm_grad_kernel<T, Piece<T>, CENTRED, CH, RAGGED, false>;
    return norm_grad_kernel<T, Piece<T>, CENTRED, CH, RAGGED, true>;
}
template <typename T, bool CENTRED, bool RAGGED>
auto norm_grad_of(const Layout& l) {
    if constexpr (sizeof(T) == 4 || CENTRED)
        if (l.pieces == 4) return norm_grad_of<T, CENTRED, 4, RAGGED>(l);
    return l.pieces == 1 ? norm_grad_of<T, CENTRED, 1, RAGGED>(l) : norm_grad_of<T, CENTRED, 2, RAGGED>(l);
}
template <typename T>
auto norm_grad_of(const Layout& l, int n, bool centred) {
    if (n < Piece<T>::V) return centred ? norm_grad_kernel<T, Single<T>, true, 1, false, false> : norm_grad_kernel<T, Single<T>, false, 1, false, false>;
    if (centred) return l.ragged ? norm_grad_of<T, true, true>(l) : norm_grad_of<T, true, false>(l);
    return l.ragged ? norm_grad_of<T, false, true>(l) : norm_grad_of<T, false, false>(l);
}
}  // namespace

muon_hip_norm_route norm_route(int kind, int dtype, int rows, int n, bool backward, int cus) {
    const Layout l = backward ? lay_grad(kind, dtype, rows, n) : lay_norm(dtype, rows, n);
    const long groups = backward ? grad_groups(kind, dtype, rows, n, l, cus) : std::min(up(rows, l.rows()) / l.rows(), MOST_THREADS / l.threads);
    return muon_hip_norm_route{l.lanes, l.pieces, l.ragged, l.threads, groups};
}

hipError_t launch_norm(const muon_hip_norm& p, hipStream_t stream) {
    if (p.rows == 0 || p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    const Layout l = lay_norm(p.dtype, p.rows, p.n);
    if (l.pieces == 0) {
        void (*kern)(const muon_hip_norm);
        if (bf) kern = centred ? norm_streamed_kernel<bf16_t, true> : norm_streamed_kernel<bf16_t, false>;
        else kern = centred ? norm_streamed_kernel<float, true> : norm_streamed_kernel<float, false>;
        hipLaunchKernelGGL(kern, dim3(grid_of(p.rows)), dim3(256), 0, stream, p);
        return hipGetLastError();
    }
    const auto kern = bf ? norm_of<bf16_t>(l, p.n, centred) : norm_of<float>(l, p.n, centred);
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min(up(p.rows, l.rows()) / l.rows(), MOST_THREADS / l.threads)), dim3(l.threads), 0, stream, p, l.lanes);
    return hipGetLastError();
}

hipError_t launch_norm_grad(const muon_hip_norm_grad& p, float* partials, int cus, hipStream_t stream) {
    if (p.n == 0) return hipSuccess;
    const bool bf = p.dtype == MUON_HIP_BF16, centred = p.kind == MUON_HIP_NORM_LAYER;
    const Layout l = lay_grad(p.kind, p.dtype, p.rows, p.n);
    const long groups = grad_groups(p.kind, p.dtype, p.rows, p.n, l, cus);
    if (groups > 0) {
        if (l.pieces == 0 || !p.s) {  // (sums of a bias alone read nothing else)
            void (*row_kern)(const muon_hip_norm_grad);
            void (*column_kern)(const muon_hip_norm_grad, float*, int);
            if (bf) row_kern = centred ? norm_grad_streamed_kernel<bf16_t, true> : norm_grad_streamed_kernel<bf16_t, false>;
            else row_kern = centred ? norm_grad_streamed_kernel<float, true> : norm_grad_streamed_kernel<float, false>;
            if (bf) column_kern = centred ? norm_columns_kernel<bf16_t, true> : norm_columns_kernel<bf16_t, false>;
            else column_kern = centred ? norm_columns_kernel<float, true> : norm_columns_kernel<float, false>;
            if (p.dx) hipLaunchKernelGGL(row_kern, dim3(grid_of(p.rows)), dim3(256), 0, stream, p);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            if (p.dweight || p.dbias)
                hipLaunchKernelGGL(column_kern, dim3((unsigned)(groups * (up(p.n, 256) / 256))), dim3(256), 0, stream, p, partials, (int)groups);
        } else {
            const auto kern = bf ? norm_grad_of<bf16_t>(l, p.n, centred) : norm_grad_of<float>(l, p.n, centred);
            const size_t lds = l.threads > std::max(l.lanes, 64) && (p.dweight || p.dbias) ? (size_t)p.n * 4 : 0;
            hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(l.threads), lds, stream, p, partials, l.lanes);
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

namespace {
// Lanes for a row of n values in pieces of v, at least 8 and at most `most`, with `pieces` each.
Cut cut_row(int n, int v, int pieces, int most) {
    Cut c{3, 1};
    while ((1 << c.shift) < most && (1L << c.shift) * v * pieces < n) ++c.shift;
    const long each = (1L << c.shift) * v * pieces;
    c.segments = (int)(up(n, each) / each);
    return c;
}
template <typename T, typename P, int CH>
hipError_t run_embedding(const EmbeddingArgs& a, hipStream_t stream) {
    const Cut c = cut_row(a.n, P::V, CH, 64);
    const long groups = (long)a.tokens * c.segments, each = 256 >> c.shift;
    hipLaunchKernelGGL((embedding_kernel<T, P, CH>), dim3(grid_of(up(groups, each) / each)), dim3(256), 0, stream, a, c);
    return hipGetLastError();
}
template <typename T>
hipError_t run_embedding(const EmbeddingArgs& a, hipStream_t stream) {
    if (a.n < Piece<T>::V) return run_embedding<T, Single<T>, 1>(a, stream);
    // few tokens are spread over more lanes
    if ((long)a.tokens * a.n < 1 << 20) return run_embedding<T, Piece<T>, 1>(a, stream);
    return run_embedding<T, Piece<T>, 4>(a, stream);
}
}  // namespace

hipError_t launch_embedding(const EmbeddingArgs& a, hipStream_t stream) {
    if (a.tokens == 0 || a.n == 0) return hipSuccess;
    return a.dtype == MUON_HIP_BF16 ? run_embedding<bf16_t>(a, stream) : run_embedding<float>(a, stream);
}

namespace {
// Chunks are as many as fill the machine two waves deep on each of its 1024 SIMDs, and at most 1024, so that the parts of a run over all of them
// are few (four waves deep 1 % slower at 8192 tokens of 4096 values, the same elsewhere); at least 8 tokens, whose rows are asked for at once.
Cut cut_sums(int n, int dtype) {
    const int v = dtype == MUON_HIP_BF16 ? 8 : 4;
    return cut_row(n, n < v ? 1 : v, 1, 64);
}
Chunks chunks_of(int tokens, int n, int dtype) {
    const Cut cut = cut_sums(n, dtype);
    const long chunks = std::max(1L, std::min(1024L, 2048L * 64 / ((long)cut.segments << cut.shift)));
    Chunks c;
    c.length = (int)std::max(8L, (tokens + chunks - 1) / chunks);
    c.count = (tokens + c.length - 1) / c.length;
    return c;
}
struct Lists {
    Sorted sorted, other;
    float* parts;
    long bytes;
};
Lists lay_out(void* workspace, int tokens, int n, int dtype) {
    const long list = up(tokens, 64);
    int* p = (int*)workspace;
    Lists l{{p, p + list}, {}, nullptr, 0};
    p += 2 * list;
    if (tokens > SORT_TOKENS) {
        l.other = Sorted{p, p + list};
        p += 2 * list;
    }
    l.parts = (float*)p;
    l.bytes = ((char*)p - (char*)workspace) + 2L * chunks_of(tokens, n, dtype).count * n * 4;
    return l;
}
}  // namespace

long embedding_grad_workspace(int tokens, int vocab, int n, int dtype) {
    return tokens == 0 || vocab == 0 || n == 0 ? 0 : lay_out(nullptr, tokens, n, dtype).bytes;
}

template <typename T>
static hipError_t run_embedding_grad(const EmbeddingArgs& a, void* workspace, hipStream_t stream) {
    const long bytes = (long)a.vocab * a.n * (long)sizeof(T);
    const int sorters = (int)(up(a.tokens, SORT_TOKENS) / SORT_TOKENS);
    int bits = 1;
    while (a.vocab >> bits) ++bits;  // ids and `vocab` itself
    Lists l = lay_out(workspace, a.tokens, a.n, a.dtype);
    const long clear = std::min(up(bytes, CLEAR_BYTES) / CLEAR_BYTES, MOST_THREADS / SORT_THREADS - sorters);
    hipLaunchKernelGGL(embedding_sort_kernel<T>, dim3((unsigned)(sorters + clear)), dim3(SORT_THREADS), 0, stream, a, sorters, bits, l.sorted);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || a.tokens == 0) return e;
    for (long length = SORT_TOKENS; length < a.tokens; length *= MERGE_LISTS) {
        hipLaunchKernelGGL(embedding_merge_kernel, dim3((unsigned)(up(a.tokens, MERGE_THREADS) / MERGE_THREADS)), dim3(MERGE_THREADS), 0, stream, l.sorted, l.other, a.tokens, (int)length);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        std::swap(l.sorted, l.other);
    }
    const Chunks c = chunks_of(a.tokens, a.n, a.dtype);
    const Cut cut = cut_sums(a.n, a.dtype);
    const long lanes = ((long)c.count * cut.segments) << cut.shift;
    const auto kern = a.n < Piece<T>::V ? embedding_add_kernel<T, Single<T>, false>
                    : cut.shift < 6     ? embedding_add_kernel<T, Piece<T>, false>
                                        : embedding_add_kernel<T, Piece<T>, true>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(up(lanes, 256) / 256)), dim3(256), 0, stream, a, l.sorted, c, cut, l.parts);
    if (hipError_t e = hipGetLastError(); e != hipSuccess || c.count == 1) return e;
    hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((unsigned)(up(c.count - 1, JOIN_WAVES) / JOIN_WAVES * (up(a.n, 512) / 512))), dim3(JOIN_WAVES * 64), 0, stream, a,
                       l.sorted, c, l.parts);
    return hipGetLastError();
}
hipError_t launch_embedding_grad(const EmbeddingArgs& a, void* workspace, hipStream_t stream) {
    if (a.vocab == 0 || a.n == 0) return hipSuccess;
    return a.dtype == MUON_HIP_BF16 ? run_embedding_grad<bf16_t>(a, workspace, stream) : run_embedding_grad<float>(a, workspace, stream);
}

hipError_t launch_dropout(const DropoutArgs& a, hipStream_t stream) {
    if (a.count == 0) return hipSuccess;
    // A block of eight values to a thread, and two of them, half of the tensor apart, where bf16 values fill the machine many times over: 8192 x 12288 take 7 %
    // less, with a residual 2 %; fp32 values, of which a thread has twice the bytes, lose 3 %, four blocks 2 %.
    const long each = a.dtype == MUON_HIP_BF16 && a.count >= 1L << 24 ? 4096 : 2048;
    const auto kern = a.dtype == MUON_HIP_BF16 ? dropout_kernel<bf16_t> : dropout_kernel<float>;
    hipLaunchKernelGGL(kern, dim3(grid_of(up(a.count, each) / each)), dim3(256), 0, stream, a);
    return hipGetLastError();
}
