// Products of layers on gfx950: out[i][j] = sum_l a[i][l] b[j][l] with the layer's own arithmetic in the epilogue.
//
//   LINEAR  out = act(a b^T + bias) + residual, and act'(.) for the backward pass where it is asked for
//   GATED   g = a b0^T + bias0, u = a b1^T + bias1, out = act(g) u, and act(g), u act'(g) for the backward pass: both products in one
//           kernel, a tile holds the same columns of g and u
//   SUM     out = a0 b0^T + a1 b1^T (the gradient of a gated pair's input): one reduction that runs over both products
//   EACH    out0 = a0 b0^T, out1 = a1 b0^T (the gradients of its weights): the tiles of both in one launch
//
// Operands may lie with the reduction index contiguous (rows of x and W in a forward pass) or with the other index contiguous (W in the
// gradient of the input, x and dz in that of the weight): the kernel reads both as they lie, so nothing is transposed in memory.  Anything
// else is packed into rows of whole 16-byte pieces first.
//
// bf16 operands are multiplied by v_mfma_f32_16x16x32_bf16, fp32 ones by v_mfma_f32_16x16x4_f32 (full single precision); sums, biases,
// activations and residuals are fp32, and results are rounded once.
#include <atomic>
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "gemm_nt.h"
#include "product.h"

namespace {

typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// s_waitcnt with only vmcnt set: vmcnt is split over bits [3:0] and [15:14] (N < 64)
#define WAIT_VM(N) __builtin_amdgcn_s_waitcnt(0x0F70 | ((N) & 15) | (((N) >> 4) << 14))

constexpr int ROWB = 128;  // bytes of a k-tile per row of an operand: 64 bf16 or 32 fp32 values

template <typename T>
struct Elem;
template <>
struct Elem<bf16_t> {
    static constexpr int BK = 64, PIECE = 8;  // reduction steps of a k-tile, values in 16 bytes
    typedef bf16x8 frag;
};
template <>
struct Elem<float> {
    static constexpr int BK = 32, PIECE = 4;
    typedef f32x4 frag;
};

struct KernelArgs {
    const void* a[2];
    const void* b[2];
    long pitch_a, pitch_b;  // elements between rows (reduction index contiguous) or between reduction steps (the other one contiguous)
    int m, n, k;
    int nk, segments;       // k-tiles of one product, products that are summed
    int splits, per_split;  // parts of the k-tiles, k-tiles of each
    int tiles_m, tiles_n, outs;
    int act;
    const void* bias[2];
    const void* residual;
    long res_row, res_col;
    void* out[2];
    void* aux[2];
    float* partial;  // [split][out or factor][m][n], null: one part
    int vec;         // rows of out, aux and partial are whole 16-byte pieces
    int vec_res;
    int xcd_shift;
};

// ---- activations -----------------------------------------------------------------------------
// act(z) and act'(z).  The factor of a gated pair's gradient and the activation itself come out of one evaluation.
//
// Results of bf16 tensors are rounded to 8 bits, so theirs take the hardware's exponential and reciprocal (one step of fp32 each), and the
// complementary error function by the rational approximation 7.1.26 of Abramowitz and Stegun, off by 1.5e-7 at most: 8192 x
// 4096 x 4096 with silu take 196 us (178 without), with the full functions 217.  fp32 tensors get those.
struct ActPair {
    float a, d;
};
template <bool FAST>
__device__ __forceinline__ float exp_of(float z) {
    return FAST ? __builtin_amdgcn_exp2f(1.4426950408889634f * z) : expf(z);
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_of(float z) {
    const float e = 1.0f + exp_of<FAST>(-z);
    return FAST ? __builtin_amdgcn_rcpf(e) : 1.0f / e;
}
template <bool FAST>
__device__ __forceinline__ ActPair activate(int act, float z) {
    switch (act) {
        case ACT_RELU: return ActPair{z <= 0.f ? 0.f : z, z <= 0.f ? 0.f : 1.f};  // (NaN stays NaN)
        case ACT_SIGMOID: {
            const float s = sigmoid_of<FAST>(z);
            return ActPair{s, s * (1.f - s)};
        }
        case ACT_SILU: {
            const float s = sigmoid_of<FAST>(z);
            return ActPair{z * s, s * (1.f + z * (1.f - s))};
        }
        case ACT_GELU: {  // z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2: no cancellation at the lower end
            const float gauss = exp_of<FAST>(-0.5f * z * z);
            float phi;
            if constexpr (FAST) {
                const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678f * fabsf(z));
                const float lower = 0.5f * gauss * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
                phi = z < 0.f ? lower : 1.f - lower;
            } else {
                phi = 0.5f * erfcf(-0.70710678118654752f * z);
            }
            return ActPair{z * phi, phi + z * 0.3989422804014327f * gauss};
        }
        case ACT_GELU_TANH: {  // (1 + tanh y) / 2 = sigmoid(2 y), y = c (z + 0.044715 z^3)
            const float c2 = 2.f * 0.7978845608028654f, q = 0.044715f * z * z;
            const float s = sigmoid_of<FAST>(c2 * z * (1.f + q)), w = s * (1.f - s);
            return ActPair{z * s, s + (w == 0.f ? 0.f : z * w * (c2 * (1.f + 3.f * q)))};
        }
        default: return ActPair{z, 1.f};
    }
}

// ---- eight values of a row ----------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void load8(const T* p, long step, bool whole, int count, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        if (whole) {
            const bf16x8 w = *(const bf16x8*)p;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = bf2f(w[e]);
            return;
        }
    } else {
        if (whole) {
            const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = lo[e], v[e + 4] = hi[e];
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? (float)p[e * step] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool whole, int count, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        if (whole) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
            *(u32x4*)p = w;
            return;
        }
    } else {
        if (whole) {
            *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
            *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
            return;
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = (T)v[e];
}

// The layer's arithmetic on eight sums of row i, columns j .. j + 7 (of both factors of a gated pair), and their way to memory.
template <typename T, bool GATED>
__device__ __forceinline__ void finish8(const KernelArgs& g, int z, long i, int j, float (&v)[8], float (&u)[8]) {
    const int count = g.n - j < 8 ? g.n - j : 8;
    const bool whole = g.vec && count == 8;
    const long at = i * g.n + j;
    if constexpr (GATED) {
        if (g.bias[0]) {
            float b[8];
            load8((const T*)g.bias[0] + j, 1, false, count, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b[e];
        }
        if (g.bias[1]) {
            float b[8];
            load8((const T*)g.bias[1] + j, 1, false, count, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] += b[e];
        }
        float h[8], s[8], t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const ActPair p = activate<sizeof(T) == 2>(g.act, v[e]);
            h[e] = p.a * u[e];
            s[e] = p.a;
            t[e] = p.d * u[e];
        }
        store8((T*)g.out[0] + at, whole, count, h);
        if (g.aux[0]) {
            // Rounded once each to the tensors' type, like the activations that any layer keeps: the backward pass multiplies them by the
            // incoming gradient and nothing else, one rounding less than from g and u themselves.
            store8((T*)g.aux[0] + at, whole, count, s);
            store8((T*)g.aux[1] + at, whole, count, t);
        }
    } else {
        if (g.bias[0]) {
            float b[8];
            load8((const T*)g.bias[0] + j, 1, false, count, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b[e];
        }
        if (g.act != ACT_NONE) {
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const ActPair p = activate<sizeof(T) == 2>(g.act, v[e]);
                v[e] = p.a;
                d[e] = p.d;
            }
            if (g.aux[0]) store8((T*)g.aux[0] + at, whole, count, d);
        }
        if (g.residual) {
            float r[8];
            load8((const T*)g.residual + i * g.res_row + j * g.res_col, g.res_col, g.vec_res && count == 8, count, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        store8((T*)g.out[z] + at, whole, count, v);
    }
}

// Eight sums on their way: to the parts of a split reduction, or through the layer's arithmetic.
template <typename T, bool GATED>
__device__ __forceinline__ void emit8(const KernelArgs& g, int split, int z, long i, int j, float (&v)[8], float (&u)[8]) {
    if (!g.partial) {
        finish8<T, GATED>(g, z, i, j, v, u);
        return;
    }
    const int parts = GATED ? 2 : g.outs, count = g.n - j < 8 ? g.n - j : 8;
    float* p = g.partial + (((long)split * parts + z) * g.m + i) * g.n + j;
    store8(p, g.vec && count == 8, count, v);
    if (GATED) store8(p + (long)g.m * g.n, g.vec && count == 8, count, u);
}

// ---- operand tiles in LDS -------------------------------------------------------------------------
// A k-tile of an operand of R rows takes R * 128 bytes, in one of two orders:
//   rows   row r holds its 8 pieces of 16 bytes; piece c lies at place c ^ swizzle(r)
//   steps  reduction step k holds R values; 16-byte piece c lies at place c ^ swizzle(k)
// The loads write LDS in lane order, so the exchange happens on the side of memory: a lane fetches the piece whose place is its own.
//
// Fragments: lane l takes row l % 16 of a fragment and the reduction steps of group l / 16.  The rows of the right operand are dealt to
// its fragments so that a lane ends up with eight neighbouring columns of the result: row i of fragment j is row
// (j / 2) * 32 + (i / 4) * 8 + (j % 2) * 4 + i % 4 of the wave's columns, and the four sums that a lane holds of fragment j are
// columns (j / 2) * 32 + (l / 16) * 8 + (j % 2) * 4 + 0..3.  Results then leave as 16-byte pieces without a trip through LDS.
//
// The swizzles: reads are served 16 lanes (16-byte reads) or 32 lanes (8-byte transposing reads) at a time, and the lanes that are served
// together are to touch different banks.  For 16-byte reads of rows the left operand's (r >> 1) & 7 does that for every order of lanes, and
// the right operand's is the same function of the fragment's row number.  Transposing reads: eight steps, four pieces of 8 bytes each.  The
// right operand's pieces are 16 bytes apart, which costs it two turns instead of one.
template <bool RIGHT>
__device__ __forceinline__ int swizzle_rows(int r) {
    return RIGHT ? ((r >> 1) & 1) | ((r >> 3) & 3) << 1 : (r >> 1) & 7;
}
template <typename T, int R, bool RIGHT>
__device__ __forceinline__ int swizzle_steps(int k) {
    if constexpr (sizeof(T) == 2) {
        if (RIGHT) return R >= 128 ? (k & 3) << 2 : ((k >> 1) & 1) << 2;
        return R >= 128 ? ((k & 3) | ((k >> 3) & 1) << 2) << 1 : (((k >> 1) & 1) | ((k >> 3) & 1) << 1) << 1;
    } else {
        return RIGHT ? ((k >> 2) & 1) << 3 | ((k >> 3) & 1) : ((k >> 2) & 3) << 2;
    }
}

// Where a lane finds its parts of the F fragments of its wave, whose rows start at `first`: as few addresses as the swizzle allows, everything
// else is a constant that fits a read's offset (a k-tile half h, and the stages of an operand, which lie one behind the other).
template <typename T, int R, bool STEPS, bool RIGHT, int F>
struct Reader {
    static constexpr bool HALF = sizeof(T) == 2;
    static constexpr int N = !STEPS ? 2 : HALF ? (RIGHT ? F / 2 : F) : (RIGHT || F < 4 ? F : 4);
    unsigned at[N];
    __device__ __forceinline__ void init(unsigned base, int first, int lane) {
        const int i = lane & 15, grp = lane >> 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (!STEPS) {  // n: half of the k-tile
                const int r = first + (RIGHT ? (i >> 2) * 8 + (i & 3) : i);
                at[n] = base + r * ROWB + (((n * 4 + grp) ^ swizzle_rows<RIGHT>(r)) << 4);
            } else if constexpr (HALF) {
                // lane i of a group of 16 addresses piece i (step i / 4, rows of quarter i % 4) and receives row i of steps 0 to 3
                const int k = grp * 8 + (i >> 2), r = first + (RIGHT ? n * 32 + (i & 3) * 8 : n * 16 + (i & 3) * 4);
                at[n] = base + k * (R * 2) + (((r >> 3) ^ swizzle_steps<T, R, RIGHT>(k)) << 4) + (r & 4) * 2;
            } else {
                const int k = grp * 4, r = first + (RIGHT ? (n >> 1) * 32 + (i >> 2) * 8 + (n & 1) * 4 + (i & 3) : n * 16 + i);
                at[n] = base + k * (R * 4) + (((r >> 2) ^ swizzle_steps<T, R, RIGHT>(k)) << 4) + (r & 3) * 4;
            }
        }
    }
    __device__ __forceinline__ void move(int bytes) {
#pragma unroll
        for (int n = 0; n < N; ++n) at[n] += bytes;
    }
    __device__ __forceinline__ typename Elem<T>::frag read(const unsigned char* smem, int stage, int f, int h) const {
        const int st = stage * (R * ROWB);
        if constexpr (!STEPS) {
            return *(const typename Elem<T>::frag*)(smem + at[h] + st + (RIGHT ? (f >> 1) * 32 + (f & 1) * 4 : f * 16) * ROWB);
        } else if constexpr (HALF) {
            s16x4 part[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const unsigned char* q = smem + at[RIGHT ? f >> 1 : f] + st + (h * 32 + p * 4) * (R * 2) + (RIGHT ? (f & 1) * 8 : 0);
                part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_void_ptr)q);
            }
            const s16x8 w = {part[0][0], part[0][1], part[0][2], part[0][3], part[1][0], part[1][1], part[1][2], part[1][3]};
            return __builtin_bit_cast(bf16x8, w);
        } else {
            f32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = *(const float*)(smem + at[f % N] + st + (h * 16 + e) * (R * 4) + f / N * 256);
            return w;
        }
    }
};

__device__ __forceinline__ f32x4 mfma_step(const bf16x8& a, const bf16x8& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_step(const f32x4& a, const f32x4& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ u32x4 uniform_rsrc(const char* base, unsigned bytes) {
    const unsigned long long v = (unsigned long long)base;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((unsigned)v);
    r[1] = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32) & 0xffffu);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00027000;
    return r;
}
// 16 bytes per lane from base + offset into LDS, 1 KB from `lds_byte` in lane order; what lies past the buffer's end is not read.
__device__ __forceinline__ void load_lds(const u32x4& rsrc, unsigned offset, unsigned lds_byte) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds_byte), "v"(offset), "s"(rsrc) : "memory");
}

// One operand's way into LDS: which pieces a lane fetches, and what of memory may be read.
template <typename T, int R, int NW, bool STEPS, bool RIGHT, bool GATED>
struct Feed {
    static constexpr int LOADS = R / 8 / NW;  // wave instructions of 1 KB
    static constexpr int BK = Elem<T>::BK, PIECE = Elem<T>::PIECE, PIECES = R / PIECE;
    static_assert(R % (8 * NW) == 0, "whole instructions");
    static_assert(!GATED || (!STEPS && RIGHT), "the factors of a gated pair are interleaved by rows");
    unsigned off[LOADS];
    const char *base0, *base1;  // the tile's first row at reduction step 0, of each product (of each factor, GATED)
    unsigned step_bytes;        // STEPS: from one reduction step to the next
    unsigned span;              // bytes that may be read from there on: of all steps (rows), of one step
    int wave;

    __device__ __forceinline__ void init(const void* m0, const void* m1, long row0, int rows, long pitch, int k, int wave_, int lane) {
        constexpr int S = sizeof(T);
        wave = wave_;
        const long skip = (STEPS ? row0 : row0 * pitch) * S;
        base0 = (const char*)m0 + skip;
        base1 = (const char*)m1 + skip;
        const int used = GATED ? R / 2 : R, r = rows < used ? rows : used;
        // whole pieces, so that none is cut in the middle
        span = STEPS ? (unsigned)(r * S + 15) / 16 * 16 : (unsigned)((r - 1) * pitch * S + ((long)k * S + 15) / 16 * 16);
        step_bytes = (unsigned)(pitch * S);
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int at = wave * LOADS + n;
            if constexpr (!STEPS) {
                const int line = at * 8 + (lane >> 3), c = (lane & 7) ^ swizzle_rows<RIGHT>(line);
                const int src = GATED ? (line >> 6) * 32 + (line & 31) : line;
                off[n] = src * step_bytes + c * 16;
            } else {
                const int idx = at * 64 + lane, step = idx / PIECES, c = (idx % PIECES) ^ swizzle_steps<T, R, RIGHT>(step);
                off[n] = step * step_bytes + c * 16;
            }
        }
    }
    // Reduction steps k0 .. k0 + BK - 1 of product `seg`, of which `left` are there.
    __device__ __forceinline__ void issue(int seg, int k0, int left, unsigned lds) const {
        const char* base = seg ? base1 : base0;
        long skip;
        unsigned bytes;
        if constexpr (STEPS) {
            skip = (long)k0 * step_bytes;
            bytes = ((left < BK ? left : BK) - 1) * step_bytes + span;
        } else {
            skip = (long)k0 * (long)sizeof(T);
            bytes = span - (unsigned)skip;
        }
        if (left <= 0) bytes = 0;  // a k-tile that there is none of: nothing is read
        const u32x4 r0 = uniform_rsrc((GATED ? base0 : base) + skip, bytes);
        u32x4 r1 = r0;
        if constexpr (GATED) r1 = uniform_rsrc(base1 + skip, bytes);
#pragma unroll
        for (int n = 0; n < LOADS; ++n) {
            const int at = wave * LOADS + n;
            if (GATED && (at & 4)) load_lds(r1, off[n], lds + at * 1024);
            else load_lds(r0, off[n], lds + at * 1024);
        }
    }
    // Zeros in place of what this lane has fetched past the end of the reduction: the last k-tile of a product that is not whole.
    __device__ __forceinline__ void clear_tail(unsigned char* tile, int left, int lane) const {
        asm volatile("" : "+v"(lane));  // (what depends on it is not worth registers across the loop over k-tiles)
#pragma unroll 1
        for (int n = 0; n < LOADS; ++n) {
            const int idx = (wave * LOADS + n) * 64 + lane;
            int keep;  // values of the piece that belong to the reduction
            if constexpr (!STEPS) keep = left - ((lane & 7) ^ swizzle_rows<RIGHT>(idx >> 3)) * PIECE;
            else keep = idx / PIECES < left ? PIECE : 0;
            T* p = (T*)(tile + idx * 16);
#pragma unroll
            for (int e = 0; e < PIECE; ++e)
                if (e >= keep) p[e] = (T)0.f;
        }
    }
};

// ---- tiles ----------------------------------------------------------------------------------------
// Which tile of which result over which k-tiles a workgroup computes.
struct Tile {
    int split, z, first, last;
    long m0, n0;
};
template <int BM, int TN>
__device__ __forceinline__ Tile tile_of(const KernelArgs& g) {
    // 4 x 8 tiles make one XCD's run of 32, and four of them above each other a block of 16 x 8: what all XCDs work on at a time is as
    // square as can be.
    constexpr int HIGH = 16, WIDE = 8, GM = 4;
    Tile r;
    const int tiles = g.tiles_m * g.tiles_n;
    int t = xcd_remap(blockIdx.x, gridDim.x, g.xcd_shift);
    r.split = t / (tiles * g.outs);
    t -= r.split * tiles * g.outs;
    r.z = t / tiles;
    t -= r.z * tiles;
    const int band = t / (HIGH * g.tiles_n), high = g.tiles_m - band * HIGH < HIGH ? g.tiles_m - band * HIGH : HIGH;
    t -= band * HIGH * g.tiles_n;
    const int block = t / (high * WIDE), wide = g.tiles_n - block * WIDE < WIDE ? g.tiles_n - block * WIDE : WIDE;
    t -= block * high * WIDE;
    const int group = t / (GM * wide), gm = high - group * GM < GM ? high - group * GM : GM;
    t -= group * GM * wide;
    r.m0 = (long)(band * HIGH + group * GM + t % gm) * BM;
    r.n0 = (long)(block * WIDE + t / gm) * TN;
    const int all = g.nk * g.segments;
    r.first = r.split * g.per_split;
    r.last = r.first + g.per_split < all ? r.first + g.per_split : all;
    return r;
}

// Both operands of a tile: what a wave fetches of a k-tile.
template <typename T, int BM, int BN, int NW, bool ASTEPS, bool BSTEPS, bool GATED>
struct Panels {
    static constexpr int BK = Elem<T>::BK;
    typedef Feed<T, BM, NW, ASTEPS, false, false> FeedA;
    typedef Feed<T, BN, NW, BSTEPS, true, GATED> FeedB;
    static constexpr int LOADS = FeedA::LOADS + FeedB::LOADS;
    FeedA fa;
    FeedB fb;
    int nk, k, wave, lane;
    __device__ __forceinline__ Panels(const KernelArgs& g, const Tile& t, int wave_, int lane_) : nk(g.nk), k(g.k), wave(wave_), lane(lane_) {
        const bool each = g.outs > 1;
        fa.init(each && t.z ? g.a[1] : g.a[0], each && !t.z ? g.a[0] : g.a[1], t.m0, (int)(g.m - t.m0), g.pitch_a, k, wave, lane);
        fb.init(g.b[0], g.b[1], t.n0, (int)(g.n - t.n0), g.pitch_b, k, wave, lane);
    }
    // Loads of k-tile kt, LOADS of a wave for each operand; past the last one of the workgroup they read nothing.
    __device__ __forceinline__ void issue_a(int kt, int last, unsigned lds) const {
        const int seg = kt >= nk ? 1 : 0, k0 = (kt - seg * nk) * BK;
        fa.issue(seg, k0, kt < last ? k - k0 : 0, lds);
    }
    __device__ __forceinline__ void issue_b(int kt, int last, unsigned lds) const {
        const int seg = kt >= nk ? 1 : 0, k0 = (kt - seg * nk) * BK;
        fb.issue(seg, k0, kt < last ? k - k0 : 0, lds);
    }
    // What this wave has fetched of k-tile kt has landed: nothing of it lies past the end of the reduction any more.
    __device__ __forceinline__ void landed(int kt, unsigned char* tile_a, unsigned char* tile_b) const {
        const int left = k - (kt - (kt >= nk ? nk : 0)) * BK;
        if (left < BK) {
            fa.clear_tail(tile_a, left, lane);
            fb.clear_tail(tile_b, left, lane);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
};

// A barrier that waits for no load.
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
#define WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

// Row i of the fragments, for an i that is no constant but the same in every lane.
template <int I = 0, int FM, int FN>
__device__ __forceinline__ void pick_row(const f32x4 (&acc)[FM][FN], int i, f32x4 (&row)[FN]) {
    if constexpr (I + 1 < FM) {
        if (i != I) {
            pick_row<I + 1>(acc, i, row);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        row[j] = acc[I][j];
        asm volatile("; row %1" : "+v"(row[j]) : "n"(I));  // (merged, the copies would become a look-up in memory)
    }
}
// The sums of a wave's part of a tile on their way to memory: one row of fragments after the other, in a loop that is not unrolled (the
// activations of all of them are more code than the instruction cache holds).
template <typename T, bool GATED, int FM, int FN>
__device__ __forceinline__ void finish_tile(const KernelArgs& g, const Tile& t, const f32x4 (&acc)[FM][FN], int row0, int col0, int lane) {
    const int quad = lane >> 4;
#pragma unroll 1
    for (int i = 0; i < FM; ++i) {
        const long row = t.m0 + row0 + i * 16 + (lane & 15);
        f32x4 sums[FN];
        pick_row(acc, i, sums);
#pragma unroll
        for (int jp = 0; jp < FN / 2; jp += GATED ? 2 : 1) {
            const long col = t.n0 + col0 + jp * 32 + quad * 8;
            if (row >= g.m || col >= g.n) continue;
            float v[8], u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = sums[2 * jp + (e >> 2)][e & 3];
                u[e] = GATED ? sums[(2 * jp + 2 + (e >> 2)) % FN][e & 3] : 0.f;
            }
            emit8<T, GATED>(g, t.split, t.z, row, (int)col, v, u);
        }
    }
}

// ---- small tiles -----------------------------------------------------------------------------------
// S stages: a wave waits for its own loads of k-tile t, crosses the one barrier of the k-tile (behind which every wave has read all of k-tile
// t - 1), issues the loads of k-tile t + S - 1 into the stage that is free now, and multiplies.
template <typename T, int BM, int BN, int WGM, int WGN, int S, bool ASTEPS, bool BSTEPS, bool GATED>
__global__ void __launch_bounds__(WGM* WGN * 64) product_kernel(const KernelArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int NW = WGM * WGN;
    constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 16, FN = WTN / 16;
    constexpr int UNIT_A = BM * ROWB, UNIT_B = BN * ROWB, B_AT = S * UNIT_A;
    static_assert(!GATED || WTN == 64, "a wave holds 32 columns of each factor");
    typedef Panels<T, BM, BN, NW, ASTEPS, BSTEPS, GATED> P;
    typedef typename Elem<T>::frag frag;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const Tile t = tile_of<BM, GATED ? BN / 2 : BN>(g);
    const P panels(g, t, wave, lane);
    const unsigned lds = (unsigned)(uintptr_t)(lds_void_ptr)smem;
    Reader<T, BM, ASTEPS, false, FM> ra;
    Reader<T, BN, BSTEPS, true, FN> rb;
    ra.init(0, wm * WTM, lane);
    rb.init(B_AT, wn * WTN, lane);

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto issue = [&](int kt, int s) {
        panels.issue_a(kt, t.last, lds + s * UNIT_A);
        panels.issue_b(kt, t.last, lds + B_AT + s * UNIT_B);
    };
    if (t.first < t.last) {
#pragma unroll
        for (int n = 0; n < S - 1; ++n) issue(t.first + n, n);
        int s = 0;  // stage of k-tile kt
#pragma unroll 1
        for (int kt = t.first; kt < t.last; ++kt) {
            WAIT_VM((S - 2) * P::LOADS);
            panels.landed(kt, smem + s * UNIT_A, smem + B_AT + s * UNIT_B);
            barrier();
            issue(kt + S - 1, s == 0 ? S - 1 : s - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                frag va[FM], vb[FN];
#pragma unroll
                for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, 0, i, h);
#pragma unroll
                for (int j = 0; j < FN; ++j) vb[j] = rb.read(smem, 0, j, h);
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int i = 0; i < FM; ++i) acc[i][j] = mfma_step(vb[j], va[i], acc[i][j]);
            }
            const int s1 = s + 1 == S ? 0 : s + 1;
            ra.move((s1 - s) * UNIT_A);
            rb.move((s1 - s) * UNIT_B);
            s = s1;
            WAIT_LDS();
        }
        WAIT_VM(0);  // (the loads of no k-tile have to end before the workgroup's LDS is another's)
    }
    finish_tile<T, GATED>(g, t, acc, wm * WTM, GATED ? wn * 32 : wn * WTN, lane);
}

// ---- 256x256 tiles: eight waves in two groups that alternate between memory and products -------------------
// Wave w and wave w + 4 share a SIMD.  Each runs  { M(t, h): read the fragments of half h of k-tile t, issue loads;  barrier;  C(t, h): the
// half's products;  barrier }  and waves 4 to 7 enter one barrier later than waves 0 to 3, so that at any time one wave of a SIMD issues
// nothing but matrix instructions from registers while the other reads LDS and issues loads.
//
// LDS holds three k-tiles of the left operand and two of the right one, all 160 KB: M(t, 0) reads the right operand's fragments of both
// halves, so that its stage is free half a k-tile earlier and a third one would buy nothing.
// Phases between barriers: group 0 runs M(t, 0) in phase 4t, C(t, 0) in 4t + 1, M(t, 1) in 4t + 2, C(t, 1) in 4t + 3, group 1 each of them
// one phase later.  The left operand's stage of k-tile t is last read in phase 4t + 3; k-tile t + 3 is issued into it in M(t + 1, 0), phases
// 4t + 4 and 4t + 5.  The right operand's is last read in phase 4t + 1; k-tile t + 2 is issued into it in M(t, 1), phases 4t + 2 and 4t + 3.  At
// the end of M(t, 1) each wave waits for its own loads of k-tile t + 1, the last of which are one k-tile old: the two groups issued after
// them stay in flight.  k-tile t + 1 is first read in phase 4t + 4.
template <typename T, int BM, int BN, int WGM, int WGN, bool ASTEPS, bool BSTEPS, bool GATED>
__global__ void __launch_bounds__(512, BM == 128 ? 4 : 2) product_pp_kernel(const KernelArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int NW = WGM * WGN;
    constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 16, FN = WTN / 16;
    constexpr int UNIT_A = BM * ROWB, UNIT_B = BN * ROWB, A_AT = 2 * UNIT_B;  // stages; the left operand's lie behind the right one's
    static_assert(NW == 8 && WTN == 64, "two groups of four waves; a wave of a gated pair holds 32 columns of each factor");
    typedef Panels<T, BM, BN, NW, ASTEPS, BSTEPS, GATED> P;
    typedef typename Elem<T>::frag frag;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave >> 2, wm = wave / WGN, wn = wave % WGN;
    const Tile t = tile_of<BM, GATED ? BN / 2 : BN>(g);
    const P panels(g, t, wave, lane);
    const unsigned lds = (unsigned)(uintptr_t)(lds_void_ptr)smem;

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    Reader<T, BM, ASTEPS, false, FM> ra;
    Reader<T, BN, BSTEPS, true, FN> rb;
    ra.init(A_AT, wm * WTM, lane);
    rb.init(0, wn * WTN, lane);
    auto multiply = [&](const frag (&va)[FM], const frag (&vb)[FN]) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int ii = 0; ii < FM; ++ii) {
                const int i = (j & 1) ? FM - 1 - ii : ii;
                acc[i][j] = mfma_step(vb[j], va[i], acc[i][j]);
            }
    };
    auto fence = [] {
        __builtin_amdgcn_sched_barrier(0);
        barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    if (t.first < t.last) {
        auto slot_a = [](int s) { return A_AT + s * UNIT_A; };
        auto slot_b = [](int s) { return s * UNIT_B; };
        for (int n = 0; n < 2; ++n) {
            panels.issue_a(t.first + n, t.last, lds + slot_a(n));
            panels.issue_b(t.first + n, t.last, lds + slot_b(n));
        }
        WAIT_VM(P::LOADS);
        panels.landed(t.first, smem + slot_a(0), smem + slot_b(0));
        barrier();
        if (grp) barrier();
        int sa = 0, sb = 0;  // stages of k-tile kt
#pragma unroll 1
        for (int kt = t.first; kt < t.last; ++kt) {
            const int sa1 = sa == 2 ? 0 : sa + 1, sa2 = sa1 == 2 ? 0 : sa1 + 1;
            frag va[FM], vb[2][FN];
#pragma unroll
            for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, 0, i, 0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < FN; ++j) vb[h][j] = rb.read(smem, 0, j, h);
            panels.issue_a(kt + 2, t.last, lds + slot_a(sa2));
            WAIT_LDS();
            fence();
            multiply(va, vb[0]);
            fence();
#pragma unroll
            for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, 0, i, 1);
            panels.issue_b(kt + 2, t.last, lds + slot_b(sb));
            ra.move((sa1 - sa) * UNIT_A);
            rb.move(sb ? -UNIT_B : UNIT_B);
            sa = sa1;
            sb ^= 1;
            WAIT_LDS();
            WAIT_VM(P::LOADS);
            if (kt + 1 < t.last) panels.landed(kt + 1, smem + slot_a(sa), smem + slot_b(sb));
            fence();
            multiply(va, vb[1]);
            fence();
        }
        if (!grp) barrier();
        WAIT_VM(0);  // (the loads of no k-tile have to end before the workgroup's LDS is another's)
    }
    finish_tile<T, GATED>(g, t, acc, wm * WTM, GATED ? wn * 32 : wn * WTN, lane);
}

// ---- few rows: the right operand is read once, straight into registers ---------------------------------------
// For a few rows on the left (tokens that are being answered) the product is a walk over the weight.  A workgroup takes 16 rows of it (of both
// factors of a gated pair), its eight waves an eighth of the reduction each: a wave's load is 16 rows x 64 bytes, a fragment as the matrix
// instruction takes it, and the fragments of x come out of the caches the same way.  The next STEPS of them are on their way while the last
// are multiplied.  The waves' sums meet in LDS.  Rows may start at any element: the hardware reads vectors from any address.
template <typename T, bool GATED>
__global__ void __launch_bounds__(512) product_rows_kernel(const KernelArgs g) {
    typedef typename Elem<T>::frag frag;
    typedef frag __attribute__((aligned(sizeof(T)))) frag_any;
    constexpr int W = GATED ? 2 : 1, NW = 8, PIECE = Elem<T>::PIECE, STEP = 4 * PIECE;  // reduction steps of a fragment
    constexpr int STEPS = GATED ? 4 : 6;
    __shared__ __align__(16) float part[NW][W][16][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, grp = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const int row = n0 + i < g.n ? n0 + i : g.n - 1;  // (rows past the end are the last one again: what they give is not wanted)
    const T* wp[W];
#pragma unroll
    for (int w = 0; w < W; ++w) wp[w] = (const T*)g.b[w] + row * g.pitch_b + grp * PIECE;
    const T* xp = (const T*)g.a[0] + (i < g.m ? i : g.m - 1) * g.pitch_a + grp * PIECE;

    f32x4 acc[W];
#pragma unroll
    for (int w = 0; w < W; ++w) acc[w] = f32x4{0.f, 0.f, 0.f, 0.f};
    // this wave's part of the reduction, in whole fragments; the last one of all may be cut
    const int all = g.k / STEP, mine = (all + NW - 1) / NW;
    int s = wave * mine;
    const int end = s + mine < all ? s + mine : all;
    frag vw[2][STEPS][W], vx[2][STEPS];
    auto load = [&](int b, int s, int count) {
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            if (c >= count) break;
#pragma unroll
            for (int w = 0; w < W; ++w) vw[b][c][w] = *(const frag_any*)(wp[w] + (long)(s + c) * STEP);
            vx[b][c] = *(const frag_any*)(xp + (long)(s + c) * STEP);
        }
    };
    auto multiply = [&](int b, int count) {
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            if (c >= count) break;
#pragma unroll
            for (int w = 0; w < W; ++w) acc[w] = mfma_step(vw[b][c][w], vx[b][c], acc[w]);
        }
    };
    const int batches = s < end ? (end - s) / STEPS : 0;
    if (batches > 0) load(0, s, STEPS);
    for (int n = 0; n < batches; n += 2) {
        if (n + 1 < batches) load(1, s + STEPS, STEPS);
        multiply(0, STEPS);
        s += STEPS;
        if (n + 1 >= batches) break;
        if (n + 2 < batches) load(0, s + STEPS, STEPS);
        multiply(1, STEPS);
        s += STEPS;
    }
    if (s < end) {
        load(0, s, end - s);
        multiply(0, end - s);
    }
    if (wave == NW - 1 && all * STEP < g.k) {  // what is left of the reduction, value by value
        const int k0 = all * STEP + grp * PIECE;
        frag tw[W], tx;
#pragma unroll
        for (int e = 0; e < PIECE; ++e) {
            const bool there = k0 + e < g.k;
#pragma unroll
            for (int w = 0; w < W; ++w) tw[w][e] = there ? wp[w][(long)all * STEP + e] : (T)0.f;
            tx[e] = there ? xp[(long)all * STEP + e] : (T)0.f;
        }
#pragma unroll
        for (int w = 0; w < W; ++w) acc[w] = mfma_step(tw[w], tx, acc[w]);
    }
    // a lane holds rows n0 + 4 grp .. + 3 of the weight against row i of x
#pragma unroll
    for (int w = 0; w < W; ++w) *(f32x4*)&part[wave][w][i][grp * 4] = acc[w];
    __syncthreads();
    const int half = (tid & 1) * 8, j = n0 + half, token = tid >> 1;
    if (token >= g.m || j >= g.n) return;  // (g.m <= 16)
    float v[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = u[e] = 0.f;
#pragma unroll
        for (int q = 0; q < NW; ++q) {
            v[e] += part[q][0][token][half + e];
            if (GATED) u[e] += part[q][W - 1][token][half + e];
        }
    }
    finish8<T, GATED>(g, 0, token, j, v, u);
}

// The parts of a reduction that several workgroups took, added in their order, and the layer's arithmetic.  Without any part (k = 0)
// the sums are zero.
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) product_join_kernel(const KernelArgs g) {
    const long pieces = (g.n + 7) / 8, all = pieces * g.m * g.outs;
    for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < all; at += (long)gridDim.x * 256) {
        const int j = (int)(at % pieces) * 8;
        const long r = at / pieces;
        const int z = (int)(r / g.m);
        const long i = r - (long)z * g.m;
        const int count = g.n - j < 8 ? g.n - j : 8, parts = GATED ? 2 : g.outs;
        float v[8] = {}, u[8] = {};
        for (int s = 0; s < g.splits; ++s) {
            const float* p = g.partial + (((long)s * parts + z) * g.m + i) * g.n + j;
            float w[8];
            load8(p, 1, g.vec && count == 8, count, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += w[e];
            if (GATED) {
                load8(p + (long)g.m * g.n, 1, g.vec && count == 8, count, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] += w[e];
            }
        }
        finish8<T, GATED>(g, z, i, j, v, u);
    }
}

// ---- packing ------------------------------------------------------------------------------------
// rows x cols values from any strides into rows `pitch` apart (whole 16-byte pieces; what lies past cols is left as it is: the products
// clear it).  64 x 64 values go through LDS, read along the nearer stride.
template <typename T>
__global__ void __launch_bounds__(256) product_pack_kernel(const T* src, long row, long col, int rows, int cols, T* dst, long pitch, int along) {
    __shared__ T tile[64][65];
    const unsigned across = (unsigned)((cols + 63L) / 64);
    const long r0 = (long)(blockIdx.x / across) * 64, c0 = (long)(blockIdx.x % across) * 64;
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
    for (int s = y; s < 64; s += 4) {
        const int r = along ? x : s, c = along ? s : x;
        if (r0 + r < rows && c0 + c < cols) tile[r][c] = src[(r0 + r) * row + (c0 + c) * col];
    }
    __syncthreads();
    for (int s = y; s < 64; s += 4)
        if (r0 + s < rows && c0 + x < cols) dst[(r0 + s) * pitch + c0 + x] = tile[s][x];
}

// ---- activation gradients and sums over rows ----------------------------------------------------------
// A workgroup takes 256 columns (32 threads, eight columns each) of GRAD_ROWS rows; eight rows at a time.
constexpr int GRAD_ROWS = 64;
template <typename T, bool PAIR>
__global__ void __launch_bounds__(256) act_grad_kernel(const ActGradArgs g, int vec, int chunks) {
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int blocks = (g.n + 255) / 256;
    const int chunk = blockIdx.x / blocks;
    const int j = (blockIdx.x - chunk * blocks) * 256 + tx * 8;
    const int count = g.n - j < 8 ? g.n - j : 8;
    const bool whole = vec && count == 8;
    float sum[PAIR ? 2 : 1][8] = {};
    if (j < g.n) {
        const long r0 = (long)chunk * GRAD_ROWS;
#pragma unroll 2
        for (int s = ty; s < GRAD_ROWS; s += 8) {
            const long i = r0 + s;
            if (i >= g.m) break;
            float dy[8];
            load8((const T*)g.dy + i * g.n + j, 1, whole, count, dy);
#pragma unroll
            for (int f = 0; f < (PAIR ? 2 : 1); ++f) {
                float v[8];
                if (g.factors > f) {
                    load8((const T*)g.d[f] + i * g.n + j, 1, whole, count, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= dy[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = dy[e];
                }
                if (g.dz[f]) store8((T*)g.dz[f] + i * g.pitch + j, whole, count, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[f][e] += v[e];
            }
        }
    }
    if (!g.partials) return;
    __shared__ float part[8][32][9];
#pragma unroll
    for (int f = 0; f < (PAIR ? 2 : 1); ++f) {
        if (!g.db[f]) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) part[ty][tx][e] = sum[f][e];
        __syncthreads();
        const int c = threadIdx.x, col = (blockIdx.x - chunk * blocks) * 256 + c;
        if (col < g.n) {
            float v = 0.f;
#pragma unroll
            for (int y = 0; y < 8; ++y) v += part[y][c >> 3][c & 7];
            g.partials[((long)f * chunks + chunk) * g.n + col] = v;
        }
    }
}
// Four rows of threads take the parts in turn; their sums are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) row_sum_kernel(const float* partials, int chunks, int n, T* out0, T* out1) {
    __shared__ float part[4][64];
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6, f = blockIdx.y;
    T* out = f ? out1 : out0;
    if (!out) return;
    const int j = blockIdx.x * 64 + x;
    float v = 0.f;
    if (j < n)
        for (int c = y; c < chunks; c += 4) v += partials[((long)f * chunks + c) * n + j];
    part[y][x] = v;
    __syncthreads();
    if (y == 0 && j < n) out[j] = (T)((part[0][x] + part[1][x]) + (part[2][x] + part[3][x]));
}

// ---- host side ----------------------------------------------------------------------------------------
inline long up(long v, long m) { return (v + m - 1) / m * m; }
inline int elem_size(int dtype) { return dtype == MUON_HIP_BF16 ? 2 : 4; }

enum { LIE_ROWS = 0, LIE_STEPS = 1, LIE_PACKED = 2 };
struct Plan {
    int lie_a, lie_b;
    long pitch_a, pitch_b;        // elements
    long pack_a, pack_b;          // bytes of one packed matrix
    int count_a, count_b;         // matrices of each operand
    int tile, splits, per_split, nk, segments, outs;  // tile 0: the kernel of few rows
    long partial_bytes, bytes;
};

// What a way of computing a product of bf16 (fp32) matrices takes, in microseconds, as measured on 256 compute units: `start`, and for every
// workgroup of a compute unit `each` and its k-tiles, which take `alone` while it has the compute unit for itself and `busy` where there are
// more.  256-tiles reach 1.5 PFLOP/s where they fill the machine, 128-tiles 1.0; over few or short products the smaller ones win because they
// start and end sooner.
struct Cost {
    float start, each, alone, busy;
};
constexpr Cost kCost[2][3] = {{{4.5f, 0.5f, 0.72f, 0.50f}, {5.f, 1.f, 2.2f, 1.88f}, {0.f, 0.f, 0.f, 0.f}},   // fp32: tiles of 64 and 128 (no 256)
                              {{2.5f, 0.5f, 0.30f, 0.22f}, {3.f, 1.f, 0.66f, 0.52f}, {3.f, 3.f, 1.15f, 1.35f}}};  // bf16: 64, 128, 256
constexpr float kJoinStart = 4.f, kJoinBytes = 5.5e6f;  // of a split reduction: its launch, and bytes in a microsecond
constexpr int kTile[3] = {64, 128, 256};

// How an operand is read: as it lies where 16-byte pieces of its rows (or of its reduction steps) are aligned and 32 bits span a tile of it.
int lie_of(const ProductOperand& o, int count, int rows, int k, int size, bool steps_ok, long& pitch) {
    const long piece = 16 / size;
    auto fits = [&](long p, long lines) { return p % piece == 0 && p <= (0x7fff0000L / size) / lines; };
    bool by_rows = true, by_steps = steps_ok;
    for (int i = 0; i < count; ++i) {
        if (((uintptr_t)o.base[i]) & 15) by_rows = by_steps = false;
        // (one row, or one step, has no stride that matters)
        if (!(o.col[i] == 1 || k == 1) || !(rows == 1 || (fits(o.row[i], 256) && o.row[i] == o.row[0]))) by_rows = false;
        if (!(o.row[i] == 1 || rows == 1) || !(k == 1 || (fits(o.col[i], 64) && o.col[i] == o.col[0]))) by_steps = false;
    }
    if (k > 0x7fff0000L / size) by_rows = false;
    if (by_rows) {
        pitch = rows == 1 ? 0 : o.row[0];
        return LIE_ROWS;
    }
    if (by_steps) {
        pitch = k == 1 ? 0 : o.col[0];
        return LIE_STEPS;
    }
    pitch = up(k, piece);
    return LIE_PACKED;
}

// Few rows against rows of a weight, wherever they start: one launch, where tiles that leave most of the machine idle would have to share the
// reduction and be joined (1 x 4096 x 4096: 9 us against 14).  From 9 rows on the fragments of x are as much to fetch as the weight and the
// tiles, which keep theirs in LDS, are faster (16 x 4096 x 12288: 24 us against 30).
constexpr int kFewRows = 8;
bool few_rows(const ProductArgs& p, Plan& l) {
    if (p.m > kFewRows || (p.kind != PRODUCT_LINEAR && p.kind != PRODUCT_GATED)) return false;
    if (p.k > 16384 && p.n < 1024) return false;  // long rows on few compute units
    if (p.k > 1 && (p.a.col[0] != 1 || p.b.col[0] != 1)) return false;
    if (p.kind == PRODUCT_GATED && ((p.k > 1 && p.b.col[1] != 1) || p.b.row[1] != p.b.row[0])) return false;
    l.tile = 0;
    l.pitch_a = p.a.row[0];
    l.pitch_b = p.b.row[0];
    l.segments = l.outs = l.splits = 1;
    return true;
}

bool make_plan(const ProductArgs& p, int cus, Plan& l) {
    const int size = elem_size(p.dtype), bk = ROWB / size;
    const bool gated = p.kind == PRODUCT_GATED;
    l = Plan{};
    l.count_a = p.kind == PRODUCT_SUM || p.kind == PRODUCT_EACH ? 2 : 1;
    l.count_b = gated || p.kind == PRODUCT_SUM ? 2 : 1;
    l.segments = p.kind == PRODUCT_SUM ? 2 : 1;
    l.outs = p.kind == PRODUCT_EACH ? 2 : 1;
    if (p.m == 0 || p.n == 0) return true;
    if (p.k == 0) return true;
    if (few_rows(p, l)) return true;
    l.lie_a = lie_of(p.a, l.count_a, p.m, p.k, size, true, l.pitch_a);
    l.lie_b = lie_of(p.b, l.count_b, p.n, p.k, size, !gated, l.pitch_b);
    for (const long pitch : {l.lie_a == LIE_PACKED ? l.pitch_a : 0, l.lie_b == LIE_PACKED ? l.pitch_b : 0})
        if (pitch > (0x7fff0000L / size) / 256) return false;
    l.pack_a = l.lie_a == LIE_PACKED ? up(p.m * l.pitch_a * size, 256) : 0;
    l.pack_b = l.lie_b == LIE_PACKED ? up(p.n * l.pitch_b * size, 256) : 0;
    l.nk = (int)((p.k + (long)bk - 1) / bk);
    auto tiles_of = [&](int t) { return up(p.m, t) / t * (up(p.n, gated ? t / 2 : t) / (gated ? t / 2 : t)) * l.outs; };
    const long all = (long)l.nk * l.segments;
    if (all > 0x3fffffffL) return false;
    const bool bf = p.dtype == MUON_HIP_BF16;
    float best = 1e30f;
    long tiles = 0;
    for (int c = 0; c < (bf ? 3 : 2); ++c) {
        const long here = tiles_of(kTile[c]);
        const Cost& q = kCost[bf][c];
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (want > 1 && (want > all / 4 || here * want > 8L * cus)) break;
            const long per = (all + want - 1) / want, parts = (all + per - 1) / per;
            const long load = (here * parts + cus - 1) / cus;
            float t = q.start + q.each * load + (float)per * (load <= 1 ? q.alone : std::max(q.alone, q.busy * load));
            if (parts > 1) t += kJoinStart + (float)p.m * p.n * (gated ? 2 : l.outs) * 8.f * parts / kJoinBytes;
            if (t < best) {
                best = t;
                tiles = here;
                l.tile = kTile[c];
                l.per_split = (int)per;
                l.splits = (int)parts;
            }
        }
    }
    if (tiles > 0x3fffffffL) return false;
    if (tiles * l.splits > 0x7fffffffL) return false;
    if (l.splits > 1) l.partial_bytes = (long)l.splits * (gated ? 2 : l.outs) * p.m * p.n * 4;
    l.bytes = l.pack_a * l.count_a + l.pack_b * l.count_b + l.partial_bytes;
    return true;
}

template <typename T, int BM, int BN, int WGM, int WGN, int S, bool AS, bool BS, bool GATED>
hipError_t launch_tiles(const KernelArgs& g, hipStream_t stream) {
    constexpr int smem = S * (BM + BN) * ROWB;
    static std::atomic<unsigned long long> configured{0};
    const auto kern = product_kernel<T, BM, BN, WGM, WGN, S, AS, BS, GATED>;
    if (hipError_t e = allow_dynamic_lds((const void*)kern, smem, configured); e != hipSuccess) return e;
    const long grid = (long)g.tiles_m * g.tiles_n * g.outs * g.splits;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(WGM * WGN * 64), smem, stream, g);
    return hipGetLastError();
}
template <typename T, int BM, int BN, int WGM, int WGN, bool AS, bool BS, bool GATED>
hipError_t launch_pp(const KernelArgs& g, hipStream_t stream) {
    constexpr int smem = (3 * BM + 2 * BN) * ROWB;
    static std::atomic<unsigned long long> configured{0};
    const auto kern = product_pp_kernel<T, BM, BN, WGM, WGN, AS, BS, GATED>;
    if (hipError_t e = allow_dynamic_lds((const void*)kern, smem, configured); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)g.tiles_m * g.tiles_n * g.outs * g.splits)), dim3(512), smem, stream, g);
    return hipGetLastError();
}
template <typename T, bool AS, bool BS, bool GATED>
hipError_t launch_tile(int tile, const KernelArgs& g, int cus, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (tile == 256) return launch_pp<T, 256, 256, 2, 4, AS, BS, GATED>(g, s);
    }
    if (tile == 128) {
        // Where every compute unit has at most one of them, eight waves and four stages (4096 x 4096 x 1024: 48 us against 55); otherwise two
        // workgroups of four waves share one.
        if (sizeof(T) == 2 && (long)g.tiles_m * g.tiles_n * g.outs * g.splits <= cus) return launch_tiles<T, 128, 128, 4, 2, 4, AS, BS, GATED>(g, s);
        return launch_tiles<T, 128, 128, 2, 2, 2, AS, BS, GATED>(g, s);
    }
    return launch_tiles<T, 64, 64, 4, 1, 3, AS, BS, GATED>(g, s);
}
template <typename T, bool GATED>
hipError_t launch_rows(const KernelArgs& g, hipStream_t s) {
    hipLaunchKernelGGL((product_rows_kernel<T, GATED>), dim3((unsigned)(up(g.n, 16) / 16)), dim3(512), 0, s, g);
    return hipGetLastError();
}

template <typename T>
hipError_t run_product(const ProductArgs& p, const Plan& l, void* workspace, int cus, int xcd_shift, hipStream_t s) {
    constexpr int S = sizeof(T);
    const bool gated = p.kind == PRODUCT_GATED;
    KernelArgs g{};
    char* ws = (char*)workspace;
    auto pack = [&](const ProductOperand& o, int lie, int count, int rows, long pitch, long bytes, const void** at) {
        for (int i = 0; i < count; ++i) {
            at[i] = o.base[i];
            if (lie != LIE_PACKED) continue;
            const int along = o.row[i] < o.col[i];
            const dim3 grid((unsigned)(up(p.k, 64) / 64 * (up(rows, 64) / 64)));
            hipLaunchKernelGGL(product_pack_kernel<T>, grid, dim3(256), 0, s, (const T*)o.base[i], o.row[i], o.col[i], rows, p.k, (T*)ws, pitch, along);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            at[i] = ws;
            ws += bytes;
        }
        return hipSuccess;
    };
    g.m = p.m;
    g.n = p.n;
    g.k = p.k;
    g.outs = l.outs;
    g.act = p.act;
    for (int i = 0; i < 2; ++i) {
        g.bias[i] = p.bias[i];
        g.out[i] = p.out[i];
        g.aux[i] = p.aux[i];
    }
    g.residual = p.residual;
    g.res_row = p.res_row;
    g.res_col = p.res_col;
    auto aligned = [](const void* q) { return (((uintptr_t)q) & 15) == 0; };
    g.vec = p.n % 8 == 0 && aligned(p.out[0]) && aligned(p.out[1]) && aligned(p.aux[0]) && aligned(p.aux[1]);
    g.vec_res = p.residual && p.n % 8 == 0 && p.res_col == 1 && p.res_row % (16 / S) == 0 && aligned(p.residual);
    g.xcd_shift = xcd_shift;
    if (p.k > 0) {
        if (hipError_t e = pack(p.a, l.lie_a, l.count_a, p.m, l.pitch_a, l.pack_a, g.a); e != hipSuccess) return e;
        if (hipError_t e = pack(p.b, l.lie_b, l.count_b, p.n, l.pitch_b, l.pack_b, g.b); e != hipSuccess) return e;
        g.pitch_a = l.pitch_a;
        g.pitch_b = l.pitch_b;
        g.nk = l.nk;
        g.segments = l.segments;
        g.splits = l.splits;
        g.per_split = l.per_split;
        const int tn = gated ? l.tile / 2 : l.tile;
        if (l.tile) {
            g.tiles_m = (int)(up(p.m, l.tile) / l.tile);
            g.tiles_n = (int)(up(p.n, tn) / tn);
        }
        g.partial = l.splits > 1 ? (float*)ws : nullptr;
        const bool as = l.lie_a == LIE_STEPS, bs = l.lie_b == LIE_STEPS;
        hipError_t e;
        if (l.tile == 0) e = gated ? launch_rows<T, true>(g, s) : launch_rows<T, false>(g, s);
        else if (gated) e = as ? launch_tile<T, true, false, true>(l.tile, g, cus, s) : launch_tile<T, false, false, true>(l.tile, g, cus, s);
        else if (as) e = bs ? launch_tile<T, true, true, false>(l.tile, g, cus, s) : launch_tile<T, true, false, false>(l.tile, g, cus, s);
        else e = bs ? launch_tile<T, false, true, false>(l.tile, g, cus, s) : launch_tile<T, false, false, false>(l.tile, g, cus, s);
        if (e != hipSuccess || l.splits == 1) return e;
    }
    const long work = up(p.n, 8) / 8 * p.m * l.outs;
    const unsigned grid = (unsigned)(up(work, 256) / 256 < 65536 ? up(work, 256) / 256 : 65536);
    if (gated) hipLaunchKernelGGL((product_join_kernel<T, true>), dim3(grid), dim3(256), 0, s, g);
    else hipLaunchKernelGGL((product_join_kernel<T, false>), dim3(grid), dim3(256), 0, s, g);
    return hipGetLastError();
}

}  // namespace

long product_workspace(const ProductArgs& p, int cus) {
    Plan l;
    return make_plan(p, cus, l) ? l.bytes : -1;
}

hipError_t launch_product(const ProductArgs& p, void* workspace, int cus, int xcd_shift, hipStream_t stream) {
    Plan l;
    if (!make_plan(p, cus, l)) return hipErrorInvalidValue;
    if (p.m == 0 || p.n == 0) return hipSuccess;
    return p.dtype == MUON_HIP_BF16 ? run_product<bf16_t>(p, l, workspace, cus, xcd_shift, stream) : run_product<float>(p, l, workspace, cus, xcd_shift, stream);
}

long act_grad_partials(long m, long n) { return up(m, GRAD_ROWS) / GRAD_ROWS * n; }

hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t stream) {
    const bool pair = a.factors > 1;
    const long chunks = up(a.m, GRAD_ROWS) / GRAD_ROWS, blocks = up(a.n, 256) / 256 * chunks;
    auto aligned = [](const void* q) { return (((uintptr_t)q) & 15) == 0; };
    const int vec = a.n % 8 == 0 && a.pitch % 8 == 0 && aligned(a.dy) && aligned(a.d[0]) && aligned(a.d[1]) && aligned(a.dz[0]) && aligned(a.dz[1]);
    const bool bf = a.dtype == MUON_HIP_BF16;
    if (blocks > 0) {
        if (bf && pair) hipLaunchKernelGGL((act_grad_kernel<bf16_t, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vec, (int)chunks);
        else if (bf) hipLaunchKernelGGL((act_grad_kernel<bf16_t, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vec, (int)chunks);
        else if (pair) hipLaunchKernelGGL((act_grad_kernel<float, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vec, (int)chunks);
        else hipLaunchKernelGGL((act_grad_kernel<float, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a, vec, (int)chunks);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if ((!a.db[0] && !a.db[1]) || a.n == 0) return hipSuccess;
    const dim3 grid((unsigned)(up(a.n, 64) / 64), pair ? 2 : 1);
    if (bf) hipLaunchKernelGGL(row_sum_kernel<bf16_t>, grid, dim3(256), 0, stream, a.partials, (int)chunks, a.n, (bf16_t*)a.db[0], (bf16_t*)a.db[1]);
    else hipLaunchKernelGGL(row_sum_kernel<float>, grid, dim3(256), 0, stream, a.partials, (int)chunks, a.n, (float*)a.db[0], (float*)a.db[1]);
    return hipGetLastError();
}
