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
    int xcd_shift;
};

// ---- activations -----------------------------------------------------------------------------
// act(z) and act'(z).  The factor of a gated pair's gradient and the activation itself come out of one evaluation.
//
// Results of bf16 tensors are rounded to 8 bits, so theirs take the hardware's exponential and reciprocal (one step of fp32 each).  Their
// normal distribution function is exp(-z^2 / 2) / 2 times a polynomial of degree 6 in t = 1 / (1 + 0.42 |z| / sqrt 2) for z <= 0, fitted to
// erfc(x) exp(x^2) over 0 <= x <= 9.6 for the smallest largest error, relative to the value where that is small: in fp32 off by 3.3e-7 at
// most, and by 2.1e-5 of itself down to where z Phi(z) leaves the normal numbers.  8192 x 4096 x 4096 with silu takes 198 us where it
// takes 188 without, with gelu 207.  fp32 tensors get the full functions.
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
template <bool FAST, int ACT>
__device__ __forceinline__ ActPair activate(float z) {
    if constexpr (ACT == ACT_RELU) {
        return ActPair{z <= 0.f ? 0.f : z, z <= 0.f ? 0.f : 1.f};  // (NaN stays NaN)
    } else if constexpr (ACT == ACT_SIGMOID) {
        const float s = sigmoid_of<FAST>(z);
        return ActPair{s, s * (1.f - s)};
    } else if constexpr (ACT == ACT_SILU) {
        const float s = sigmoid_of<FAST>(z);
        return ActPair{z * s, s * (1.f + z * (1.f - s))};
    } else if constexpr (ACT == ACT_GELU) {  // z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2: no cancellation at the lower end
        const float gauss = exp_of<FAST>(-0.5f * z * z);
        float phi;
        if constexpr (FAST) {
            const float t = __builtin_amdgcn_rcpf(1.f + 0.42f * 0.70710678f * fabsf(z));
            const float lower = 0.5f * gauss * t *
                                (0.23817688f + t * (0.21978962f + t * (0.31046286f + t * (-0.0839581f + t * (0.47992118f + t * -0.16439275f)))));
            phi = z < 0.f ? lower : 1.f - lower;
        } else {
            phi = 0.5f * erfcf(-0.70710678118654752f * z);
        }
        return ActPair{z * phi, phi + z * 0.3989422804014327f * gauss};
    } else if constexpr (ACT == ACT_GELU_TANH) {  // (1 + tanh y) / 2 = sigmoid(2 y), y = c (z + 0.044715 z^3)
        const float c2 = 2.f * 0.7978845608028654f, q = 0.044715f * z * z;
        const float s = sigmoid_of<FAST>(c2 * z * (1.f + q)), w = s * (1.f - s);
        return ActPair{z * s, s + (w == 0.f ? 0.f : z * w * (c2 * (1.f + 3.f * q)))};
    } else {
        return ActPair{z, 1.f};
    }
}
// Eight of them behind one decision (one for each value took the epilogue of a 256-tile 8 us, for a relu).
template <bool FAST>
__device__ __forceinline__ void activate8(int act, const float (&z)[8], float (&a)[8], float (&d)[8]) {
    auto all = [&](auto act_c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const ActPair p = activate<FAST, decltype(act_c)::value>(z[e]);
            a[e] = p.a;
            d[e] = p.d;
        }
    };
    switch (act) {
        case ACT_RELU: return all(std::integral_constant<int, ACT_RELU>{});
        case ACT_SIGMOID: return all(std::integral_constant<int, ACT_SIGMOID>{});
        case ACT_SILU: return all(std::integral_constant<int, ACT_SILU>{});
        case ACT_GELU: return all(std::integral_constant<int, ACT_GELU>{});
        case ACT_GELU_TANH: return all(std::integral_constant<int, ACT_GELU_TANH>{});
        default: return all(std::integral_constant<int, ACT_NONE>{});
    }
}

// ---- eight values of a row ----------------------------------------------------------------------
// Read and written whole where there are eight, at any address (common.h), and one by one at the end of a row.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef u32x2 __attribute__((aligned(1))) u32x2_any;
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[8]) {
    if (count >= 8) {
        if constexpr (sizeof(T) == 2) {
            const bf16x8 w = *(const bf16x8_any*)p;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = bf2f(w[e]);
        } else {
            const f32x4 lo = *(const f32x4_any*)p, hi = *(const f32x4_any*)(p + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = lo[e], v[e + 4] = hi[e];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? (float)p[e] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[8]) {
    if (count >= 8) {
        if constexpr (sizeof(T) == 2) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
            *(u32x4_any*)p = w;
        } else {
            *(f32x4_any*)p = f32x4{v[0], v[1], v[2], v[3]};
            *(f32x4_any*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < count) p[e] = (T)v[e];
}

// Factors that are kept for the backward pass of bf16 tensors: each rounded to its upper 24 bits, in a plane of the upper 16 and one of the
// other 8.  So they are off by 2^-16 at most, to either side (cut off: 2^-15, all towards zero, which sums over rows do not even out).  Rounded
// to bf16 like any activation they are off by 2^-8, as much as the rounding of dy * d behind them, and gradients then were 1.7 times as far
// from the formula's as results that are rounded once (2.9e-3 against 1.66e-3 in the 2-norm; so it is 2.35e-3).
// The third byte costs 2 % of a gated training step over 8192 x 4096 x 12288 and half as much memory again; fp32 tensors keep all 32 bits.
template <typename T>
__device__ __forceinline__ void keep8(void* base, long all, long at, int count, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        store8((float*)base + at, count, v);
    } else {
        uint16_t* high = (uint16_t*)base + at;
        uint8_t* low = (uint8_t*)base + 2 * all + at;
        uint32_t b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = __builtin_bit_cast(uint32_t, v[e]) + 0x80;  // (a NaN stays one: its lower half is zero, as the bf16 value's that it comes from)
        if (count >= 8) {
            u32x4 h;
            u32x2 l;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __builtin_amdgcn_perm(b[2 * e + 1], b[2 * e], 0x07060302);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                l[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[4 * e + 3], b[4 * e + 2], 0x0c0c0501), __builtin_amdgcn_perm(b[4 * e + 1], b[4 * e], 0x0c0c0501),
                                             0x05040100);
            *(u32x4_any*)high = h;
            *(u32x2_any*)low = l;
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) high[e] = (uint16_t)(b[e] >> 16), low[e] = (uint8_t)(b[e] >> 8);
    }
}
template <typename T>
__device__ __forceinline__ void kept8(const void* base, long all, long at, int count, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        load8((const float*)base + at, count, v);
    } else {
        const uint16_t* high = (const uint16_t*)base + at;
        const uint8_t* low = (const uint8_t*)base + 2 * all + at;
        if (count >= 8) {
            const u32x4 h = *(const u32x4_any*)high;
            const u32x2 l = *(const u32x2_any*)low;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t top = e & 1 ? h[e >> 1] & 0xffff0000u : h[e >> 1] << 16;
                v[e] = __builtin_bit_cast(float, top | ((l[e >> 2] >> (8 * (e & 3))) & 0xffu) << 8);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < count ? __builtin_bit_cast(float, (uint32_t)high[e] << 16 | (uint32_t)low[e] << 8) : 0.f;
    }
}

// The layer's arithmetic on eight sums of row i, columns j .. j + 7 (of both factors of a gated pair), and their way to memory.
template <typename T, bool GATED>
__device__ __forceinline__ void finish8(const KernelArgs& g, int z, long i, int j, float (&v)[8], float (&u)[8]) {
    const int count = g.n - j < 8 ? g.n - j : 8;
    const long at = i * g.n + j, all = (long)g.m * g.n;
    auto add = [&](float (&x)[8], const void* base, long off) {
        float b[8];
        load8((const T*)base + off, count, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] += b[e];
    };
    if (g.bias[0]) add(v, g.bias[0], j);
    if constexpr (GATED) {
        if (g.bias[1]) add(u, g.bias[1], j);
        float h[8], s[8], t[8];
        activate8<sizeof(T) == 2>(g.act, v, s, t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[e] = s[e] * u[e];
            t[e] *= u[e];
        }
        store8((T*)g.out[0] + at, count, h);
        if (g.aux[0]) {
            keep8<T>(g.aux[0], all, at, count, s);
            keep8<T>(g.aux[1], all, at, count, t);
        }
    } else {
        if (g.act != ACT_NONE) {
            float z8[8], d[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z8[e] = v[e];
            activate8<sizeof(T) == 2>(g.act, z8, v, d);
            if (g.aux[0]) keep8<T>(g.aux[0], all, at, count, d);
        }
        if (g.residual) {
            const T* r = (const T*)g.residual + i * g.res_row + j * g.res_col;
            if (g.res_col == 1) {
                add(v, r, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < count) v[e] += (float)r[e * g.res_col];
            }
        }
        store8((T*)g.out[z] + at, count, v);
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
    store8(p, count, v);
    if (GATED) store8(p + (long)g.m * g.n, count, u);
}

// ---- operand tiles in LDS -------------------------------------------------------------------------
// A k-tile of an operand of R rows takes R * 128 bytes, in one of two orders:
//   rows   row r holds its 8 pieces of 16 bytes; piece c lies at place c ^ swizzle(r)
//   steps  reduction step k holds R values; 16-byte piece c lies at place c ^ swizzle(k)
// The loads write LDS in lane order, so the exchange happens on the side of memory: a lane fetches the piece whose place is its own.
//
// Fragments: lane l takes row l % 16 of a fragment and the reduction steps of group l / 16, and holds four neighbouring columns of the result.
//
// The swizzles: reads are served 16 lanes (16-byte reads) or 32 lanes (8-byte transposing reads) at a time, and the lanes that are served
// together are to touch different banks: sixteen rows of one step group, and the 32-byte pieces of eight reduction steps.
__device__ __forceinline__ int swizzle_rows(int r) { return (r >> 1) & 7; }
template <typename T, int R>
__device__ __forceinline__ int swizzle_steps(int k) {
    if constexpr (sizeof(T) == 2) return R >= 128 ? ((k & 3) | ((k >> 3) & 1) << 2) << 1 : (((k >> 1) & 1) | ((k >> 3) & 1) << 1) << 1;
    else return ((k >> 2) & 3) << 2;
}

// Where a lane finds its parts of the F fragments of its wave, whose rows start at `first`: as few addresses as the swizzle allows, everything
// else is a constant that fits a read's offset (a k-tile half h, and the stages of an operand, which lie one behind the other).
template <typename T, int R, bool STEPS, int F>
struct Reader {
    static constexpr bool HALF = sizeof(T) == 2;
    static constexpr int N = STEPS ? F : 2;
    unsigned at[N];
    __device__ __forceinline__ void init(unsigned base, int first, int lane) {
        const int i = lane & 15, grp = lane >> 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (!STEPS) {  // n: half of the k-tile
                const int r = first + i;
                at[n] = base + r * ROWB + (((n * 4 + grp) ^ swizzle_rows(r)) << 4);
            } else if constexpr (HALF) {
                // lane i of a group of 16 addresses piece i (step i / 4, rows of quarter i % 4) and receives row i of steps 0 to 3
                const int k = grp * 8 + (i >> 2), r = first + n * 16 + (i & 3) * 4;
                at[n] = base + k * (R * 2) + (((r >> 3) ^ swizzle_steps<T, R>(k)) << 4) + (r & 4) * 2;
            } else {
                const int k = grp * 4, r = first + n * 16 + i;
                at[n] = base + k * (R * 4) + (((r >> 2) ^ swizzle_steps<T, R>(k)) << 4) + (r & 3) * 4;
            }
        }
    }
    __device__ __forceinline__ void move(int bytes) {
#pragma unroll
        for (int n = 0; n < N; ++n) at[n] += bytes;
    }
    __device__ __forceinline__ typename Elem<T>::frag read(const unsigned char* smem, int f, int h) const {
        if constexpr (!STEPS) {
            return *(const typename Elem<T>::frag*)(smem + at[h] + f * 16 * ROWB);
        } else if constexpr (HALF) {
            s16x4 part[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const unsigned char* q = smem + at[f] + (h * 32 + p * 4) * (R * 2);
                part[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_void_ptr)q);
            }
            const s16x8 w = {part[0][0], part[0][1], part[0][2], part[0][3], part[1][0], part[1][1], part[1][2], part[1][3]};
            return __builtin_bit_cast(bf16x8, w);
        } else {
            f32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = *(const float*)(smem + at[f] + (h * 16 + e) * (R * 4));
            return w;
        }
    }
};

// Two fragments side by side, of which a lane holds four columns each (4 q .. 4 q + 3 of its 16, q the lane's sixteenth): afterwards it holds
// eight neighbouring columns, 16 (q % 2) + 8 (q / 2) .. + 7 of their 32, so that results leave in 16-byte pieces without a trip through LDS.
__device__ __forceinline__ void pair_columns(f32x4& lo, f32x4& hi) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float a = lo[r], b = hi[r];  // (a cast of a vector's element is one of its first element)
        const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
        const unsigned c = s[0], d = s[1];
        lo[r] = __builtin_bit_cast(float, c);
        hi[r] = __builtin_bit_cast(float, d);
    }
}

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
template <typename T, int R, int NW, bool STEPS, bool GATED>
struct Feed {
    static constexpr int LOADS = R / 8 / NW;  // wave instructions of 1 KB
    static constexpr int BK = Elem<T>::BK, PIECE = Elem<T>::PIECE, PIECES = R / PIECE;
    static_assert(R % (8 * NW) == 0, "whole instructions");
    static_assert(!GATED || !STEPS, "the factors of a gated pair are interleaved by rows");
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
                const int line = at * 8 + (lane >> 3), c = (lane & 7) ^ swizzle_rows(line);
                const int src = GATED ? (line >> 6) * 32 + (line & 31) : line;
                off[n] = src * step_bytes + c * 16;
            } else {
                const int idx = at * 64 + lane, step = idx / PIECES, c = (idx % PIECES) ^ swizzle_steps<T, R>(step);
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
            if constexpr (!STEPS) keep = left - ((lane & 7) ^ swizzle_rows(idx >> 3)) * PIECE;
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
    typedef Feed<T, BM, NW, ASTEPS, false> FeedA;
    typedef Feed<T, BN, NW, BSTEPS, GATED> FeedB;
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
        for (int j = 0; j < FN; j += 2) pair_columns(sums[j], sums[j + 1]);
#pragma unroll
        for (int jp = 0; jp < FN / 2; jp += GATED ? 2 : 1) {
            const long col = t.n0 + col0 + jp * 32 + (quad & 1) * 16 + (quad >> 1) * 8;
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
// What seems to bound them (from times, no counter) is the way from the caches to LDS, 11 to 12 TB/s over the machine for rows as tensors
// have them: 32 KB a k-tile of a 128-tile take 0.63 us while it has its compute unit for itself (its matrix instructions 0.25), so it
// reaches 0.75 PFLOP/s where a 256-tile, which needs half as much for the same work, reaches twice that.  Fragments of the next half read
// ahead of the products: 10 to 20 % slower; two k-tiles to a barrier: nothing.
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
    Reader<T, BM, ASTEPS, FM> ra;
    Reader<T, BN, BSTEPS, FN> rb;
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
            const int free = s == 0 ? S - 1 : s - 1;
            if constexpr (sizeof(T) == 2) {
                // Every fragment of the k-tile first, then the loads, whose addresses are worked out while the reads are on their way
                // (4096 x 4096 x 1024 on 128-tiles 45 us, 49 to 53 half by half).
                frag va[2][FM], vb[2][FN];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < FM; ++i) va[h][i] = ra.read(smem, i, h);
#pragma unroll
                    for (int j = 0; j < FN; ++j) vb[h][j] = rb.read(smem, j, h);
                }
                __builtin_amdgcn_sched_barrier(0);
                issue(kt + S - 1, free);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int i = 0; i < FM; ++i) acc[i][j] = mfma_step(vb[h][j], va[h][i], acc[i][j]);
            } else {
                // Four instructions for each pair of fragments are time enough for the reads of the next (4096 x 4096 x 4096 966 us, all of
                // them first 986).
                issue(kt + S - 1, free);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    frag va[FM], vb[FN];
#pragma unroll
                    for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, i, h);
#pragma unroll
                    for (int j = 0; j < FN; ++j) vb[j] = rb.read(smem, j, h);
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int i = 0; i < FM; ++i) acc[i][j] = mfma_step(vb[j], va[i], acc[i][j]);
                }
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
//
// Measured, 8192 x 12288 x 4096 (rows against rows): two stages each and one k-tile of distance 1320 TFLOP/s, this 1450 to 1570, as much as the
// library's product of the same matrices (1540 to 1600); gradients, whose operands come through transposing reads, 1230 to 1430 (the
// library 1130 to 1330).  64 KB a k-tile are 12 TB/s over the machine, as in the small tiles.  Loads or fragments of the right operand
// moved into the multiplying phases cost 10 %, a higher priority for those phases does nothing.
template <typename T, bool ASTEPS, bool BSTEPS, bool GATED>
__global__ void __launch_bounds__(512, 2) product_pp_kernel(const KernelArgs g) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int BM = 256, BN = 256, WGM = 2, WGN = 4, NW = WGM * WGN;
    constexpr int WTM = BM / WGM, WTN = BN / WGN, FM = WTM / 16, FN = WTN / 16;
    constexpr int UNIT_A = BM * ROWB, UNIT_B = BN * ROWB, A_AT = 2 * UNIT_B;  // stages; the left operand's lie behind the right one's
    static_assert(WTN == 64, "a wave of a gated pair holds 32 columns of each factor");
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

    Reader<T, BM, ASTEPS, FM> ra;
    Reader<T, BN, BSTEPS, FN> rb;
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
            for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, i, 0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < FN; ++j) vb[h][j] = rb.read(smem, j, h);
            panels.issue_a(kt + 2, t.last, lds + slot_a(sa2));
            WAIT_LDS();
            fence();
            multiply(va, vb[0]);
            fence();
#pragma unroll
            for (int i = 0; i < FM; ++i) va[i] = ra.read(smem, i, 1);
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
// are multiplied.  The waves' sums meet in LDS.  Rows may start at any element: the hardware reads vectors from any address.  Bound by
// memory: two factors of 12288 x 4096, 201 MB, take 40 us (5.0 TB/s), one 21.  Deeper batches in one workgroup a compute unit: 41 and 23.
template <typename T, bool GATED>
__global__ void __launch_bounds__(512, 4) product_rows_kernel(const KernelArgs g) {
    typedef typename Elem<T>::frag frag;
    typedef frag __attribute__((aligned(sizeof(T)))) frag_any;
    constexpr int W = GATED ? 2 : 1, NW = 8, PIECE = Elem<T>::PIECE, STEP = 4 * PIECE;  // reduction steps of a fragment
    constexpr int STEPS = GATED ? 3 : 4;  // (in the registers that two workgroups of a compute unit have)
    __shared__ __align__(16) float part[NW][W][16][16];
    // (Matrix instructions run whichever lanes are switched on: what decides over them has to be known to be the same in all of a wave's.)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, grp = lane >> 4;
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
    const long pieces = (g.n + 7L) / 8, all = pieces * g.m * g.outs;
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
            load8(p, count, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += w[e];
            if (GATED) {
                load8(p + (long)g.m * g.n, count, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] += w[e];
            }
        }
        finish8<T, GATED>(g, z, i, j, v, u);
    }
}

// ---- packing ------------------------------------------------------------------------------------
// Operands whose lines are no whole 16-byte pieces, copied to lines `pitch` values apart (what lies past a line's end is left as it is: the
// products clear it).  A line is a row or a reduction step, whichever is contiguous; a thread copies a piece, the matrices of a product one
// after the other.
struct PackJob {
    const void* src;
    void* dst;
    long stride, pitch;  // between lines
    long first;          // piece of the launch that the job starts with
    int lines, length;
};
struct PackList {
    int n;
    long pieces;
    PackJob job[4];
};
template <typename T>
__global__ void __launch_bounds__(256) product_pack_kernel(const PackList l) {
    constexpr int PIECE = 16 / sizeof(T);
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    if (at >= l.pieces) return;
    int n = 0;
    while (n + 1 < l.n && at >= l.job[n + 1].first) ++n;
    const PackJob& j = l.job[n];
    const long each = (j.length + PIECE - 1) / PIECE, line = (at - j.first) / each;
    const int c = (int)((at - j.first) - line * each) * PIECE;
    const T* src = (const T*)j.src + line * j.stride + c;
    T* dst = (T*)j.dst + line * j.pitch + c;
    if (c + PIECE <= j.length) {
        if constexpr (sizeof(T) == 2) *(bf16x8*)dst = *(const bf16x8_any*)src;
        else *(f32x4*)dst = *(const f32x4_any*)src;
    } else {
        for (int e = 0; c + e < j.length; ++e) dst[e] = src[e];
    }
}
// rows x cols values of any strides into rows `pitch` apart: 64 x 64 of them go through LDS, read along the nearer stride.
template <typename T>
__global__ void __launch_bounds__(256) product_gather_kernel(const T* src, long row, long col, int rows, int cols, T* dst, long pitch, int along) {
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
// dz is an operand of two products, whose matrix instructions take the tensors' type, and is rounded to it (bf16: 2^-8 of each value at most);
// the sums over rows add the values before that.
// A workgroup takes 256 columns (32 threads, eight columns each) of `rows` rows, eight at a time.  Bound by memory: the pair of gradients of
// 8192 x 12288 bf16 values, 12 bytes a value, takes 245 us (4.9 TB/s, the rate of a copy).
template <typename T, bool PAIR>
__global__ void __launch_bounds__(256) act_grad_kernel(const ActGradArgs g, int chunks, int rows) {
    constexpr int F = PAIR ? 2 : 1;
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int blocks = (int)((g.n + 255L) / 256);
    const int chunk = blockIdx.x / blocks, j0 = (blockIdx.x - chunk * blocks) * 256, j = j0 + tx * 8;
    const int count = g.n - j < 8 ? g.n - j : 8;
    const long all = (long)g.m * g.n;
    float sum[F][8] = {};
    if (j < g.n) {
        const long r0 = (long)chunk * rows;
#pragma unroll 2
        for (int s = ty; s < rows; s += 8) {
            const long i = r0 + s;
            if (i >= g.m) break;
            float dy[8];
            load8((const T*)g.dy + i * g.n + j, count, dy);
#pragma unroll
            for (int f = 0; f < F; ++f) {
                float v[8];
                if (g.factors > f) {
                    kept8<T>(g.d[f], all, i * g.n + j, count, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= dy[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = dy[e];
                }
                if (g.dz[f]) store8((T*)g.dz[f] + i * g.pitch + j, count, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[f][e] += v[e];
            }
        }
    }
    if (!g.partials) return;
    __shared__ float part[8][32][9];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        if (!g.db[f]) continue;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) part[ty][tx][e] = sum[f][e];
        __syncthreads();
        const int c = threadIdx.x;
        if (j0 + c < g.n) {
            float v = 0.f;
#pragma unroll
            for (int y = 0; y < 8; ++y) v += part[y][c >> 3][c & 7];
            g.partials[((long)f * chunks + chunk) * g.n + j0 + c] = v;
        }
    }
}
// Sixteen rows of threads take the parts of sixteen columns in turn; their sums are added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) row_sum_kernel(const float* partials, int chunks, int n, T* out0, T* out1) {
    __shared__ float part[16][16];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4, f = blockIdx.y;
    T* out = f ? out1 : out0;
    if (!out) return;
    for (long j0 = blockIdx.x * 16L; j0 < n; j0 += gridDim.x * 16L) {
        const long j = j0 + x;
        float v = 0.f;
        if (j < n) {
#pragma unroll 4
            for (int c = y; c < chunks; c += 16) v += partials[((long)f * chunks + c) * n + j];
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

// ---- host side ----------------------------------------------------------------------------------------
inline long up(long v, long m) { return (v + m - 1) / m * m; }
constexpr long MOST_THREADS = 0xffffffffL;  // of a launch
inline int elem_size(int dtype) { return dtype == MUON_HIP_BF16 ? 2 : 4; }

// How an operand is read: rows or reduction steps as they lie, or copies of them, or rows put together from any strides.
enum {
    LIE_ROWS = MUON_HIP_OPERAND_ROWS,
    LIE_STEPS = MUON_HIP_OPERAND_STEPS,
    LIE_PACKED_ROWS = MUON_HIP_OPERAND_ROWS_COPIED,
    LIE_PACKED_STEPS = MUON_HIP_OPERAND_STEPS_COPIED,
    LIE_GATHERED = MUON_HIP_OPERAND_GATHERED
};
inline bool by_steps(int lie) { return lie == LIE_STEPS || lie == LIE_PACKED_STEPS; }
struct Plan {
    int lie_a, lie_b;
    long pitch_a, pitch_b;        // elements
    long pack_a, pack_b;          // bytes of one packed matrix
    int count_a, count_b;         // matrices of each operand
    int tile, splits, per_split, nk, segments, outs;  // tile 0: the kernel of few rows
    long groups;                  // workgroups of the launch
    int threads;                  // of each
    long copies;                  // threads of the largest launch that packs
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
                              {{2.5f, 0.5f, 0.30f, 0.22f}, {3.f, 1.f, 0.62f, 0.50f}, {3.f, 3.f, 1.15f, 1.35f}}};  // bf16: 64, 128, 256
constexpr float kJoinStart = 4.f, kJoinBytes = 5.5e6f;  // of a split reduction: its launch, and bytes in a microsecond
constexpr int kTile[3] = {64, 128, 256};

// Threads of a workgroup of such a tile.  128-tiles of bf16 matrices that have a compute unit each take eight waves and four stages
// (4096 x 4096 x 1024: 45 us against 52); otherwise two workgroups of four waves share one.
inline int threads_of(int tile, int size, long groups, int cus) { return tile == 256 || (tile == 128 && size == 2 && groups <= cus) ? 512 : 256; }

// Lines may lie where 16-byte pieces of them are aligned and 31 bits span a tile's: 256 rows, or the 64 reduction steps of a k-tile.
int lie_of(const ProductOperand& o, int count, int rows, int k, int size, bool steps_ok, long& pitch) {
    const long piece = 16 / size, lines = rows < 256 ? rows : 256;
    auto fits = [&](long p, long lines) { return p % piece == 0 && p <= (0x7fff0000L / size) / lines; };
    bool rows_lie = k <= 0x7fff0000L / size, steps_lie = steps_ok, rows_run = true, steps_run = steps_ok;
    for (int i = 0; i < count; ++i) {
        const bool aligned = (((uintptr_t)o.base[i]) & 15) == 0;
        // (one row, or one step, has no stride that matters)
        rows_run = rows_run && (o.col[i] == 1 || k == 1);
        steps_run = steps_run && (o.row[i] == 1 || rows == 1);
        rows_lie = rows_lie && aligned && (rows == 1 || (fits(o.row[i], lines) && o.row[i] == o.row[0]));
        steps_lie = steps_lie && aligned && (k == 1 || (fits(o.col[i], 64) && o.col[i] == o.col[0]));
    }
    if (rows_lie && rows_run) {
        pitch = rows == 1 ? 0 : o.row[0];
        return LIE_ROWS;
    }
    if (steps_lie && steps_run) {
        pitch = k == 1 ? 0 : o.col[0];
        return LIE_STEPS;
    }
    const long row_pitch = up(k, piece), step_pitch = up(rows, piece);
    if (steps_run && (!rows_run || !fits(row_pitch, lines)) && fits(step_pitch, 64)) {
        pitch = step_pitch;
        return LIE_PACKED_STEPS;
    }
    pitch = row_pitch;
    return rows_run ? LIE_PACKED_ROWS : LIE_GATHERED;
}

// Few rows against rows of a weight, wherever they start: one launch, where tiles that leave most of the machine idle would have to share the
// reduction and be joined (1 x 4096 x 4096: 9 us against 14).  From 9 rows on the fragments of x are as much to fetch as the weight and the
// tiles, which keep theirs in LDS, are faster (16 x 4096 x 12288: 24 us against 30; a gated pair of 8 rows: 40 against 44, of 4 rows 40 both, of
// 4 x 4096 x 4096 18 against 16).
constexpr int kFewRows = 8, kFewRowsGated = 4;
bool few_rows(const ProductArgs& p, Plan& l) {
    if (p.kind == PRODUCT_GATED ? p.m > kFewRowsGated : p.kind != PRODUCT_LINEAR || p.m > kFewRows) return false;
    if (p.k > 16384 && p.n < 1024) return false;  // long rows on few compute units
    if (up(p.n, 16) / 16 * 512 > MOST_THREADS) return false;
    if (p.k > 1 && (p.a.col[0] != 1 || p.b.col[0] != 1)) return false;
    if (p.kind == PRODUCT_GATED && ((p.k > 1 && p.b.col[1] != 1) || p.b.row[1] != p.b.row[0])) return false;
    l.tile = 0;
    l.pitch_a = p.a.row[0];
    l.pitch_b = p.b.row[0];
    l.segments = l.outs = l.splits = 1;
    l.groups = up(p.n, 16) / 16;
    l.threads = 512;
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
    auto pack_bytes = [&](int lie, long pitch, long rows) {
        if (lie == LIE_ROWS || lie == LIE_STEPS) return 0L;
        if (lie != LIE_PACKED_STEPS && pitch > (0x7fff0000L / size) / (rows < 256 ? rows : 256)) return -1L;
        if (lie == LIE_GATHERED) l.copies = std::max(l.copies, up(p.k, 64) / 64 * (up(rows, 64) / 64) * 256);
        return up((lie == LIE_PACKED_STEPS ? p.k : rows) * pitch * size, 256);
    };
    l.pack_a = pack_bytes(l.lie_a, l.pitch_a, p.m);
    l.pack_b = pack_bytes(l.lie_b, l.pitch_b, p.n);
    if (l.pack_a < 0 || l.pack_b < 0) return false;
    auto pieces = [&](int lie, long rows, int count) {  // of lines that are copied whole, a thread each
        const long length = lie == LIE_PACKED_STEPS ? rows : p.k, lines = lie == LIE_PACKED_STEPS ? p.k : rows;
        return lie == LIE_PACKED_ROWS || lie == LIE_PACKED_STEPS ? up(length, 16 / size) / (16 / size) * lines * count : 0L;
    };
    l.copies = std::max(l.copies, up(pieces(l.lie_a, p.m, l.count_a) + pieces(l.lie_b, p.n, l.count_b), 256));
    if (l.copies > MOST_THREADS) return false;
    l.nk = (int)((p.k + (long)bk - 1) / bk);
    auto tiles_of = [&](int t) { return up(p.m, t) / t * (up(p.n, gated ? t / 2 : t) / (gated ? t / 2 : t)) * l.outs; };
    const long all = (long)l.nk * l.segments;
    if (all > 0x3fffffffL) return false;
    const bool bf = p.dtype == MUON_HIP_BF16;
    float best = 1e30f;
    for (int c = 0; c < (bf ? 3 : 2); ++c) {
        const long here = tiles_of(kTile[c]);
        const Cost& q = kCost[bf][c];
        for (int want : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (want > 1 && (want > all / 4 || here * want > 8L * cus)) break;
            const long per = (all + want - 1) / want, parts = (all + per - 1) / per;
            if (here * parts > MOST_THREADS / threads_of(kTile[c], size, here * parts, cus)) break;
            const long load = (here * parts + cus - 1) / cus;
            float t = q.start + q.each * load + (float)per * (load <= 1 ? q.alone : std::max(q.alone, q.busy * load));
            if (parts > 1) t += kJoinStart + (float)p.m * p.n * (gated ? 2 : l.outs) * 8.f * parts / kJoinBytes;
            if (t < best) {
                best = t;
                l.tile = kTile[c];
                l.per_split = (int)per;
                l.splits = (int)parts;
                l.groups = here * parts;
                l.threads = threads_of(kTile[c], size, l.groups, cus);
            }
        }
    }
    if (l.tile == 0) return false;
    if (l.splits > 1) l.partial_bytes = (long)l.splits * (gated ? 2 : l.outs) * p.m * p.n * 4;
    l.bytes = l.pack_a * l.count_a + l.pack_b * l.count_b + l.partial_bytes;
    return true;
}

template <typename T, int BM, int BN, int WGM, int WGN, int S, bool AS, bool BS, bool GATED>
hipError_t launch_tiles(const KernelArgs& g, const Plan& l, hipStream_t stream) {
    constexpr int smem = S * (BM + BN) * ROWB;
    static std::atomic<unsigned long long> configured{0};
    const auto kern = product_kernel<T, BM, BN, WGM, WGN, S, AS, BS, GATED>;
    if (hipError_t e = allow_dynamic_lds((const void*)kern, smem, configured); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)l.groups), dim3(WGM * WGN * 64), smem, stream, g);
    return hipGetLastError();
}
template <typename T, bool AS, bool BS, bool GATED>
hipError_t launch_pp(const KernelArgs& g, const Plan& l, hipStream_t stream) {
    constexpr int smem = 5 * 256 * ROWB;
    static std::atomic<unsigned long long> configured{0};
    const auto kern = product_pp_kernel<T, AS, BS, GATED>;
    if (hipError_t e = allow_dynamic_lds((const void*)kern, smem, configured); e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)l.groups), dim3(512), smem, stream, g);
    return hipGetLastError();
}
template <typename T, bool AS, bool BS, bool GATED>
hipError_t launch_tile(const KernelArgs& g, const Plan& l, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (l.tile == 256) return launch_pp<T, AS, BS, GATED>(g, l, s);
        if (l.tile == 128 && l.threads == 512) return launch_tiles<T, 128, 128, 4, 2, 4, AS, BS, GATED>(g, l, s);
    }
    if (l.tile == 128) return launch_tiles<T, 128, 128, 2, 2, 2, AS, BS, GATED>(g, l, s);
    return launch_tiles<T, 64, 64, 4, 1, 3, AS, BS, GATED>(g, l, s);
}
template <typename T, bool GATED>
hipError_t launch_rows(const KernelArgs& g, const Plan& l, hipStream_t s) {
    hipLaunchKernelGGL((product_rows_kernel<T, GATED>), dim3((unsigned)l.groups), dim3(l.threads), 0, s, g);
    return hipGetLastError();
}

template <typename T>
hipError_t run_product(const ProductArgs& p, const Plan& l, void* workspace, int xcd_shift, hipStream_t s) {
    constexpr int S = sizeof(T);
    const bool gated = p.kind == PRODUCT_GATED;
    KernelArgs g{};
    char* ws = (char*)workspace;
    PackList copies{};
    auto pack = [&](const ProductOperand& o, int lie, int count, int rows, long pitch, long bytes, const void** at) {
        for (int i = 0; i < count; ++i) {
            at[i] = o.base[i];
            if (bytes == 0) continue;
            if (lie == LIE_GATHERED) {
                const dim3 grid((unsigned)(up(p.k, 64) / 64 * (up(rows, 64) / 64)));
                hipLaunchKernelGGL(product_gather_kernel<T>, grid, dim3(256), 0, s, (const T*)o.base[i], o.row[i], o.col[i], rows, p.k, (T*)ws, pitch,
                                   (int)(o.row[i] < o.col[i]));
                if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            } else {
                const bool steps = lie == LIE_PACKED_STEPS;
                PackJob& j = copies.job[copies.n++];
                j = PackJob{o.base[i], ws, steps ? o.col[i] : o.row[i], pitch, copies.pieces, steps ? p.k : rows, steps ? rows : p.k};
                copies.pieces += j.lines * (up(j.length, 16 / S) / (16 / S));
            }
            at[i] = ws;
            ws += bytes;
        }
        return hipSuccess;
    };
    g.m = p.m;
    g.n = p.n;
    g.k = p.k;
    g.outs = l.outs;
    // No activation, but its factor to write: a code of its own that computes nothing either, so that the epilogue has one decision to make
    // (24 x 12288 x 4096 in four parts: 25.0 us, with two of them 25.3).
    g.act = p.act == ACT_NONE && p.aux[0] ? ACT_COUNT : p.act;
    for (int i = 0; i < 2; ++i) {
        g.bias[i] = p.bias[i];
        g.out[i] = p.out[i];
        g.aux[i] = p.aux[i];
    }
    g.residual = p.residual;
    g.res_row = p.res_row;
    g.res_col = p.res_col;
    g.xcd_shift = xcd_shift;
    if (p.k > 0) {
        if (hipError_t e = pack(p.a, l.lie_a, l.count_a, p.m, l.pitch_a, l.pack_a, g.a); e != hipSuccess) return e;
        if (hipError_t e = pack(p.b, l.lie_b, l.count_b, p.n, l.pitch_b, l.pack_b, g.b); e != hipSuccess) return e;
        if (copies.n > 0) {
            hipLaunchKernelGGL(product_pack_kernel<T>, dim3((unsigned)(up(copies.pieces, 256) / 256)), dim3(256), 0, s, copies);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
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
        const bool as = by_steps(l.lie_a), bs = by_steps(l.lie_b);
        hipError_t e;
        if (l.tile == 0) e = gated ? launch_rows<T, true>(g, l, s) : launch_rows<T, false>(g, l, s);
        else if (gated) e = as ? launch_tile<T, true, false, true>(g, l, s) : launch_tile<T, false, false, true>(g, l, s);
        else if (as) e = bs ? launch_tile<T, true, true, false>(g, l, s) : launch_tile<T, true, false, false>(g, l, s);
        else e = bs ? launch_tile<T, false, true, false>(g, l, s) : launch_tile<T, false, false, false>(g, l, s);
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

bool plan_product(const ProductArgs& p, int cus, muon_hip_product_route& out) {
    Plan l;
    if (!make_plan(p, cus, l)) return false;
    out = muon_hip_product_route{l.tile, l.splits, l.lie_a, l.lie_b, l.groups, l.threads, l.copies};
    return true;
}

hipError_t launch_product(const ProductArgs& p, void* workspace, int cus, int xcd_shift, hipStream_t stream) {
    Plan l;
    if (!make_plan(p, cus, l)) return hipErrorInvalidValue;
    if (p.m == 0 || p.n == 0) return hipSuccess;
    return p.dtype == MUON_HIP_BF16 ? run_product<bf16_t>(p, l, workspace, xcd_shift, stream) : run_product<float>(p, l, workspace, xcd_shift, stream);
}

// Rows of a workgroup: as many as leave the machine enough of them, so that small gradients are not a loop and large ones have few parts.
static long act_grad_groups(long m, long n, long rows) { return up(m, rows) / rows * (up(n, 256) / 256); }
static long act_grad_rows(long m, long n) {
    long rows = 64;
    while (rows > 8 && act_grad_groups(m, n, rows) < 1024) rows /= 2;
    while (rows < (1 << 20) && act_grad_groups(m, n, rows) > MOST_THREADS / 256) rows *= 2;  // (more than a launch has)
    return rows;
}
bool act_grad_fits(long m, long n) { return act_grad_groups(m, n, act_grad_rows(m, n)) <= MOST_THREADS / 256; }
long act_grad_partials(long m, long n) {
    const long rows = act_grad_rows(m, n);
    return up(m, rows) / rows * n;
}

hipError_t launch_act_grad(const ActGradArgs& a, hipStream_t stream) {
    const bool pair = a.factors > 1;
    const long rows = act_grad_rows(a.m, a.n), chunks = up(a.m, rows) / rows, blocks = up(a.n, 256) / 256 * chunks;
    const bool bf = a.dtype == MUON_HIP_BF16;
    if (blocks > 0) {
        void (*kern)(const ActGradArgs, int, int);
        if (bf) kern = pair ? act_grad_kernel<bf16_t, true> : act_grad_kernel<bf16_t, false>;
        else kern = pair ? act_grad_kernel<float, true> : act_grad_kernel<float, false>;
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, a, (int)chunks, (int)rows);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if ((!a.db[0] && !a.db[1]) || a.n == 0) return hipSuccess;
    const dim3 grid((unsigned)std::min(up(a.n, 16) / 16, 65536L), pair ? 2 : 1);
    if (bf) hipLaunchKernelGGL(row_sum_kernel<bf16_t>, grid, dim3(256), 0, stream, a.partials, (int)chunks, a.n, (bf16_t*)a.db[0], (bf16_t*)a.db[1]);
    else hipLaunchKernelGGL(row_sum_kernel<float>, grid, dim3(256), 0, stream, a.partials, (int)chunks, a.n, (float*)a.db[0], (float*)a.db[1]);
    return hipGetLastError();
}
