// Pieces shared by the kernels that work row by row over channels (row_norm.hip, row_norm_grad.hip).  gfx950 only.
#pragma once
#include "ydet_internal.h"

namespace ydet {
namespace rows {

// A row of C values is held in registers by LPR lanes (a power of two: a part of a wave, a wave, or the 256 lanes of a
// workgroup), CH pieces of VEC values each; piece c of lane l starts at column (c * LPR + l) * VEC.  At most 32 values a lane.
constexpr int kMaxC = 8192;
constexpr int kThreads = 256;

struct Shape {
    int lpr, ch;
};
static inline int pow2_at_least(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}
// cols: values of a row that are read or written; vec: values of a 16-byte piece (8 or 4); rows up to wave_cols stay inside a wave
static inline Shape shape_of(int cols, int vec, int wave_cols) {
    const int n = (cols + vec - 1) / vec;
    if (n <= 64) {
        const int l = pow2_at_least(n);
        return Shape{l < 4 ? 4 : l, 1};
    }
    return n * vec <= wave_cols ? Shape{64, pow2_at_least((n + 63) / 64)} : Shape{256, pow2_at_least((n + 255) / 256)};
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);      // (every lane has a source)
}
// Combines the LPR <= 64 lanes of a group so that every lane holds the result; op is commutative and the tree is the same for
// every lane, so all lanes hold the same bits.  Neighbours by DPP inside 16 lanes, then by the lane-row swaps.
template <int LPR, typename F>
__device__ __forceinline__ unsigned lanes_reduce(unsigned v, F op) {
    if constexpr (LPR >= 2) v = op(v, dpp<0xB1>(v));       // quad_perm [1,0,3,2]
    if constexpr (LPR >= 4) v = op(v, dpp<0x4E>(v));       // quad_perm [2,3,0,1]
    if constexpr (LPR >= 8) v = op(v, dpp<0x141>(v));      // row_half_mirror
    if constexpr (LPR >= 16) v = op(v, dpp<0x140>(v));     // row_mirror
    if constexpr (LPR >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    if constexpr (LPR >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    return v;
}
struct AddF {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }
};
struct MaxU {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a > b ? a : b; }
};
// The same over a group of LPR lanes where LPR may be the whole workgroup: its four waves meet in LDS.  `red` has two slots
// of four words used in turn: a wave that writes a slot again has passed the barrier of the other one, which every wave
// reaches only after it has read this one.
template <int LPR, typename F>
__device__ __forceinline__ unsigned group_reduce(unsigned v, F op, unsigned (&red)[2][4], int& slot) {
    if constexpr (LPR <= 64) {
        return lanes_reduce<LPR>(v, op);
    } else {
        v = lanes_reduce<64>(v, op);
        if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
        __syncthreads();
        v = op(op(red[slot][0], red[slot][1]), op(red[slot][2], red[slot][3]));
        slot ^= 1;
        return v;
    }
}
template <int LPR>
__device__ __forceinline__ float group_sum(float v, unsigned (&red)[2][4], int& slot) {
    return __uint_as_float(group_reduce<LPR>(__float_as_uint(v), AddF{}, red, slot));
}

// a / b rounded once, with y the nearest number to 1 / b.  Markstein's step: q = a y, then q + (a - b q) y rounded once is the nearest
// number to the quotient, as long as the remainder is exact, which tiny a do not allow.
__device__ __forceinline__ float quotient(float a, float b, float y) {
    const float q = a * y;
    return fmaf(fmaf(-b, q, a), y, q);
}

// Nearest integer to v / s (ties to even), exactly, as a float's bits whose low byte is the integer.  The product with 1 / s
// is within 3e-5 of the quotient, so rounding it (adding 1.5 * 2^23 leaves the integer in the low bits) is right unless it
// lies that close to a border; there the remainder decides, which the fused multiply-add gives without error: near a
// border |v - r s| is about s / 2 and a multiple of s's last place.
constexpr float kRound = 12582912.f;        // 1.5 * 2^23
__device__ __forceinline__ unsigned quantise_exact(float v, float s, float inv) {
    float r = (v * inv + kRound) - kRound;
    const float d = fmaf(-r, s, v), d2 = 2.f * fabsf(d);
    if (d2 > s || (d2 == s && ((int)r & 1))) r += copysignf(1.f, d);
    return __float_as_uint(r + kRound);
}

// N values rounded the quick way into m; returns how far the worst of them lies from its integer, for the caller to round all
// exactly where one is next to a border (seldom).  pack_bytes: the low bytes of N such values as N / 4 words.
template <int N>
__device__ __forceinline__ float quantise_near(const float (&v)[N], float inv, unsigned (&m)[N]) {
    float near = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = v[i] * inv, k = t + kRound;
        near = fmaxf(near, fabsf(t - (k - kRound)));
        m[i] = __float_as_uint(k);
    }
    return near;
}
template <int N>
__device__ __forceinline__ void pack_bytes(const unsigned (&m)[N], unsigned (&out)[N / 4]) {
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
        const unsigned lo = __builtin_amdgcn_perm(m[4 * j + 1], m[4 * j], 0x0c0c0400u);
        const unsigned hi = __builtin_amdgcn_perm(m[4 * j + 3], m[4 * j + 2], 0x0c0c0400u);
        out[j] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
}

// A row's scale from its largest magnitude, given by its bits (a NaN is above an infinity, and that above every number): `given`
// is what the caller gets, s and inv what the values are quantised with.  A row below 127 * 2^-126 counts as zero, so that s is
// a normal number: its inv is 0, and so are its values.  bad: the row has a NaN or an infinity, hence no scale, and zeros.
struct RowScale {
    float given, s, inv;
    bool bad;
};
__device__ __forceinline__ RowScale row_scale(unsigned top) {
    const float amax = __uint_as_float(top);
    RowScale r;
    r.bad = top >= 0x7f800000u;
    const bool some = !r.bad && amax >= 127.f * 1.17549435e-38f;
    r.s = !some ? 1.f : amax < 1e-25f ? amax / 127.f : quotient(amax, 127.f, 1.f / 127.f);
    r.inv = some ? __builtin_amdgcn_rcpf(r.s) : 0.f;
    r.given = some ? r.s : r.bad ? __uint_as_float(0x7fc00000u) : 0.f;
    return r;
}

// A piece: VEC consecutive values, 16 bytes.  Rows may begin at any value's address (gfx950 moves 16 bytes from and to any
// address), so a row is dealt to the lanes the same way wherever it lies, and its result does not depend on that.  RAG: C is no
// multiple of VEC, and the row's last piece, `n` < VEC values of it, is moved value by value (zeros behind it).
template <typename T, int VEC, bool RAG>
struct Piece {
    typedef T type __attribute__((ext_vector_type(VEC)));
    typedef type loose __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ type load(const T* p, int n) {
        if (!RAG || n >= VEC) return *reinterpret_cast<const loose*>(p);
        type v{};
#pragma unroll
        for (int i = 0; i < VEC - 1; ++i)
            if (i < n) v[i] = p[i];
        return v;
    }
    static __device__ __forceinline__ void store(T* p, const type& v, int n) {
        if (!RAG || n >= VEC) {
            *reinterpret_cast<loose*>(p) = v;
            return;
        }
#pragma unroll
        for (int i = 0; i < VEC - 1; ++i)
            if (i < n) p[i] = v[i];
    }
    // whether value i of a piece with n values of the row left is one of them
    static __device__ __forceinline__ bool has(int i, int n) { return RAG ? i < n : n > 0; }
};

// The per-channel parameters (weight or bias) of a piece, of either type: `none` where there are none, zeros behind the row
template <int VEC, bool RAG>
__device__ __forceinline__ void load_params(const char* p, int dtype, int col, int n, float none, float* out) {
    if (dtype == YDET_BF16) {
        typedef Piece<__bf16, VEC, RAG> P;
        typename P::type v{};
        if (p && n > 0) v = P::load(reinterpret_cast<const __bf16*>(p) + col, n);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = !P::has(i, n) ? 0.f : p ? (float)v[i] : none;
    } else {
        typedef Piece<float, VEC, RAG> P;
        typename P::type v{};
        if (p && n > 0) v = P::load(reinterpret_cast<const float*>(p) + col, n);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = !P::has(i, n) ? 0.f : p ? v[i] : none;
    }
}

}  // namespace rows
}  // namespace ydet
