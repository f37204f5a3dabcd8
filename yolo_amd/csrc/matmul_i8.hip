// Product of rows held in 8 bits with weights held in 8 bits, a scale for every row and one for every output channel: the
// 1x1 convolution (a token-wise linear layer) in 8-bit integers, with the epilogue of the floating convolutions.
//
//   acc[m, n] = sum_k x[m, k] w[n, k]   (32-bit integers: exact, whatever the order)
//   y[m, n]   = act(acc * x_scale[m] * w_scale[n] + bias[n])  [+ res]          (or the residual before the activation)
//
// v_mfma_i32_16x16x64_i8: both operands are K-contiguous, a lane holds 16 consecutive k of one row.  Channels sit on the
// MFMA row, pixels on its column, and weight rows are fetched in an order that leaves a lane with whole runs of
// consecutive channels of one pixel, which it finishes and stores in 16-byte pieces.
#include "conv_common.h"
#include "rows_common.h"

namespace ydet {
namespace i8 {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const char* x;          // first value of the slice
    const float* xs;
    const char* w;          // [n_pad][kp], zero behind K and N
    const float* ws;        // n_pad values
    const float* bias;      // n_pad values, or null
    const char* res;
    char* y;
    int M, K, N, kp, n_pad;
    long long x_ld, y_ld, res_ld;
    int act, res_mode;
    float slope;
    int tiles_n;
};

__device__ __forceinline__ i32x4 mma(const i32x4& a, const i32x4& b, const i32x4& c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// Epilogue variants, fixed at compile time so that a lane's values run through straight-line code: SiLU or leaky (slope 1 is "no
// activation"), and where the residual goes in.
template <bool SILU, int RES>
struct Mode {
    static constexpr bool silu = SILU;
    static constexpr int res = RES;
};
template <typename F>
__device__ __forceinline__ void with_mode(const Args& a, F f) {
    if (a.act == YDET_ACT_SILU) {
        if (a.res_mode == YDET_RES_NONE) f(Mode<true, YDET_RES_NONE>{});
        else if (a.res_mode == YDET_RES_AFTER_ACT) f(Mode<true, YDET_RES_AFTER_ACT>{});
        else f(Mode<true, YDET_RES_BEFORE_ACT>{});
    } else {
        if (a.res_mode == YDET_RES_NONE) f(Mode<false, YDET_RES_NONE>{});
        else if (a.res_mode == YDET_RES_AFTER_ACT) f(Mode<false, YDET_RES_AFTER_ACT>{});
        else f(Mode<false, YDET_RES_BEFORE_ACT>{});
    }
}
template <typename M>
__device__ __forceinline__ float finish(float v, float r, const Args& a) {
    if constexpr (M::res == YDET_RES_BEFORE_ACT) v += r;
    if constexpr (M::silu) v = v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
    else v = v > 0.f ? v : v * a.slope;
    if constexpr (M::res == YDET_RES_AFTER_ACT) v += r;
    return v;
}

// Which channel of a group of 16 F (F fragments: F MFMA row blocks of 16) MFMA row (q, e) of fragment i holds.  A lane ends with the
// rows 4 q .. 4 q + 3 of every fragment; in this order they are pieces of PE consecutive channels (16 bytes of output), and the
// four lane groups' pieces lie side by side: one store writes 64 consecutive bytes of each of 16 pixels.
template <int PE>
__device__ __forceinline__ int channel_of(int i, int q, int e) {
    return PE == 8 ? (i >> 1) * 32 + q * 8 + (i & 1) * 4 + e : i * 16 + q * 4 + e;
}

// What a lane holds of one pixel in a group of 16 F channels: NP pieces of PE channels, piece k from channel n + 4 PE k on
// (n: the group's first channel + PE q).
template <typename OUT, int F>
struct Run {
    static constexpr int PE = F == 1 ? 4 : 16 / (int)sizeof(OUT), NP = 4 * F / PE, C = 4 * F;
    typedef OUT piece __attribute__((ext_vector_type(PE)));
    typedef piece loose __attribute__((aligned(sizeof(OUT))));      // (gfx950 moves 16 bytes from and to any address)
    piece r[NP];        // the residual

    template <typename M>
    __device__ __forceinline__ void load_residual(const Args& a, int m, int n) {
        if constexpr (M::res != YDET_RES_NONE) {
            const OUT* p = reinterpret_cast<const OUT*>(a.res) + m * a.res_ld + n;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                r[k] = piece{};
                if (m >= a.M) continue;
                if (n + 4 * PE * k + PE <= a.N) {
                    r[k] = *reinterpret_cast<const loose*>(p + 4 * PE * k);
                } else {
#pragma unroll
                    for (int e = 0; e < PE - 1; ++e)
                        if (n + 4 * PE * k + e < a.N) r[k][e] = p[4 * PE * k + e];
                }
            }
        }
    }
    // acc: the pieces' sums; ws, bias: their channels' scales and biases
    template <typename M>
    __device__ __forceinline__ void store(const Args& a, int m, int n, float xs, const int (&acc)[C], const float (&ws)[C], const float (&bias)[C]) {
        if (m >= a.M) return;
        OUT* y = reinterpret_cast<OUT*>(a.y) + m * a.y_ld + n;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            piece o;
#pragma unroll
            for (int e = 0; e < PE; ++e) {
                float rr = 0.f;
                if constexpr (M::res != YDET_RES_NONE) rr = (float)r[k][e];
                o[e] = (OUT)finish<M>(fmaf((float)acc[k * PE + e] * xs, ws[k * PE + e], bias[k * PE + e]), rr, a);
            }
            if (n + 4 * PE * k + PE <= a.N) {
                *reinterpret_cast<loose*>(y + 4 * PE * k) = o;
            } else {
#pragma unroll
                for (int e = 0; e < PE - 1; ++e)
                    if (n + 4 * PE * k + e < a.N) y[4 * PE * k + e] = o[e];
            }
        }
    }
};

// scales and biases of a run's channels, from memory or LDS (both arrays are padded to whole groups)
template <typename R>
__device__ __forceinline__ void load_channels(const float* ws, const float* bias, float (&s)[R::C], float (&b)[R::C]) {
#pragma unroll
    for (int k = 0; k < R::NP; ++k)
#pragma unroll
        for (int e = 0; e < R::PE; ++e) {
            s[k * R::PE + e] = ws[4 * R::PE * k + e];
            b[k * R::PE + e] = bias ? bias[4 * R::PE * k + e] : 0.f;
        }
}

// ---- tiles: BN channels x BM pixels, operands through LDS --------------------------------------------------------------
// LDS image of a stage: BN weight rows, then BM pixel rows, 128 bytes of K each; row r's 16-byte piece c lies at place
// c ^ ((r >> 1) & 7), so that the 16 rows a fragment read touches fall into 16 different places of the banks.  Stages are filled by
// LDS-DMA (eight rows an instruction), from rows at any 4-byte address and pitch; rows behind the last pixel and channels behind
// n_pad lie outside the buffer descriptors, which are checked word by word, and read as zeros.  NST stages; the fragments of a half stage are read while the previous half's MFMAs run.
// What bounds it: for long K the operands' way through L2 (52 us for 23104 x 4096 -> 512 with 256 x 192 tiles: 1.85 POP/s, the matrix
// units busy 37 % of the time; a library product of 8192^3 reaches 2.26 in bursts of eight and 2.5 in a long train), for short K
// the rows and the output (51 us for 409600 x 128 -> 128 with SiLU and residual: 5.1 TB/s), for many channels and short K the
// epilogue, about ten operations a value, two of them transcendental (73 us for 102400 x 256 -> 1024, the vector units busy 63 % of
// the time, where the rows have just been written and lie in the last-level cache; 93 where they come from memory, whose latency a
// tile of two stages does not hide; what the bytes are changes neither by more than the clock does).
template <typename OUT, int BN, int BM, int WAVES_N, int WAVES_M, int NST = 2>
__global__ __launch_bounds__(64 * WAVES_N * WAVES_M, 2) void tile_kernel(const Args a) {
    constexpr int NW = WAVES_N * WAVES_M, WN = BN / WAVES_N, WM = BM / WAVES_M, FN = WN / 16, FM = WM / 16;
    constexpr int RB = 128, STAGE = (BN + BM) * RB, LW = BN / 8 / NW, LX = BM / 8 / NW;
    static_assert(WN % 64 == 0 && BN % (8 * NW) == 0 && BM % (8 * NW) == 0, "tile shape");
    extern __shared__ __attribute__((aligned(128))) char smem[];
    char* const stages = smem + (2 * BN + BM) * 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WAVES_N, wm = wave / WAVES_N;
    const unsigned t = xcd_remap(blockIdx.x, gridDim.x);
    const int n0 = (int)(t % (unsigned)a.tiles_n) * BN, m0 = (int)(t / (unsigned)a.tiles_n) * BM;

    const long long w_span = (long long)(a.n_pad - n0) * a.kp, x_span = (long long)(a.M - 1 - m0) * a.x_ld + ((a.K + 3) & ~3);
    const unsigned cap = 0xffffffffu;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.w + (long long)n0 * a.kp), 0,
                                                                        (int)(w_span < cap ? (unsigned)w_span : cap), 0x00020000);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(a.x + m0 * a.x_ld), 0,
                                                                        (int)(x_span < cap ? (unsigned)x_span : cap), 0x00020000);
    const int halves = (a.K + 63) / 64, nk = (halves + 1) / 2;
    unsigned ow[LW], ox[LX];
#pragma unroll
    for (int j = 0; j < LW; ++j) {
        const int r = (j * NW + wave) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        const int chan = (r & ~63) + channel_of<Run<OUT, 4>::PE>((r >> 4) & 3, (r >> 2) & 3, r & 3);
        ow[j] = (unsigned)chan * (unsigned)a.kp + c * 16;
    }
#pragma unroll
    for (int j = 0; j < LX; ++j) {
        const int r = (j * NW + wave) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        ox[j] = (unsigned)r * (unsigned)a.x_ld + c * 16;
    }
    // scales of the tile's channels and rows, and the biases, wait in LDS in front of the stages: the epilogue reads memory for
    // the residual only
    float* sc = reinterpret_cast<float*>(smem);         // [BN] channel scales, [BN] biases, [BM] row scales
    {
        const float* none = nullptr;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.ws + n0), 0, (a.n_pad - n0) * 4, 0x00020000);
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.bias ? a.bias + n0 : none), 0,
                                                                            a.bias ? (a.n_pad - n0) * 4 : 0, 0x00020000);
        const __amdgpu_buffer_rsrc_t rr = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.xs + m0), 0, (BM < a.M - m0 ? BM : a.M - m0) * 4,
                                                                            0x00020000);
        for (int k = wave; k < (2 * BN + BM) / 64; k += NW) {
            __attribute__((address_space(3))) void* dst = (__attribute__((address_space(3))) void*)(sc + k * 64);
            // (whole offsets in the vector register: they may lie behind the extent, where zeros are read)
            if (k < BN / 64) __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 4, (k * 64 + lane) * 4, 0, 0, 0);
            else if (k < 2 * BN / 64) __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, dst, 4, ((k - BN / 64) * 64 + lane) * 4, 0, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rr, dst, 4, ((k - 2 * BN / 64) * 64 + lane) * 4, 0, 0, 0);
        }
    }
    // (kt's part may ride in the scalar offset: below K, it lies below every extent, of at least one row's K and of one channel's kp)
    auto issue = [&](int stage, int kt) {
        kt *= RB;
        char* dst = stages + stage * STAGE + wave * 1024;
#pragma unroll
        for (int j = 0; j < LW; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(dst + j * NW * 1024), 16, (int)ow[j],
                                                     kt, 0, 0);
#pragma unroll
        for (int j = 0; j < LX; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(dst + BN * RB + j * NW * 1024), 16,
                                                     (int)ox[j], kt, 0, 0);
    };
    int fo[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) fo[kk] = (lane & 15) * RB + (((kk * 4 + (lane >> 4)) ^ ((lane & 15) >> 1)) * 16);
    i32x4 fa[2][FN], fb[2][FM], acc[FN][FM];
    auto read = [&](int stage, int kk, i32x4 (&A)[FN], i32x4 (&B)[FM]) {
        const char* pw = stages + stage * STAGE + wn * WN * RB + fo[kk];
        const char* px = stages + stage * STAGE + (BN + wm * WM) * RB + fo[kk];
#pragma unroll
        for (int i = 0; i < FN; ++i) A[i] = *reinterpret_cast<const i32x4*>(pw + i * 16 * RB);
#pragma unroll
        for (int j = 0; j < FM; ++j) B[j] = *reinterpret_cast<const i32x4*>(px + j * 16 * RB);
    };
    auto product = [&](const i32x4 (&A)[FN], const i32x4 (&B)[FM]) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = mma(A[i], B[j], acc[i][j]);
    };
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    constexpr int L = LW + LX;
#pragma unroll
    for (int k = 0; k < NST; ++k)
        if (k < nk) issue(k, k);
    if (nk >= NST) conv::wait_vmcnt<(NST - 1) * L>();       // (the scales are older than every stage)
    else conv::wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0, fa[0], fb[0]);
    // One stage: its second half is read under the first half's MFMAs; then every wave has its fragments and its own pieces
    // of the next stage, the barrier makes both common, the stage is refilled and the next one's first half is read under the second
    // half's MFMAs.  REFILL / MORE / WHOLE: a stage to refill, a next stage, a second half exist (compile-time, so
    // that reads and MFMAs share a basic block).
    int cur = 0;
    auto stage_step = [&](auto refill, auto more, auto whole, int kt) {
        constexpr bool REFILL = decltype(refill)::value, MORE = decltype(more)::value, WHOLE = decltype(whole)::value;
        const int next = cur + 1 == NST ? 0 : cur + 1;
        if constexpr (WHOLE) {
            read(cur, 1, fa[1], fb[1]);
            product(fa[0], fb[0]);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
            for (int r = 0; r < FN + FM; ++r) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            }
            if constexpr (MORE) {
                // the next stage has landed once only the stages behind it are in flight
                if constexpr (REFILL) conv::wait_vmcnt<(NST - 2) * L>();
                else conv::wait_vmcnt<0>();
                conv::wait_lgkmcnt<0>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if constexpr (REFILL) issue(cur, kt + NST);
                read(next, 0, fa[0], fb[0]);
            }
            product(fa[1], fb[1]);
            if constexpr (MORE) {
                if constexpr (REFILL) __builtin_amdgcn_sched_group_barrier(0x020, L, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
#pragma unroll
                for (int r = 0; r < FN + FM; ++r) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                }
            }
        } else {
            product(fa[0], fb[0]);
        }
        cur = next;
    };
    constexpr std::true_type Y{};
    constexpr std::false_type N{};
    int kt = 0;
    for (; kt + NST < nk; ++kt) stage_step(Y, Y, Y, kt);
    for (; kt + 1 < nk; ++kt) stage_step(N, Y, Y, kt);
    if (halves & 1) stage_step(N, N, N, kt);
    else stage_step(N, N, Y, kt);

    // lane (q, p): pixel p of every pixel fragment
    using R = Run<OUT, 4>;
    const int q = lane >> 4, p = lane & 15, mw = m0 + wm * WM + p;
    float xs[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) xs[j] = sc[2 * BN + wm * WM + j * 16 + p];
    with_mode(a, [&](auto mode) {
        using M = decltype(mode);
#pragma unroll
        for (int g = 0; g < FN / 4; ++g) {
            const int nl = wn * WN + g * 64 + q * R::PE, n = n0 + nl;
            float ws[16], bias[16];
            load_channels<R>(sc + nl, sc + BN + nl, ws, bias);
            R run[FM];
#pragma unroll
            for (int j = 0; j < FM; ++j) run[j].template load_residual<M>(a, mw + j * 16, n);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                int v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = acc[g * 4 + (i >> 2)][j][i & 3];
                run[j].template store<M>(a, mw + j * 16, n, xs[j], v, ws, bias);
            }
        }
    });
}

// ---- few rows: the K of a small tile is shared by the waves of a workgroup ------------------------------------------------
// 16 FN channels x 16 FM pixels a workgroup; each of its NW waves takes every NW-th 64 bytes of K, its operands straight
// from memory into registers (all loads of a wave in flight together: the call costs one or two memory latencies), and the
// waves' integer sums meet in LDS.  ANY: rows of x at any byte address and pitch.  Pieces may reach behind a row's K (the weights
// are zero there), but not behind the last row's: `left` bytes of x lie from p on.
template <bool ANY>
__device__ __forceinline__ i32x4 load_k16(const char* p, long long left) {
    if constexpr (!ANY) return *reinterpret_cast<const i32x4*>(p);
    i32x4 v{0, 0, 0, 0};
    if (left >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else {
        unsigned u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 15; ++i)
            if (i < left) u[i >> 2] |= (unsigned)(unsigned char)p[i] << (8 * (i & 3));
        v = i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    }
    return v;
}

// The waves' sums meet in LDS; wave j finishes pixel fragment j (xs: the scales of the lane's pixel in every fragment).
template <typename OUT, int FN, int FM, int NW>
__device__ __forceinline__ void finish_few(const Args& a, const i32x4 (&acc)[FN][FM], const float (&xs)[FM], i32x4 (*meet)[FN * FM][64], int n0,
                                           int m0) {
    static_assert(FM <= NW, "a wave for every pixel fragment");
    using R = Run<OUT, FN>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, p = lane & 15;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) meet[wave][j * FN + i][lane] = acc[i][j];
    __syncthreads();
    float x = xs[0];
#pragma unroll
    for (int j = 1; j < FM; ++j) x = wave == j ? xs[j] : x;
    if (wave >= FM) return;
    const int j = wave, m = m0 + j * 16 + p, n = n0 + q * R::PE;
    int v[4 * FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
        i32x4 s = meet[0][j * FN + i][lane];
#pragma unroll
        for (int k = 1; k < NW; ++k) s += meet[k][j * FN + i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i * 4 + e] = s[e];
    }
    float ws[4 * FN], bias[4 * FN];
    load_channels<R>(a.ws + n, a.bias ? a.bias + n : nullptr, ws, bias);
    with_mode(a, [&](auto mode) {
        using M = decltype(mode);
        R run;
        run.template load_residual<M>(a, m, n);
        run.template store<M>(a, m, n, x, v, ws, bias);
    });
}

template <typename OUT, int FN, int FM, int NW, bool ANY>
__global__ __launch_bounds__(64 * NW) void few_rows_kernel(const Args a) {
    constexpr int AHEAD = 4;        // steps of K whose loads are in flight
    __shared__ __attribute__((aligned(16))) i32x4 meet[NW][FN * FM][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, p = lane & 15;
    const unsigned t = xcd_remap(blockIdx.x, gridDim.x);
    const int n0 = (int)(t % (unsigned)a.tiles_n) * (16 * FN), m0 = (int)(t / (unsigned)a.tiles_n) * (16 * FM);
    using R = Run<OUT, FN>;
    const char* pw[FN];
    const char* px[FM];
    long long left[FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) pw[i] = a.w + (long long)(n0 + channel_of<R::PE>(i, p >> 2, p & 3)) * a.kp;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int m = m0 + j * 16 + p < a.M ? m0 + j * 16 + p : a.M - 1;
        px[j] = a.x + m * a.x_ld;
        left[j] = (a.M - 1 - m) * a.x_ld + a.K;
    }
    i32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    const int steps = (a.K + 63) / 64;
    for (int s0 = wave; s0 < steps; s0 += NW * AHEAD) {
        i32x4 fa[AHEAD][FN], fb[AHEAD][FM];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int s = s0 + u * NW, k = s * 64 + q * 16;
            const bool in = s < steps;
#pragma unroll
            for (int i = 0; i < FN; ++i) fa[u][i] = in ? *reinterpret_cast<const i32x4*>(pw[i] + k) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < FM; ++j) fb[u][j] = k < a.K ? load_k16<ANY>(px[j] + k, left[j] - k) : i32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = mma(fa[u][i], fb[u][j], acc[i][j]);
    }
    float xs[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) xs[j] = a.xs[m0 + j * 16 + p < a.M ? m0 + j * 16 + p : a.M - 1];
    finish_few<OUT, FN, FM, NW>(a, acc, xs, meet, n0, m0);
}

// The same from floating rows, 16 x 16 outputs a workgroup: its waves first find the rows' largest values together (their own K in
// registers, so the rows are read once), then each quantises what it holds.  K up to 2048.  One launch instead of two at the
// same time on the GPU (1 x 1024 -> 1024: 5.5 us against 5.8, 100 x 1024 -> 512: 7.4 against 6.9), which is less than the host's
// time for a launch and a workspace.
template <typename OUT, typename T, bool RAG>
__global__ __launch_bounds__(512) void few_float_rows_kernel(const Args a) {
    using namespace rows;
    constexpr int NW = 8, AHEAD = 4, VEC = 16 / (int)sizeof(T), NV = 16 / VEC;
    using P = Piece<T, VEC, true>;
    using R = Run<OUT, 1>;
    __shared__ __attribute__((aligned(16))) i32x4 meet[NW][1][64];
    __shared__ unsigned tops[NW][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, p = lane & 15;
    const unsigned t = xcd_remap(blockIdx.x, gridDim.x);
    const int n0 = (int)(t % (unsigned)a.tiles_n) * 16, m0 = (int)(t / (unsigned)a.tiles_n) * 16;
    const int steps = (a.K + 63) / 64, m = m0 + p < a.M ? m0 + p : a.M - 1;
    // Every load is made, pieces behind K from a page of zeros, so that all are in flight together.  RAG: the piece that holds the row's
    // end also holds what follows it, cleared below; behind the last row it is read value by value.
    typename P::type raw[AHEAD][NV];
    i32x4 fa[AHEAD];
    const T* px = reinterpret_cast<const T*>(a.x) + m * a.x_ld;
    const char* pw = a.w + (long long)(n0 + channel_of<R::PE>(0, p >> 2, p & 3)) * a.kp + q * 16;
    const long long left = (a.M - 1 - m) * a.x_ld + a.K;         // values from the row's first one to the end of all rows
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        const int s = wave + u * NW;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = s * 64 + q * 16 + i * VEC;
            const T* from = k < a.K && (!RAG || k + VEC <= left) ? px + k : reinterpret_cast<const T*>(conv::g_zero_chunk);
            raw[u][i] = *reinterpret_cast<const typename P::loose*>(from);
        }
        fa[u] = *reinterpret_cast<const i32x4*>(s < steps ? pw + s * 64 : reinterpret_cast<const char*>(conv::g_zero_chunk));
    }
    unsigned top = 0;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (wave + u * NW) * 64 + q * 16 + i * VEC;
            if (RAG && k < a.K && k + VEC > left) raw[u][i] = P::load(px + k, (int)(left - k));
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (RAG) raw[u][i][e] = k + e < a.K ? raw[u][i][e] : (T)0.f;
                top = MaxU{}(top, __float_as_uint((float)raw[u][i][e]) & 0x7fffffffu);
            }
        }
    // the four lane groups hold the row's other columns
    const auto r16 = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = MaxU{}(r16[0], r16[1]);
    const auto r32 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = MaxU{}(r32[0], r32[1]);
    if (q == 0) tops[wave][p] = top;
    __syncthreads();
    top = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = MaxU{}(top, tops[w][p]);
    const RowScale rs = row_scale(top);
    i32x4 acc[1][1] = {{i32x4{0, 0, 0, 0}}};
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
        if (wave + u * NW >= steps) break;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = (float)raw[u][i / VEC][i % VEC];
        unsigned m[16], d[4];
        if (quantise_near(v, rs.inv, m) > 0.4999f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) m[i] = quantise_exact(v[i], rs.s, rs.inv);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) m[i] = rs.bad ? 0u : m[i];
        pack_bytes(m, d);
        acc[0][0] = mma(fa[u], i32x4{(int)d[0], (int)d[1], (int)d[2], (int)d[3]}, acc[0][0]);
    }
    const float xs[1] = {rs.given};
    finish_few<OUT, 1, 1, NW>(a, acc, xs, meet, n0, m0);
}

template <typename OUT, int BN, int BM, int WAVES_N, int WAVES_M, int NST = 2>
static int launch_tile(Args a, hipStream_t stream) {
    constexpr int scales = (2 * BN + BM) * 4, stage = (BN + BM) * 128, most = scales + NST * stage;
    const int used = (a.K + 127) / 128, lds = scales + (used < NST ? used : NST) * stage;      // (fewer stages leave room for more workgroups)
    a.tiles_n = (a.N + BN - 1) / BN;
    const long long blocks = (long long)a.tiles_n * ((a.M + BM - 1) / BM);
    YDET_CHECK_ARG(blocks * 64 * WAVES_N * WAVES_M <= UINT32_MAX, "matmul_i8: %d rows x %d channels are too many tiles", a.M, a.N);
    static unsigned char done[kMaxDevices];
    const int rc = raise_dynamic_lds_limit(reinterpret_cast<const void*>(&tile_kernel<OUT, BN, BM, WAVES_N, WAVES_M, NST>), most, done, "matmul_i8");
    if (rc != YDET_OK) return rc;
    hipLaunchKernelGGL((tile_kernel<OUT, BN, BM, WAVES_N, WAVES_M, NST>), dim3((unsigned)blocks), dim3(64 * WAVES_N * WAVES_M), lds, stream, a);
    YDET_CHECK_LAUNCH("matmul_i8");
    return YDET_OK;
}

template <typename OUT, int FN, int FM, int NW, bool ANY>
static int launch_few(Args a, hipStream_t stream) {
    a.tiles_n = (a.N + 16 * FN - 1) / (16 * FN);
    const long long blocks = (long long)a.tiles_n * ((a.M + 16 * FM - 1) / (16 * FM));
    YDET_CHECK_ARG(blocks * 64 * NW <= UINT32_MAX, "matmul_i8: %d rows x %d channels are too many tiles", a.M, a.N);
    hipLaunchKernelGGL((few_rows_kernel<OUT, FN, FM, NW, ANY>), dim3((unsigned)blocks), dim3(64 * NW), 0, stream, a);
    YDET_CHECK_LAUNCH("matmul_i8 (few rows)");
    return YDET_OK;
}

template <typename OUT, typename T, bool RAG>
static int launch_few_float(Args a, hipStream_t stream) {
    a.tiles_n = (a.N + 15) / 16;
    const long long blocks = (long long)a.tiles_n * ((a.M + 15) / 16);      // (one a CU at most)
    hipLaunchKernelGGL((few_float_rows_kernel<OUT, T, RAG>), dim3((unsigned)blocks), dim3(512), 0, stream, a);
    YDET_CHECK_LAUNCH("linear_i8 (few rows)");
    return YDET_OK;
}

// Rows at any address and pitch into rows of K rounded up to 16, for the tile kernels (bytes behind K: anything).
__global__ __launch_bounds__(256) void align_rows_kernel(const char* x, long long ld, int M, int K, char* to) {
    const int pieces = (K + 15) / 16;
    const long long all = (long long)M * pieces;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long m = i / pieces;
        const int k = (int)(i - m * pieces) * 16;
        *reinterpret_cast<i32x4*>(to + i * 16) = load_k16<true>(x + m * ld + k, (M - 1 - m) * ld + K - k);
    }
}

// Which kernel takes a product, by rows, channels and K alone; every one gives the same bits.  Measured on 256 CUs, us, the kernel
// alone with three inputs in turn:
//   16 x 16 outputs a workgroup, straight from memory, up to two workgroups a CU (1 x 1024 -> 1024: 3.2, in 64 x 128 tiles 5.5; 40 x
//     4096 -> 512: 6.3 against 12.8; 100 x 1024 -> 512: 3.8 against 5.9);
//   32 x 32, straight from memory, up to one a CU (400 x 1024 -> 512: 5.2, in 64 x 128 tiles 6.2; 200 x 2048 -> 1024: 7.0 against 8.3,
//     but 1600 x 512 -> 512: 7.3 against 5.1);
//   256 x 192 tiles for K >= 2048 where they leave no quarter of the CUs idle (23104 x 4096 -> 512: 55, in 128 x 128 tiles 80; but
//     25600 x 1024 -> 512: 31 against 26);
//   128 x 128 for K >= 1024 with at least a tile a CU (6400 x 1024 -> 1024: 13.5, in 64 x 128 tiles 16.2);
//   64 x 128 otherwise (409600 x 64 -> 64: 16, in 128 x 128 tiles 25; 409600 x 128 -> 128 with residual: 49 against 53), with a
//     third stage where there are fewer than two workgroups a CU (2888 x 4096 -> 512: 14.7, with two stages 18.7).
// The tile kernels want rows at 4-byte addresses and pitches: others are first copied into the workspace (2888 x 1000 -> 255: 3.4 us
// and a launch more on top of 6.7).
static long long tiles(const Args& a, int bn, int bm) { return (long long)((a.N + bn - 1) / bn) * ((a.M + bm - 1) / bm); }
static int direct_size(const Args& a) {
    const int cus = current_device_info().cus;
    return tiles(a, 16, 16) <= 2 * cus ? 16 : tiles(a, 32, 32) <= cus ? 32 : 0;
}

// Whether floating rows are quantised by the product's own kernel: K fits its registers and there is at most a workgroup a CU (400 x
// 100 -> 255, 400 workgroups, took 7.2 us, the two launches 5.6; a form for 32 x 32 outputs 12.3 us for 400 x 1024 -> 512, the two
// launches 8.1: every workgroup quantises).
static bool fuses(const Args& a) { return a.K <= 2048 && tiles(a, 16, 16) <= current_device_info().cus; }
template <typename OUT, typename T>
static int launch_fused(const Args& a, hipStream_t stream) {
    return a.K % (16 / (int)sizeof(T)) ? launch_few_float<OUT, T, true>(a, stream) : launch_few_float<OUT, T, false>(a, stream);
}

template <typename OUT>
static int launch(const Args& a, bool wide_x, hipStream_t stream) {
    const int cus = current_device_info().cus, direct = direct_size(a);
    if (direct == 16) return wide_x ? launch_few<OUT, 1, 1, 8, false>(a, stream) : launch_few<OUT, 1, 1, 8, true>(a, stream);
    if (direct == 32) return wide_x ? launch_few<OUT, 2, 2, 4, false>(a, stream) : launch_few<OUT, 2, 2, 4, true>(a, stream);
    if (a.K >= 2048 && a.N > 128 && tiles(a, 256, 192) * 4 >= cus * 3) return launch_tile<OUT, 256, 192, 2, 4>(a, stream);
    if (a.K >= 1024 && a.N > 64 && tiles(a, 128, 128) >= cus) return launch_tile<OUT, 128, 128, 2, 4>(a, stream);
    if (tiles(a, 64, 128) < 2 * cus) return launch_tile<OUT, 64, 128, 1, 4, 3>(a, stream);
    return launch_tile<OUT, 64, 128, 1, 4, 2>(a, stream);
}

}  // namespace i8
}  // namespace ydet

using namespace ydet;

// How the rows of x lie: at any byte, in whole words (for LDS-DMA), or in 16-byte pieces (for plain loads) that may reach
// behind K, so that the pitch has to hold them.
enum class Rows { bytes, words, pieces };

// Checks a descriptor and fills the launch arguments.
static int fill_args(const ydet_matmul_i8_desc* d, i8::Args& a, Rows& lie) {
    YDET_CHECK_ARG(d, "matmul_i8: null descriptor");
    YDET_CHECK_ARG(d->rows >= 0 && d->rows <= INT32_MAX - 512 && d->K > 0 && d->K <= 131071 && d->N > 0 && d->N <= (1 << 24),
                   "matmul_i8: rows=%lld K=%d N=%d (K up to 131071: the sums are 32-bit integers)", (long long)d->rows, d->K, d->N);
    YDET_CHECK_ARG(d->kp % 64 == 0 && d->kp >= d->K && d->n_pad % 128 == 0 && d->n_pad >= d->N,
                   "matmul_i8: weights padded to %d x %d (want a multiple of 128 >= %d, a multiple of 64 >= %d)", d->n_pad, d->kp, d->N, d->K);
    YDET_CHECK_ARG(d->x_coff >= 0 && d->y_coff >= 0 && (long long)d->x_coff + d->K <= d->x_ld && (long long)d->y_coff + d->N <= d->y_ld,
                   "matmul_i8: a slice lies outside its rows");
    YDET_CHECK_ARG(d->x_ld <= (1 << 23), "matmul_i8: x_ld=%d (up to %d)", d->x_ld, 1 << 23);
    YDET_CHECK_ARG(d->out_dtype == YDET_F32 || d->out_dtype == YDET_BF16, "matmul_i8: out_dtype %d", d->out_dtype);
    YDET_CHECK_ARG(d->act >= YDET_ACT_NONE && d->act <= YDET_ACT_SILU && d->res_mode >= YDET_RES_NONE && d->res_mode <= YDET_RES_BEFORE_ACT,
                   "matmul_i8: act %d res_mode %d", d->act, d->res_mode);
    YDET_CHECK_ARG(d->res_mode == YDET_RES_NONE || (d->res_coff >= 0 && (long long)d->res_coff + d->N <= d->res_ld),
                   "matmul_i8: the residual's slice lies outside its rows");
    YDET_CHECK_ARG(d->rows == 0 || (d->x && d->x_scale && d->w && d->w_scale && d->y && (d->res_mode == YDET_RES_NONE || d->res)), "matmul_i8: null pointer");
    YDET_CHECK_ARG(((uintptr_t)d->w | (uintptr_t)d->w_scale | (uintptr_t)d->bias) % 16 == 0, "matmul_i8: weights, scales and bias need 16-byte alignment");
    const size_t es = dtype_size(d->out_dtype);
    a = i8::Args{};
    a.x = reinterpret_cast<const char*>(d->x) + d->x_coff;
    a.xs = d->x_scale, a.w = reinterpret_cast<const char*>(d->w), a.ws = d->w_scale, a.bias = d->bias;
    a.y = static_cast<char*>(d->y) + d->y_coff * es;
    a.res_mode = d->res_mode;
    if (a.res_mode != YDET_RES_NONE) a.res = static_cast<const char*>(d->res) + d->res_coff * es;
    YDET_CHECK_ARG(((uintptr_t)a.y | (uintptr_t)a.res) % es == 0 && (uintptr_t)a.xs % 4 == 0, "matmul_i8: misaligned tensor");
    a.M = (int)d->rows, a.K = d->K, a.N = d->N, a.kp = d->kp, a.n_pad = d->n_pad;
    a.x_ld = d->x_ld, a.y_ld = d->y_ld, a.res_ld = d->res_ld, a.act = d->act, a.slope = d->act == YDET_ACT_LEAKY ? d->slope : 1.f;
    const uintptr_t at = (uintptr_t)a.x | (uintptr_t)(unsigned)d->x_ld;
    lie = at % 16 == 0 && d->x_coff + (d->K + 15) / 16 * 16 <= d->x_ld ? Rows::pieces : at % 4 == 0 ? Rows::words : Rows::bytes;
    return YDET_OK;
}

static size_t aligned_bytes(const i8::Args& a) { return (size_t)a.M * ((a.K + 15) / 16 * 16); }

int ydet_launch_matmul_i8(const ydet_matmul_i8_desc* d, void* ws, size_t ws_bytes, hipStream_t stream) {
    i8::Args a;
    Rows lie;
    const int rc = fill_args(d, a, lie);
    if (rc != YDET_OK || a.M == 0) return rc;
    if (lie == Rows::bytes && !i8::direct_size(a)) {
        if (ws_bytes < aligned_bytes(a))
            return fail(YDET_ERR_WORKSPACE, "matmul_i8: workspace %zu < %zu bytes", ws_bytes, aligned_bytes(a));
        YDET_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0, "matmul_i8: rows of %d at this address and pitch need a 16-byte aligned workspace", a.K);
        const long long blocks = ((long long)(aligned_bytes(a) / 16) + 255) / 256;
        hipLaunchKernelGGL(i8::align_rows_kernel, dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(256), 0, stream, a.x, a.x_ld, a.M,
                           a.K, static_cast<char*>(ws));
        YDET_CHECK_LAUNCH("matmul_i8 (rows)");
        a.x = static_cast<const char*>(ws), a.x_ld = (a.K + 15) / 16 * 16;
    }
    const bool wide_x = lie == Rows::pieces;
    return d->out_dtype == YDET_BF16 ? i8::launch<__bf16>(a, wide_x, stream) : i8::launch<float>(a, wide_x, stream);
}

extern "C" size_t ydet_matmul_i8_workspace_bytes(const ydet_matmul_i8_desc* d) {
    clear_error();
    i8::Args a;
    Rows lie;
    if (fill_args(d, a, lie) != YDET_OK || lie != Rows::bytes || a.M == 0 || i8::direct_size(a)) return 0;
    return aligned_bytes(a);
}

// Checks the pair and fills the product's arguments as for rows in a workspace at `at` (any aligned address, to ask).
static int fill_linear(const ydet_quantize_desc* in, const ydet_matmul_i8_desc* product, void* at, ydet_quantize_desc& q, ydet_matmul_i8_desc& p,
                       i8::Args& a) {
    YDET_CHECK_ARG(in && product, "linear_i8: null descriptor");
    YDET_CHECK_ARG(in->rows == product->rows && in->C == product->K, "linear_i8: %lld x %d rows for a product of %lld x %d", (long long)in->rows,
                   in->C, (long long)product->rows, product->K);
    YDET_CHECK_ARG(in->rows >= 0 && in->rows <= INT32_MAX && in->C > 0 && in->C <= rows::kMaxC, "linear_i8: rows=%lld K=%d (K 1..%d)",
                   (long long)in->rows, in->C, rows::kMaxC);
    q = *in;
    p = *product;
    q.q_ld = p.x_ld = (in->C + 15) / 16 * 16, p.x_coff = 0;
    p.x = q.q = static_cast<int8_t*>(at);
    p.x_scale = q.scale = reinterpret_cast<float*>(q.q + in->rows * q.q_ld);
    Rows lie;
    return fill_args(&p, a, lie);
}

// Whether the output touches bytes of the floating rows.  Slices of one pitch that take different columns of it do not.
static bool writes_input(const ydet_quantize_desc& q, const ydet_matmul_i8_desc& p) {
    const long long xe = (long long)dtype_size(q.dtype), ye = (long long)dtype_size(p.out_dtype);
    const long long x = (long long)(uintptr_t)q.x + q.x_coff * xe, y = (long long)(uintptr_t)p.y + p.y_coff * ye;
    const long long x_row = q.C * xe, y_row = p.N * ye, x_ld = q.x_ld * xe, y_ld = p.y_ld * ye;
    if (y + (p.rows - 1) * y_ld + y_row <= x || x + (q.rows - 1) * x_ld + x_row <= y) return false;
    if (x_ld != y_ld) return true;
    const long long at = ((y - x) % x_ld + x_ld) % x_ld;       // where in a row of x one of y begins
    return at < x_row || at + y_row > x_ld;
}

static bool fused(const ydet_quantize_desc& q, const i8::Args& a) { return !q.normalize && i8::fuses(a); }

static size_t linear_bytes(const ydet_quantize_desc& q) { return (size_t)q.rows * q.q_ld + (size_t)(q.rows + 3) / 4 * 16; }

extern "C" size_t ydet_linear_i8_workspace_bytes(const ydet_quantize_desc* in, const ydet_matmul_i8_desc* product) {
    clear_error();
    ydet_quantize_desc q;
    ydet_matmul_i8_desc p;
    i8::Args a;
    if (fill_linear(in, product, reinterpret_cast<void*>(256), q, p, a) != YDET_OK || q.rows == 0 || fused(q, a)) return 0;
    return linear_bytes(q);
}

int ydet_launch_linear_i8(const ydet_quantize_desc* in, const ydet_matmul_i8_desc* product, void* ws, size_t ws_bytes, hipStream_t stream) {
    ydet_quantize_desc q;
    ydet_matmul_i8_desc p;
    i8::Args a;
    int rc = fill_linear(in, product, ws ? ws : reinterpret_cast<void*>(256), q, p, a);
    if (rc != YDET_OK || q.rows == 0) return rc;
    // (in one launch workgroups read whole rows while others already store their channels: not where those are the same bytes.  In
    // two, every row is in 8 bits before the first store.)
    if (fused(q, a) && !writes_input(q, p)) {
        rc = ydet_check_quantize_rows(&q);
        if (rc != YDET_OK) return rc;
        a.x = static_cast<const char*>(q.x) + q.x_coff * dtype_size(q.dtype), a.x_ld = q.x_ld, a.xs = nullptr;
        if (q.dtype == YDET_BF16)
            return p.out_dtype == YDET_BF16 ? i8::launch_fused<__bf16, __bf16>(a, stream) : i8::launch_fused<float, __bf16>(a, stream);
        return p.out_dtype == YDET_BF16 ? i8::launch_fused<__bf16, float>(a, stream) : i8::launch_fused<float, float>(a, stream);
    }
    YDET_CHECK_ARG(ws && (uintptr_t)ws % 16 == 0, "linear_i8: needs a 16-byte aligned workspace");
    if (ws_bytes < linear_bytes(q)) return fail(YDET_ERR_WORKSPACE, "linear_i8: workspace %zu < %zu bytes", ws_bytes, linear_bytes(q));
    rc = ydet_launch_quantize_rows(&q, stream);
    return rc != YDET_OK ? rc : ydet_launch_matmul_i8(&p, nullptr, 0, stream);
}

extern "C" int ydet_linear_i8(const ydet_quantize_desc* in, const ydet_matmul_i8_desc* product, void* workspace, size_t workspace_bytes,
                              void* stream) {
    clear_error();
    return ydet_launch_linear_i8(in, product, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int ydet_matmul_i8(const ydet_matmul_i8_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    return ydet_launch_matmul_i8(d, workspace, workspace_bytes, as_stream(stream));
}
