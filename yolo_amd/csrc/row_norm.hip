// Layer normalisation over channels and symmetric 8-bit quantisation of rows, each alone or the second behind the first, on
// NHWC slices: a row is the C channels of one pixel.
//
//   norm      mu = sum_c x_c / C,  var = sum_c (x_c - mu)^2 / C,  r = 1 / sqrt(var + eps),  y_c = (x_c - mu) * r * w_c + b_c
//   quantise  s = max_c |y_c| / 127 (rounded once),  q_c = the integer nearest y_c / s, ties to even
//
// One pass over memory: a row is read once into the registers of the lanes that share it (rows_common.h), mean, variance
// (from the differences to the mean, not as a difference of squares) and maximum are taken there, and the result is
// written.  Sums, statistics and scales are in 32 bits.  The bytes of a bf16 value (2 in, 1 or 2 out) take as long as about
// fifteen operations, so what is done once a row counts as well: rstd is the hardware's reciprocal square root, 1 / s its
// reciprocal (one unit in the last place each), mean and scale are divided by a product and a remainder.
#include "rows_common.h"

namespace ydet {
namespace rows {

struct RowArgs {
    const char* x;      // first value of the slice
    char* y;            // normalised rows, or 8-bit rows
    float* scale;
    const char* gamma;
    const char* beta;
    float* mean;
    float* rstd;
    long long rows;
    int C, cw;          // values of a row; values written of a row (8-bit rows: zeros behind C)
    int x_ld, y_ld;
    int param_dtype;
    float eps, inv_c;
};

enum { kNorm = 1, kQuant = 2 };

template <int MODE, typename T, bool RAG, int LPR, int CH, int RPT>
__global__ __launch_bounds__(kThreads) void row_norm_kernel(const RowArgs a) {
    constexpr int VEC = 16 / (int)sizeof(T);
    using P = Piece<T, VEC, RAG>;
    constexpr int G = kThreads / LPR;       // rows of a workgroup at a time
    constexpr bool NORM = (MODE & kNorm) != 0, QUANT = (MODE & kQuant) != 0;
    __shared__ unsigned red[2][4];
    int slot = 0;
    const int tid = threadIdx.x, g = tid / LPR, l = tid % LPR;
    const float fc = (float)a.C;
    float w[NORM ? CH * VEC : 1], b[NORM ? CH * VEC : 1];
    if constexpr (NORM) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + l) * VEC;
            load_params<VEC, RAG>(a.gamma, a.param_dtype, col, a.C - col, 1.f, w + c * VEC);
            load_params<VEC, RAG>(a.beta, a.param_dtype, col, a.C - col, 0.f, b + c * VEC);
        }
    }
    for (long long row0 = (long long)blockIdx.x * (G * RPT); row0 < a.rows; row0 += (long long)gridDim.x * (G * RPT)) {
        typename P::type in[RPT][CH];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            const long long row = row0 + r * G + g;
            const T* xr = reinterpret_cast<const T*>(a.x) + row * a.x_ld;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LPR + l) * VEC;
                in[r][c] = typename P::type{};
                if (row < a.rows && col < a.C) in[r][c] = P::load(xr + col, a.C - col);
            }
        }
        // (step by step over all RPT rows, whose chains of operations fill each other's gaps)
        float v[RPT][CH * VEC];
#pragma unroll
        for (int r = 0; r < RPT; ++r)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[r][c * VEC + i] = (float)in[r][c][i];
        if constexpr (NORM) {
            float mean[RPT], rstd[RPT];
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                mean[r] = 0.f;
#pragma unroll
                for (int i = 0; i < CH * VEC; ++i) mean[r] += v[r][i];
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) mean[r] = quotient(group_sum<LPR>(mean[r], red, slot), fc, a.inv_c);
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                rstd[r] = 0.f;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int left = a.C - (c * LPR + l) * VEC;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float d = P::has(i, left) ? v[r][c * VEC + i] - mean[r] : 0.f;
                        v[r][c * VEC + i] = d;
                        rstd[r] = fmaf(d, d, rstd[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) rstd[r] = __builtin_amdgcn_rsqf(fmaf(group_sum<LPR>(rstd[r], red, slot), a.inv_c, a.eps));
            if (a.mean && l == 0) {
#pragma unroll
                for (int r = 0; r < RPT; ++r) {
                    const long long row = row0 + r * G + g;
                    if (row < a.rows) a.mean[row] = mean[r], a.rstd[row] = rstd[r];
                }
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r)
#pragma unroll
                for (int i = 0; i < CH * VEC; ++i)
                    v[r][i] = P::has(i % VEC, a.C - (i / VEC * LPR + l) * VEC) ? fmaf(v[r][i] * rstd[r], w[i], b[i]) : 0.f;
        }
        if constexpr (!QUANT) {
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                const long long row = row0 + r * G + g;
                if (row >= a.rows) continue;
                T* yr = reinterpret_cast<T*>(a.y) + row * a.y_ld;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LPR + l) * VEC;
                    if (col < a.C) {
                        typename P::type o;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) o[i] = (T)v[r][c * VEC + i];
                        P::store(yr + col, o, a.C - col);
                    }
                }
            }
        } else {
            // (lanes and pieces behind the row's end hold zeros)
            unsigned top[RPT], m[RPT][CH * VEC];
            RowScale rs[RPT];
            float near = 0.f;
            bool bad = false;
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                top[r] = 0;
#pragma unroll
                for (int i = 0; i < CH * VEC; ++i) top[r] = MaxU{}(top[r], __float_as_uint(v[r][i]) & 0x7fffffffu);
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) rs[r] = row_scale(group_reduce<LPR>(top[r], MaxU{}, red, slot));
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                near = fmaxf(near, quantise_near(v[r], rs[r].inv, m[r]));
                bad = bad || rs[r].bad;
            }
            if (near > 0.4999f) {
#pragma unroll
                for (int r = 0; r < RPT; ++r)
#pragma unroll
                    for (int i = 0; i < CH * VEC; ++i) m[r][i] = quantise_exact(v[r][i], rs[r].s, rs[r].inv);
            }
            if (bad) {
#pragma unroll
                for (int r = 0; r < RPT; ++r)
#pragma unroll
                    for (int i = 0; i < CH * VEC; ++i) m[r][i] = rs[r].bad ? 0u : m[r][i];
            }
#pragma unroll
            for (int r = 0; r < RPT; ++r) {
                const long long row = row0 + r * G + g;
                if (row >= a.rows) continue;
                if (l == 0) a.scale[row] = rs[r].given;
                unsigned d[CH * VEC / 4];
                pack_bytes(m[r], d);
                char* yr = a.y + row * a.y_ld;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int col = (c * LPR + l) * VEC;
                    if (col < a.cw) {
                        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(yr + col) = make_uint2(d[2 * c], d[2 * c + 1]);
                        else *reinterpret_cast<unsigned*>(yr + col) = d[c];
                    }
                }
            }
        }
    }
}

// Workgroups: each walks over rows, weight and bias in its registers.  No more than stay resident where a workgroup reads weight and
// bias: four a CU for rows of more than 4096 values, 32 a lane (5776 x 8192 norm + quantisation in fp32 66 us, with eight 73, with 16
// 85; 23104 x 4224 in bf16 178 against 181, norm alone 77 against 79; 8192 in bf16 level), eight for shorter ones (23104 x 2048 norm
// + quantisation in bf16 39 us, with four 49; 51200 x 512 in fp32 level).  Twice as many where it reads none (25600 x 512
// quantisation 10.3 us, with eight 10.9; 23104 x 4224 103 against 106) or takes four rows at a time (409600 x 128 norm 38.6 us, with
// eight 41.2).
template <int MODE, typename T, bool RAG, int LPR, int CH, int RPT>
static int launch_rows(const RowArgs& a, hipStream_t stream) {
    constexpr int per = kThreads / LPR * RPT, per_cu = !(MODE & kNorm) || RPT > 1 ? 16 : CH * 16 / (int)sizeof(T) > 16 ? 4 : 8;
    const long long need = (a.rows + per - 1) / per, most = (long long)current_device_info().cus * per_cu;
    hipLaunchKernelGGL((row_norm_kernel<MODE, T, RAG, LPR, CH, RPT>), dim3((unsigned)(need < most ? need : most)), dim3(kThreads), 0, stream, a);
    YDET_CHECK_LAUNCH("row norm / quantise");
    return YDET_OK;
}

// Rows a lane group takes at once: four (their loads in flight together) where that still leaves eight workgroups a CU, else one;
// one where the rows are quantised (four cost 148 registers: 102400 x 256 norm + quantisation 28.2 us, with one 20.4).
template <int MODE, typename T, bool RAG, int LPR, int CH>
static int launch_depth(const RowArgs& a, hipStream_t stream) {
    if constexpr (CH == 1 && LPR <= 64 && !(MODE & kQuant)) {
        if (a.rows >= (long long)current_device_info().cus * 8 * 4 * (kThreads / LPR))
            return launch_rows<MODE, T, RAG, LPR, CH, 4>(a, stream);
    }
    return launch_rows<MODE, T, RAG, LPR, CH, 1>(a, stream);
}

// Longer rows take a whole workgroup: fewer values, weights and biases a lane leave room for more waves (norm + quantisation of
// 23104 x 2048 in bf16 41 us, inside a wave 54; of 400 x 1200 4.7 and 7.3; norm of 5000 x 1500 in fp32 12.2 and 14.5).
constexpr int kWaveCols = 1024;
template <int MODE, typename T, bool RAG>
static int launch_shape(const RowArgs& a, hipStream_t stream) {
    const Shape s = shape_of(a.cw, 16 / (int)sizeof(T), kWaveCols);
#define YDET_ROWS(L, K) \
    if (s.lpr == L && s.ch == K) return launch_depth<MODE, T, RAG, L, K>(a, stream);
    YDET_ROWS(4, 1) YDET_ROWS(8, 1) YDET_ROWS(16, 1) YDET_ROWS(32, 1) YDET_ROWS(64, 1) YDET_ROWS(64, 2) YDET_ROWS(256, 2) YDET_ROWS(256, 4)
    if constexpr (sizeof(T) == 4) {
        YDET_ROWS(64, 4) YDET_ROWS(256, 8)
    } else {
        YDET_ROWS(256, 1)
    }
#undef YDET_ROWS
    return fail(YDET_ERR_ARG, "row norm: no kernel for %d channels", a.C);
}

template <int MODE>
static int launch_mode(const RowArgs& a, int dtype, hipStream_t stream) {
    if (dtype == YDET_BF16) return a.C % 8 ? launch_shape<MODE, __bf16, true>(a, stream) : launch_shape<MODE, __bf16, false>(a, stream);
    return a.C % 4 ? launch_shape<MODE, float, true>(a, stream) : launch_shape<MODE, float, false>(a, stream);
}

}  // namespace rows
}  // namespace ydet

using namespace ydet;
using namespace ydet::rows;

int ydet_launch_layer_norm(const ydet_layer_norm_desc* d, hipStream_t stream) {
    YDET_CHECK_ARG(d, "layer_norm: null descriptor");
    YDET_CHECK_ARG(d->rows >= 0 && d->rows <= INT32_MAX && d->C > 0 && d->C <= kMaxC, "layer_norm: rows=%lld C=%d (C 1..%d)",
                   (long long)d->rows, d->C, kMaxC);
    YDET_CHECK_ARG(dtype_ok(d->dtype) && dtype_ok(d->param_dtype), "layer_norm: dtype %d / %d", d->dtype, d->param_dtype);
    YDET_CHECK_ARG(d->x_coff >= 0 && d->y_coff >= 0 && (long long)d->x_coff + d->C <= d->x_ld && (long long)d->y_coff + d->C <= d->y_ld,
                   "layer_norm: slice of %d channels at %d / %d outside rows of %d / %d", d->C, d->x_coff, d->y_coff, d->x_ld, d->y_ld);
    YDET_CHECK_ARG(d->eps >= 0.f, "layer_norm: eps=%g", (double)d->eps);
    YDET_CHECK_ARG(!d->mean == !d->rstd, "layer_norm: mean and rstd come together");
    if (d->rows == 0) return YDET_OK;
    YDET_CHECK_ARG(d->x && d->y, "layer_norm: null pointer");
    const size_t es = dtype_size(d->dtype);
    RowArgs a{};
    a.x = static_cast<const char*>(d->x) + d->x_coff * es;
    a.y = static_cast<char*>(d->y) + d->y_coff * es;
    YDET_CHECK_ARG(((uintptr_t)a.x | (uintptr_t)a.y) % es == 0, "layer_norm: misaligned tensor");
    a.gamma = static_cast<const char*>(d->gamma), a.beta = static_cast<const char*>(d->beta);
    a.mean = d->mean, a.rstd = d->rstd, a.rows = d->rows, a.C = a.cw = d->C;
    a.x_ld = d->x_ld, a.y_ld = d->y_ld, a.param_dtype = d->param_dtype, a.eps = d->eps, a.inv_c = 1.f / (float)d->C;
    return launch_mode<kNorm>(a, d->dtype, stream);
}

// What ydet_quantize_rows_i8 asks of its arguments.
int ydet_check_quantize_rows(const ydet_quantize_desc* d) {
    YDET_CHECK_ARG(d, "quantize_rows: null descriptor");
    YDET_CHECK_ARG(d->rows >= 0 && d->rows <= INT32_MAX && d->C > 0 && d->C <= kMaxC, "quantize_rows: rows=%lld C=%d (C 1..%d)",
                   (long long)d->rows, d->C, kMaxC);
    YDET_CHECK_ARG(dtype_ok(d->dtype) && dtype_ok(d->param_dtype), "quantize_rows: dtype %d / %d", d->dtype, d->param_dtype);
    const int cw = (d->C + 15) / 16 * 16;
    YDET_CHECK_ARG(d->x_coff >= 0 && (long long)d->x_coff + d->C <= d->x_ld, "quantize_rows: slice of %d channels at %d outside rows of %d",
                   d->C, d->x_coff, d->x_ld);
    YDET_CHECK_ARG(d->q_ld >= cw && d->q_ld % 16 == 0, "quantize_rows: rows of %d channels need q_ld >= %d, a multiple of 16 (got %d)", d->C,
                   cw, d->q_ld);
    YDET_CHECK_ARG(!d->normalize || d->eps >= 0.f, "quantize_rows: eps=%g", (double)d->eps);
    YDET_CHECK_ARG(d->rows == 0 || (d->x && d->q && d->scale), "quantize_rows: null pointer");
    const size_t es = dtype_size(d->dtype);
    YDET_CHECK_ARG((uintptr_t)d->x % es == 0 && (uintptr_t)d->q % 16 == 0, "quantize_rows: misaligned tensor");
    return YDET_OK;
}

int ydet_launch_quantize_rows(const ydet_quantize_desc* d, hipStream_t stream) {
    const int rc = ydet_check_quantize_rows(d);
    if (rc != YDET_OK || d->rows == 0) return rc;
    RowArgs a{};
    a.x = static_cast<const char*>(d->x) + d->x_coff * dtype_size(d->dtype);
    a.y = reinterpret_cast<char*>(d->q);
    const int cw = (d->C + 15) / 16 * 16;
    a.scale = d->scale, a.rows = d->rows, a.C = d->C, a.cw = cw, a.x_ld = d->x_ld, a.y_ld = d->q_ld;
    a.gamma = static_cast<const char*>(d->gamma), a.beta = static_cast<const char*>(d->beta);
    a.param_dtype = d->param_dtype, a.eps = d->eps, a.inv_c = 1.f / (float)d->C;
    return d->normalize ? launch_mode<kNorm | kQuant>(a, d->dtype, stream) : launch_mode<kQuant>(a, d->dtype, stream);
}

extern "C" int ydet_layer_norm(const ydet_layer_norm_desc* d, void* stream) {
    clear_error();
    return ydet_launch_layer_norm(d, as_stream(stream));
}

extern "C" int ydet_quantize_rows_i8(const ydet_quantize_desc* d, void* stream) {
    clear_error();
    return ydet_launch_quantize_rows(d, as_stream(stream));
}
