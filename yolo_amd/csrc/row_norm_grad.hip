// Gradient of the layer normalisation over channels (row_norm.hip) on NHWC slices.  With xh = (x - mu) r and g = dy * w,
//
//   dx_c = r * (g_c - sum_j g_j / C - xh_c * sum_j g_j xh_j / C)      dw_c = sum_rows dy_c xh_c      db_c = sum_rows dy_c
//
// One pass over dy and x serves all three: a row sits in the registers of the lanes that share it (rows_common.h), which take
// its two sums and write dx, while every lane keeps running sums of dw and db for the columns it owns, over all rows it
// meets.  A workgroup's lane groups then meet in LDS and leave one partial sum a column in the workspace, and a second kernel
// adds the workgroups' partial sums in a fixed order: no atomics, the same bits every time.  All sums are in 32 bits.  A lane adds
// at most kChain rows one after the other; more rows than that for every lane group (1 M of more than 2048 bf16 channels, 67 M of
// up to 16) take another launch, which adds to the partial sums.  Behind the lanes come at most 64 groups, one term a launch, and the
// tree over the workgroups.  Bound by HBM: 6 bytes a bf16 value.
#include "rows_common.h"

namespace ydet {
namespace rows {

struct GradArgs {
    const char* dy;
    const char* x;
    char* dx;               // or null
    const char* gamma;
    const float* mean;
    const float* rstd;
    float* part;            // [workgroups][2][C] partial sums of dw and db, or null
    long long rows;
    int C, dy_ld, x_ld, dx_ld, param_dtype;
    int more;               // the partial sums hold those of the rows before these
};
constexpr int kChain = 1024;

template <typename T, bool RAG, int LPR, int CH, int RPT>
__global__ __launch_bounds__(kThreads) void norm_grad_kernel(const GradArgs a) {
    constexpr int VEC = 16 / (int)sizeof(T);
    using P = Piece<T, VEC, RAG>;
    constexpr int G = kThreads / LPR, V = CH * VEC;
    __shared__ unsigned red[2][4];
    __shared__ float meet[G > 1 ? kThreads * V : 1];
    int slot = 0;
    const int tid = threadIdx.x, g = tid / LPR, l = tid % LPR;
    const float ic = 1.f / (float)a.C;
    float w[V], dw[V], db[V];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * LPR + l) * VEC;
        load_params<VEC, RAG>(a.gamma, a.param_dtype, col, a.C - col, 1.f, w + c * VEC);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;

    for (long long row0 = (long long)blockIdx.x * (G * RPT); row0 < a.rows; row0 += (long long)gridDim.x * (G * RPT)) {
        typename P::type in[RPT][CH], gr[RPT][CH];
        float mean[RPT], rstd[RPT];
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            const long long row = row0 + r * G + g;
            const bool live = row < a.rows;
            const T* xr = reinterpret_cast<const T*>(a.x) + row * a.x_ld;
            const T* gy = reinterpret_cast<const T*>(a.dy) + row * a.dy_ld;
            mean[r] = live ? a.mean[row] : 0.f;
            rstd[r] = live ? a.rstd[row] : 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int col = (c * LPR + l) * VEC;
                in[r][c] = gr[r][c] = typename P::type{};
                if (live && col < a.C) {
                    in[r][c] = P::load(xr + col, a.C - col);
                    gr[r][c] = P::load(gy + col, a.C - col);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < RPT; ++r) {
            const long long row = row0 + r * G + g;
            float xh[V], t[V], s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int left = a.C - (c * LPR + l) * VEC;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const int k = c * VEC + i;
                    const float dy = (float)gr[r][c][i];
                    xh[k] = P::has(i, left) ? ((float)in[r][c][i] - mean[r]) * rstd[r] : 0.f;
                    t[k] = dy * w[k];
                    s1 += t[k];
                    s2 = fmaf(t[k], xh[k], s2);
                    dw[k] = fmaf(dy, xh[k], dw[k]);
                    db[k] += dy;
                }
            }
            if (a.dx) {
                const float m1 = group_sum<LPR>(s1, red, slot) * ic, m2 = group_sum<LPR>(s2, red, slot) * ic;
                if (row < a.rows) {
                    T* out = reinterpret_cast<T*>(a.dx) + row * a.dx_ld;
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        const int col = (c * LPR + l) * VEC;
                        if (col < a.C) {
                            typename P::type o;
#pragma unroll
                            for (int i = 0; i < VEC; ++i) {
                                const int k = c * VEC + i;
                                o[i] = (T)(rstd[r] * (t[k] - m1 - xh[k] * m2));
                            }
                            P::store(out + col, o, a.C - col);
                        }
                    }
                }
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + (long long)blockIdx.x * 2 * a.C;
    if constexpr (G == 1) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * LPR + l) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (col + i < a.C) {
                    float& pw = part[col + i];
                    float& pb = part[a.C + col + i];
                    pw = a.more ? pw + dw[c * VEC + i] : dw[c * VEC + i];
                    pb = a.more ? pb + db[c * VEC + i] : db[c * VEC + i];
                }
        }
    } else {
        constexpr int W = LPR * V;          // columns a lane group covers
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float* v = which ? db : dw;
            if (which) __syncthreads();
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) meet[g * W + (c * LPR + l) * VEC + i] = v[c * VEC + i];
            __syncthreads();
            for (int col = tid; col < a.C; col += kThreads) {
                float s = 0.f;
#pragma unroll 4
                for (int k = 0; k < G; ++k) s += meet[k * W + col];
                float& to = part[which * a.C + col];
                to = a.more ? to + s : s;
            }
        }
    }
}

// dw and db from the workgroups' partial sums: 16 columns a workgroup (of the 2 C), 64 lanes a column, each over every 64th
// partial sum (eight loads in flight), then a tree over the 64.
__global__ __launch_bounds__(1024) void norm_grad_sum_kernel(const float* part, int parts, int C, void* dgamma, void* dbeta,
                                                             int dtype) {
    __shared__ float meet[64][17];
    const int lc = threadIdx.x & 15, sl = threadIdx.x >> 4, col = blockIdx.x * 16 + lc;
    float s = 0.f;
    if (col < 2 * C) {
        const float* p = part + col;
        for (int k = sl; k < parts; k += 64 * 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + 64 * j < parts ? p[(long long)(k + 64 * j) * 2 * C] : 0.f;
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
    }
    meet[sl][lc] = s;
    for (int h = 32; h >= 1; h >>= 1) {
        __syncthreads();
        if (sl < h) meet[sl][lc] += meet[sl + h][lc];
    }
    if (sl == 0 && col < 2 * C) {
        const float v = meet[0][lc];
        void* out = col < C ? dgamma : dbeta;
        const int c = col < C ? col : col - C;
        if (out) {
            if (dtype == YDET_BF16) static_cast<__bf16*>(out)[c] = (__bf16)v;
            else static_cast<float*>(out)[c] = v;
        }
    }
}

// Workgroups of the gradient kernel: by rows alone, so that the size of the workspace is known without a GPU.  At least 8 rows
// each (a partial sum, written and read, costs as much as three rows of bf16; with 2 rows each 3000 x 4096 took 48 us instead of
// 31), at most 1024 workgroups (four a CU).
static int grad_blocks(long long rows) {
    const long long n = (rows + 7) / 8;
    return (int)(n < 1 ? 1 : n > 1024 ? 1024 : n);
}

template <typename T, bool RAG, int LPR, int CH>
static int launch_grad(const GradArgs& a, int blocks, hipStream_t stream) {
    constexpr int RPT = CH == 1 ? 2 : 1;
    static_assert(kChain % RPT == 0, "rows of a lane group");
    const long long step = a.part ? (long long)blocks * (kThreads / LPR) * kChain : a.rows;
    for (long long row = 0; row < a.rows; row += step) {
        GradArgs b = a;
        b.rows = a.rows - row < step ? a.rows - row : step;
        b.dy += row * a.dy_ld * (long long)sizeof(T), b.x += row * a.x_ld * (long long)sizeof(T);
        if (a.dx) b.dx += row * a.dx_ld * (long long)sizeof(T);
        b.mean += row, b.rstd += row, b.more = row > 0;
        hipLaunchKernelGGL((norm_grad_kernel<T, RAG, LPR, CH, RPT>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, b);
        YDET_CHECK_LAUNCH("layer norm gradient");
    }
    return YDET_OK;
}

// Rows up to this length stay inside a wave, whose sums need no barrier (23104 x 2048 in bf16: 66 us, over a workgroup's lanes 70).
constexpr int kGradWaveCols = 2048;
template <typename T, bool RAG>
static int launch_grad_shape(const GradArgs& a, int blocks, hipStream_t stream) {
    const Shape s = shape_of(a.C, 16 / (int)sizeof(T), kGradWaveCols);
#define YDET_ROWS(L, K) \
    if (s.lpr == L && s.ch == K) return launch_grad<T, RAG, L, K>(a, blocks, stream);
    YDET_ROWS(4, 1) YDET_ROWS(8, 1) YDET_ROWS(16, 1) YDET_ROWS(32, 1) YDET_ROWS(64, 1) YDET_ROWS(64, 2) YDET_ROWS(64, 4) YDET_ROWS(256, 4)
    if constexpr (sizeof(T) == 4) {
        YDET_ROWS(64, 8) YDET_ROWS(256, 8)
    } else {
        YDET_ROWS(256, 2)
    }
#undef YDET_ROWS
    return fail(YDET_ERR_ARG, "layer_norm_backward: no kernel for %d channels", a.C);
}

}  // namespace rows
}  // namespace ydet

using namespace ydet;
using namespace ydet::rows;

extern "C" size_t ydet_layer_norm_backward_workspace_bytes(int64_t rows, int C) {
    if (rows < 0 || C <= 0 || C > kMaxC) return 0;
    return (size_t)grad_blocks(rows) * 2 * C * sizeof(float);
}

extern "C" int ydet_layer_norm_backward(const ydet_layer_norm_grad_desc* d, void* ws, size_t ws_bytes, void* stream) {
    clear_error();
    YDET_CHECK_ARG(d, "layer_norm_backward: null descriptor");
    YDET_CHECK_ARG(d->rows >= 0 && d->rows <= INT32_MAX && d->C > 0 && d->C <= kMaxC, "layer_norm_backward: rows=%lld C=%d (C 1..%d)",
                   (long long)d->rows, d->C, kMaxC);
    YDET_CHECK_ARG(dtype_ok(d->dtype) && dtype_ok(d->param_dtype), "layer_norm_backward: dtype %d / %d", d->dtype, d->param_dtype);
    const long long C = d->C;
    YDET_CHECK_ARG(d->x_coff >= 0 && d->dy_coff >= 0 && d->x_coff + C <= d->x_ld && d->dy_coff + C <= d->dy_ld &&
                       (!d->dx || (d->dx_coff >= 0 && d->dx_coff + C <= d->dx_ld)),
                   "layer_norm_backward: a slice of %d channels lies outside its rows", d->C);
    const bool params = d->dgamma || d->dbeta;
    if (!params && (!d->dx || d->rows == 0)) return YDET_OK;
    YDET_CHECK_ARG(d->rows == 0 || (d->x && d->dy && d->mean && d->rstd), "layer_norm_backward: null pointer");
    const size_t es = dtype_size(d->dtype), ps = dtype_size(d->param_dtype);
    GradArgs a{};
    a.x = static_cast<const char*>(d->x) + d->x_coff * es;
    a.dy = static_cast<const char*>(d->dy) + d->dy_coff * es;
    a.dx = d->dx ? static_cast<char*>(d->dx) + d->dx_coff * es : nullptr;
    YDET_CHECK_ARG(((uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.dx) % es == 0 && ((uintptr_t)d->dgamma | (uintptr_t)d->dbeta) % ps == 0,
                   "layer_norm_backward: misaligned tensor");
    int blocks = grad_blocks(d->rows);
    if (params) {
        YDET_CHECK_ARG(ws && (uintptr_t)ws % 4 == 0, "layer_norm_backward: the weight's gradient needs a workspace");
        const size_t need = (size_t)blocks * 2 * d->C * sizeof(float);
        if (ws_bytes < need)
            return fail(YDET_ERR_WORKSPACE, "layer_norm_backward: workspace %zu < %zu bytes", ws_bytes, need);
        a.part = static_cast<float*>(ws);
    }
    a.gamma = static_cast<const char*>(d->gamma), a.mean = d->mean, a.rstd = d->rstd, a.rows = d->rows, a.C = d->C;
    a.x_ld = d->x_ld, a.dy_ld = d->dy_ld, a.dx_ld = d->dx_ld, a.param_dtype = d->param_dtype;
    hipStream_t s = as_stream(stream);
    if (d->rows > 0) {
        int rc;
        if (d->dtype == YDET_BF16)
            rc = d->C % 8 ? launch_grad_shape<__bf16, true>(a, blocks, s) : launch_grad_shape<__bf16, false>(a, blocks, s);
        else
            rc = d->C % 4 ? launch_grad_shape<float, true>(a, blocks, s) : launch_grad_shape<float, false>(a, blocks, s);
        if (rc != YDET_OK) return rc;
    }
    if (params) {
        hipLaunchKernelGGL(norm_grad_sum_kernel, dim3((unsigned)((2 * d->C + 15) / 16)), dim3(1024), 0, s, a.part,
                           d->rows > 0 ? blocks : 0, d->C, d->dgamma, d->dbeta, d->param_dtype);
        YDET_CHECK_LAUNCH("layer norm gradient of the weight");
    }
    return YDET_OK;
}
