// gfx950 kernels of a context layer over all the tokens of a study, row by row: layer norm with its gradients,
// and rotary positions of several axes; their C ABI is in include/d8s_hip.h.
//
// Layer norm, per row x of `width` values: mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps),
//   xh = (x - mu) r,  y = xh w + b;
//   g = dy w,  dx = r (g - mean g - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy.
// All sums are float32; the variance is of the centred values (a second look at the registers), so a large mean
// costs no digits.  Bound by memory: a row is read once into the registers of the 16 lanes, the wave or the
// workgroup it is shared between, everything else happens there, and it is written once.  Measured, 98303 rows of 1024
// bfloat16: forward 76 us (5.3 TB/s; a large copy on this card 5.2), gradients 111 us (5.4 TB/s) and 8 us for the
// columns' sums.  That is the best width of 16 bits; others, of 10 to 26 million values: forward 2.4 .. 4.7 TB/s, gradients
// 1.4 .. 3.5 (2406 x 4877 20 and 49 us, 20000 x 1300 29 and 73, 3000 x 8000 22 and 64), where the last vector is
// read value by value, few waves are resident (32 values a thread) or the parts of the columns' sums are as large as the
// rows.  float32: 4.0 .. 5.5 and 2.9 .. 5.0.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "d8s_elem.h"
#include "d8s_hip.h"
#include "d8s_host.h"

namespace {

using namespace d8s;

#define CREQ(cond, msg) \
    do { if (!(cond)) return d8s_host_fail((int)hipErrorInvalidValue, std::string(what) + ": " + (msg)); } while (0)

constexpr int NORM_MAX = 16384;

// ---- layer norm -----------------------------------------------------------------------------------
// TPR threads share a row, each holding E of its values in vectors of V (16 bytes): vector v of thread t holds columns
// (v TPR + t) V ...  A row's last vector, where V does not divide the width, is read value by value, which in short rows
// costs up to half of the time.  There (WHOLE: eight values a thread) it ends with the row instead: its first `again`
// values are the ones before it once more, are left out of sums, and what is computed of them is the same bits as the
// other thread's, and both store it.  60000 rows of 300 bfloat16: forward 30 -> 25 us, gradients 57 -> 36; with more values
// a thread the sums' second form costs registers, and more than it gives (10000 rows of 2000: 53 -> 71 us).
struct Place {
    int c, n, again;                           // first column, columns from it to the row's end (0: none), and see above
};
template <int V, bool WHOLE>
DEV Place place(int vector, int width) {
    const int c = vector * V;
    if (c >= width) return {0, 0, 0};
    const int at = WHOLE && width >= V ? min(c, width - V) : c;
    return {at, width - at, c - at};
}
// The vector's own values, zeros in place of the others (whose bits may be anything)
template <int V>
DEV void only_own(const Place& at, const float* f, float* own) {
#pragma unroll
    for (int i = 0; i < V; ++i) own[i] = f[i];
    if (at.again != 0 || at.n < V) {
#pragma unroll
        for (int i = 0; i < V; ++i) own[i] = i >= at.again && i < at.n ? f[i] : 0.0f;
    }
}

template <class T, int TPR, int E>
struct NormShape {
    static constexpr int V = 16 / (int)sizeof(T), NV = E / V;
    static constexpr bool WHOLE = E == 8;
    static constexpr int THREADS = TPR > 256 ? TPR : 256, RPW = THREADS / TPR, WAVES = THREADS / 64;
    static_assert(E % V == 0, "whole vectors");
};

// Sums of a and b over the TPR threads of a row
template <int TPR, int WAVES>
DEV void row_sum2(float& a, float& b, float* red) {
    a = lanes_sum<(TPR < 64 ? TPR : 64)>(a);
    b = lanes_sum<(TPR < 64 ? TPR : 64)>(b);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x / 64;
        __syncthreads();                       // the last use of `red`
        if (threadIdx.x % 64 == 0) {
            red[w] = a;
            red[WAVES + w] = b;
        }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            a += red[i];
            b += red[WAVES + i];
        }
    }
}

template <class T, class W, int TPR, int E>
__global__ __launch_bounds__((NormShape<T, TPR, E>::THREADS)) void k_norm(D8sNormArgs p) {
    using S = NormShape<T, TPR, E>;
    constexpr int V = S::V, NV = S::NV;
    __shared__ float red[2 * S::WAVES];
    const int t = threadIdx.x % TPR;
    // every thread of a workgroup runs as many turns (the sums of a shared row synchronise)
    for (int64_t r0 = (int64_t)blockIdx.x * S::RPW; r0 < p.rows; r0 += (int64_t)gridDim.x * S::RPW) {
        const int64_t r = r0 + threadIdx.x / TPR;
        const bool on = r < p.rows;                // (rows past the end: nothing read, nothing written)
        const T* x = (const T*)p.x + (on ? r : 0) * p.x_stride;
        float f[E];
        float sum = 0.0f, zero = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
            load_n<T, V>(x + at.c, on ? at.n : 0, f + v * V);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float own[V];
            if constexpr (S::WHOLE) only_own<V>(place<V, true>(v * TPR + t, p.width), f + v * V, own);
#pragma unroll
            for (int i = 0; i < V; ++i) sum += S::WHOLE ? own[i] : f[v * V + i];
        }
        row_sum2<TPR, S::WAVES>(sum, zero, red);
        const float mean = sum / (float)p.width;
        float sq = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[v * V + i] -= mean;
            if constexpr (S::WHOLE) {
                float own[V];
                only_own<V>(place<V, true>(v * TPR + t, p.width), f + v * V, own);
#pragma unroll
                for (int i = 0; i < V; ++i) sq = __builtin_fmaf(own[i], own[i], sq);
            } else {
                const int n = p.width - (v * TPR + t) * V;
#pragma unroll
                for (int i = 0; i < V; ++i) sq = i < n ? __builtin_fmaf(f[v * V + i], f[v * V + i], sq) : sq;
            }
        }
        row_sum2<TPR, S::WAVES>(sq, zero, red);
        const float rstd = 1.0f / sqrtf(sq / (float)p.width + p.eps);
        if (!on) continue;
        if (t == 0 && p.mean) {
            p.mean[r] = mean;
            p.rstd[r] = rstd;
        }
        T* y = (T*)p.y + r * p.width;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
            if (at.n == 0) continue;
            float w[V], b[V], o[V];
            load_n<W, V>((const W*)p.w + at.c, at.n, w);
            if (p.b) load_n<W, V>((const W*)p.b + at.c, at.n, b);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = __builtin_fmaf(f[v * V + i] * rstd, w[i], p.b ? b[i] : 0.0f);
            store_n<T, V>(y + at.c, at.n, o);
        }
    }
}

// dx of the rows, and per workgroup the sums over its rows of dy xh and dy: partial[workgroup][2][width].
template <class T, class W, int TPR, int E>
__global__ __launch_bounds__((NormShape<T, TPR, E>::THREADS)) void k_norm_back(D8sNormArgs p) {
    using S = NormShape<T, TPR, E>;
    constexpr int V = S::V, NV = S::NV, RPW = S::RPW;
    __shared__ float red[2 * S::WAVES];
    __shared__ float part[RPW > 1 ? RPW * TPR * E : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const float inv = 1.0f / (float)p.width;
    float w[E], dw[E], db[E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
        load_n<W, V>((const W*)p.w + at.c, at.n, w + v * V);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.0f;
    // every thread of a workgroup runs as many turns (the sums of a shared row synchronise)
    for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < p.rows; r0 += (int64_t)gridDim.x * RPW) {
        const int64_t r = r0 + sub;
        const bool on = r < p.rows;
        const T* x = (const T*)p.x + (on ? r : 0) * p.x_stride;
        const T* dy = (const T*)p.dy + (on ? r : 0) * p.dy_stride;
        const float mean = on ? p.mean[r] : 0.0f, rstd = on ? p.rstd[r] : 0.0f;
        float f[E], g[E];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
            const int n = on ? at.n : 0;
            load_n<T, V>(x + at.c, n, f + v * V);
            load_n<T, V>(dy + at.c, n, g + v * V);
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            f[i] = (f[i] - mean) * rstd;
            dw[i] = __builtin_fmaf(g[i], f[i], dw[i]);
            db[i] += g[i];
            g[i] *= w[i];
            if constexpr (!S::WHOLE) {         // (past the row's end dy and w are zeros: nothing is added)
                s1 += g[i];
                s2 = __builtin_fmaf(g[i], f[i], s2);
            }
        }
        if constexpr (S::WHOLE) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float own[V];
                only_own<V>(place<V, true>(v * TPR + t, p.width), g + v * V, own);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s1 += own[i];
                    s2 = __builtin_fmaf(own[i], f[v * V + i], s2);
                }
            }
        }
        row_sum2<TPR, S::WAVES>(s1, s2, red);
        s1 *= inv;
        s2 *= inv;
        if (!on) continue;
        T* dx = (T*)p.dx + r * p.width;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
            if (at.n == 0) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
                o[i] = rstd * (g[v * V + i] - __builtin_fmaf(f[v * V + i], s2, s1));
            store_n<T, V>(dx + at.c, at.n, o);
        }
    }
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.width;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float* a = k ? db : dw;
        if constexpr (RPW > 1) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (!S::WHOLE) part[sub * TPR * E + (v * TPR + t) * V + i] = a[v * V + i];
                    else if (i >= at.again && i < at.n) part[sub * TPR * E + at.c + i] = a[v * V + i];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.width; c += S::THREADS) {
                float s = part[c];
#pragma unroll
                for (int i = 1; i < RPW; ++i) s += part[i * TPR * E + c];
                out[k * p.width + c] = s;
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const Place at = place<V, S::WHOLE>(v * TPR + t, p.width);
                store_n<float, V>(out + k * p.width + at.c, at.n, a + v * V);
            }
        }
    }
}

// dw and db: the sums of the workgroups' parts, 32 columns a workgroup, 8 parts at a time, in a fixed order.
template <class W>
__global__ __launch_bounds__(256) void k_norm_cols(D8sNormArgs p, int parts) {
    __shared__ float red[8][33];
    const int c = blockIdx.x * 32 + threadIdx.x % 32, k = threadIdx.x / 32, n = 2 * p.width;
    float s = 0.0f;
    if (c < n) {
        const float* a = p.partial + c;
#pragma unroll 8
        for (int i = k; i < parts; i += 8) s += a[(int64_t)i * n];
    }
    red[k][threadIdx.x % 32] = s;
    __syncthreads();
    if (k == 0 && c < n) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
        if (c < p.width) ((W*)p.dw)[c] = (W)s;
        else if (p.db) ((W*)p.db)[c - p.width] = (W)s;
    }
}

// Rows per workgroup of the shape that runs `width`
int norm_rows(int width) { return width <= 128 ? 16 : width <= 2048 ? 4 : 1; }

// Workgroups of the gradients, each of which leaves a part of the columns' sums: four a compute unit keep enough rows
// in flight (98303 x 1024 bfloat16: 111 us; two a compute unit 165 us, and 4 us less for the sums).  Measured at that
// width: of few long rows the parts are as large as the rows themselves (3000 x 8000: 131 of 275 MB)
int norm_parts(const D8sNormArgs* a) {
    const int64_t per = norm_rows(a->width), all = (a->rows + per - 1) / per;
    return (int)std::min<int64_t>(all, 4 * d8s_host_cu_count());
}

template <class T, class W, int TPR, int E>
void norm_launch(const D8sNormArgs& a, bool back, hipStream_t st) {
    using S = NormShape<T, TPR, E>;
    if (!back) {
        const int64_t blocks = std::min<int64_t>((a.rows + S::RPW - 1) / S::RPW, 1 << 20);
        hipLaunchKernelGGL((k_norm<T, W, TPR, E>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, a);
        return;
    }
    const int parts = norm_parts(&a);
    hipLaunchKernelGGL((k_norm_back<T, W, TPR, E>), dim3(parts), dim3(S::THREADS), 0, st, a);
    hipLaunchKernelGGL((k_norm_cols<W>), dim3((2 * a.width + 31) / 32), dim3(256), 0, st, a, parts);
}

template <class T, class W>
void norm_width(const D8sNormArgs& a, bool back, hipStream_t st) {
    const int w = a.width;
    if (w <= 128) norm_launch<T, W, 16, 8>(a, back, st);
    else if (w <= 512) norm_launch<T, W, 64, 8>(a, back, st);
    else if (w <= 1024) norm_launch<T, W, 64, 16>(a, back, st);
    else if (w <= 2048) norm_launch<T, W, 64, 32>(a, back, st);
    else if (w <= 4096) norm_launch<T, W, 256, 16>(a, back, st);
    else if (w <= 8192) norm_launch<T, W, 256, 32>(a, back, st);
    else norm_launch<T, W, 1024, 16>(a, back, st);
}

int norm_run(const D8sNormArgs* a, bool back, hipStream_t st) {
    const bool same = a->wdtype != D8S_F32;
    switch (a->dtype) {
        case D8S_F32: norm_width<float, float>(*a, back, st); break;
        case D8S_BF16: same ? norm_width<bf16, bf16>(*a, back, st) : norm_width<bf16, float>(*a, back, st); break;
        default: same ? norm_width<f16, f16>(*a, back, st) : norm_width<f16, float>(*a, back, st); break;
    }
    return d8s_host_launched(back ? "d8s_layer_norm_backward" : "d8s_layer_norm");
}

int norm_check(const D8sNormArgs* a, const char* what) {
    CREQ(a != nullptr, "null arguments");
    CREQ(a->dtype >= D8S_F32 && a->dtype <= D8S_F16, "dtype must be D8S_F32, D8S_BF16 or D8S_F16");
    CREQ(a->wdtype == D8S_F32 || a->wdtype == a->dtype, "wdtype must be D8S_F32 or dtype");
    CREQ(a->rows >= 1 && a->rows < (1ll << 31), "rows must be 1 .. 2^31 - 1");
    CREQ(a->width >= 1 && a->width <= NORM_MAX, "width must be 1 .. 16384");
    CREQ(a->x && a->w, "null pointer");
    CREQ(a->x_stride >= a->width || a->rows == 1, "x_stride smaller than width");
    return 0;
}

// ---- rotary positions -----------------------------------------------------------------------------
// Pair t of axis a turns by pos[a] base^(-t / pairs of a): (u, v) -> (u cos - v sin, u sin + v cos); the inverse,
// which is also the gradient, turns back.  The angle is formed in float64 as a number of turns and its whole turns
// dropped there (three operations), so any position an int32 holds is as exact as a small one; sine and cosine of
// the rest are float32.  A thread forms those of V pairs of a token once and applies them to the token's heads.
// Bound by memory: 49152 tokens of 20 heads of 128 float16 channels in 109 us (4.6 TB/s; 101 at best).
template <class T, bool ADJ>
__global__ __launch_bounds__(256) void k_rotary(D8sRotaryArgs p, int groups, int turned, int per) {
    constexpr int V = 16 / (int)sizeof(T);
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t token = id / groups;
    if (token >= (int64_t)p.B * p.S) return;
    const int g = (int)(id % groups);
    const int b = (int)(token / p.S), s = (int)(token % p.S);
    const int h0 = blockIdx.y * per, h1 = min(p.H, h0 + per);
    const T* x = (const T*)p.x + b * p.x_sb + s * p.x_ss + h0 * p.x_sh;
    T* y = (T*)p.y + b * p.y_sb + s * p.y_ss + h0 * p.y_sh;
    if (g >= turned) {                         // channels that no axis turns: 2 V of them copied
        const int c = 2 * p.pairs + (g - turned) * 2 * V, n = p.D - c;
        if (x == y) return;
        for (int h = h0; h < h1; ++h, x += p.x_sh, y += p.y_sh)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (n - k * V <= 0) break;
                float f[V];
                load_n<T, V>(x + c + k * V, n - k * V, f);
                store_n<T, V>(y + c + k * V, n - k * V, f);
            }
        return;
    }
    const int i0 = g * V, n = min(V, p.pairs - i0);
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int k = min(i0 + i, p.pairs - 1);
        const int64_t at = b * p.pos_sb + s * p.pos_ss + p.axis[k];
        const double pos = p.pos_type == 0 ? (double)((const int32_t*)p.pos)[at]
                         : p.pos_type == 1 ? (double)((const int64_t*)p.pos)[at] : (double)((const float*)p.pos)[at];
        const double turns = pos * p.freq[k];
        sincospif(2.0f * (float)(turns - rint(turns)), &sn[i], &cs[i]);
        sn[i] = p.inverse ? -sn[i] : sn[i];
    }
    for (int h = h0; h < h1; ++h, x += p.x_sh, y += p.y_sh) {
        float a[V], c[V], o[V], q[V];
        const int ca = ADJ ? 2 * i0 : i0, cb = ADJ ? 2 * i0 + V : i0 + p.pairs;
        const int na = ADJ ? 2 * n : n, nb = ADJ ? 2 * n - V : n;
        load_n<T, V>(x + ca, na, a);
        load_n<T, V>(x + cb, nb, c);
        if constexpr (ADJ) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float* f = i < V / 2 ? a : c;
                float* z = i < V / 2 ? o : q;
                const int e = 2 * (i % (V / 2));
                z[e] = f[e] * cs[i] - f[e + 1] * sn[i];
                z[e + 1] = f[e] * sn[i] + f[e + 1] * cs[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[i] = a[i] * cs[i] - c[i] * sn[i];
                q[i] = a[i] * sn[i] + c[i] * cs[i];
            }
        }
        store_n<T, V>(y + ca, na, o);
        store_n<T, V>(y + cb, nb, q);
    }
}

template <class T>
void rotary_run(const D8sRotaryArgs& a, hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    const int turned = (a.pairs + V - 1) / V, rest = a.D - 2 * a.pairs;
    const int groups = turned + (rest + 2 * V - 1) / (2 * V);
    const int64_t threads = (int64_t)a.B * a.S * groups, blocks = (threads + 255) / 256;
    // heads a thread: all of them share its sines and cosines, unless that leaves fewer than 8 waves a compute unit
    // (8 heads of 7128 tokens: 10.8 us with all heads a thread, 8.4 with two)
    const int64_t want = 8 * 64 * (int64_t)d8s_host_cu_count();
    const int ys = (int)std::min<int64_t>(a.H, std::max<int64_t>(1, want / std::max<int64_t>(1, threads)));
    const int per = (a.H + ys - 1) / ys;
    const dim3 grid((unsigned)blocks, (unsigned)ys);
    if (a.adjacent) hipLaunchKernelGGL((k_rotary<T, true>), grid, dim3(256), 0, st, a, groups, turned, per);
    else hipLaunchKernelGGL((k_rotary<T, false>), grid, dim3(256), 0, st, a, groups, turned, per);
}

}  // namespace

extern "C" int d8s_layer_norm(const D8sNormArgs* a, void* stream) {
    const char* what = "d8s_layer_norm";
    if (int rc = norm_check(a, what)) return rc;
    CREQ(a->y, "null pointer");
    CREQ((a->mean == nullptr) == (a->rstd == nullptr), "mean and rstd are given together or not at all");
    return norm_run(a, false, (hipStream_t)stream);
}

extern "C" int d8s_layer_norm_workspace(const D8sNormArgs* a, uint64_t* bytes) {
    const char* what = "d8s_layer_norm_workspace";
    if (int rc = norm_check(a, what)) return rc;
    CREQ(bytes != nullptr, "null arguments");
    *bytes = (uint64_t)norm_parts(a) * 2 * a->width * sizeof(float);
    return 0;
}

extern "C" int d8s_layer_norm_backward(const D8sNormArgs* a, void* stream) {
    const char* what = "d8s_layer_norm_backward";
    if (int rc = norm_check(a, what)) return rc;
    CREQ(a->dy && a->dx && a->dw && a->mean && a->rstd && a->partial, "null pointer");
    CREQ(a->dy_stride >= a->width || a->rows == 1, "dy_stride smaller than width");
    CREQ(a->partial_bytes >= (uint64_t)norm_parts(a) * 2 * a->width * sizeof(float),
         "partial smaller than d8s_layer_norm_workspace()");
    return norm_run(a, true, (hipStream_t)stream);
}

extern "C" int d8s_rotary(const D8sRotaryArgs* a, void* stream) {
    const char* what = "d8s_rotary";
    CREQ(a != nullptr, "null arguments");
    CREQ(a->dtype >= D8S_F32 && a->dtype <= D8S_F16, "dtype must be D8S_F32, D8S_BF16 or D8S_F16");
    CREQ(a->x && a->y && a->pos, "null pointer");
    CREQ(a->B >= 1 && a->S >= 1 && a->H >= 1 && a->H < 65536 && a->D >= 2, "bad sizes");
    CREQ(a->pairs >= 1 && a->pairs <= D8S_ROTARY_PAIRS && 2 * a->pairs <= a->D,
         "pairs must be 1 .. 256 and at most D / 2");
    CREQ((int64_t)a->B * a->S * (a->D / 8 + 2) < (1ll << 32) - 256, "too many tokens");
    CREQ(a->pos_type >= 0 && a->pos_type <= 2, "pos_type must be 0 (int32), 1 (int64) or 2 (float32)");
    for (int i = 0; i < a->pairs; ++i) CREQ(a->axis[i] < a->axes, "axis outside 0 .. axes - 1");
    switch (a->dtype) {
        case D8S_F32: rotary_run<float>(*a, (hipStream_t)stream); break;
        case D8S_BF16: rotary_run<bf16>(*a, (hipStream_t)stream); break;
        default: rotary_run<f16>(*a, (hipStream_t)stream); break;
    }
    return d8s_host_launched(what);
}
