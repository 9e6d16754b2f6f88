// gfx950 kernels of the optimizer that trains a head or a context layer: one AdamW step over many tensors at once,
// with moments in 32 or 8 bits; the C ABI is in include/d8s_hip.h.
//
// Per element, with the bias corrections c1 = 1 - beta1^t, c2 = 1 - beta2^t of step t formed on the host:
//   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2,
//   p = p (1 - lr decay) - lr / c1 * m / (sqrt(v) / sqrt(c2) + eps)
// in float32, each operation rounded by itself (no fused multiply-add), so a step has one result, to the bit.
//
// Moments in 8 bits: per block of 256 elements of a tensor a scale and a code an element.
//   m = s (c |c|) / 127^2, c in -127 .. 127, s the block's largest |m|;
//   sqrt(v) = s c^2 / 255^2, c in 0 .. 255, s the block's largest sqrt(v); c >= 1 where v > 0, so no moment that is
//   not zero is divided by as zero.
// The squares put the codes closer together towards zero, where most moments lie (the smallest step is 1 / 16129 of
// the block's largest |m| and 1 / 65025 of its largest sqrt(v)), and need no table.  The new p comes from the
// moments before they are rounded to their codes.
//
// Bound by memory: 28 bytes an element (float32 everywhere), 16 with 8-bit moments, whose three roots and a division an
// element come close to the memory's time: 98 M elements with bfloat16 gradients in 263 .. 311 us (14 bytes: 4.4 .. 5.2
// TB/s).  A wave takes four blocks of 256 elements in turn, four neighbouring elements a lane, so a block's scale is a
// reduction within the wave.
// The tensors' addresses travel in the kernel's arguments (at most 100 a launch): nothing is uploaded.
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

#define OREQ(cond, msg) \
    do { if (!(cond)) return d8s_host_fail((int)hipErrorInvalidValue, std::string(what) + ": " + (msg)); } while (0)

constexpr int BLK = D8S_ADAMW_BLOCK, TENSORS = 100, PER_WAVE = 4;
constexpr float TINY = 0x1p-100f;              // a smaller block scale cannot be divided by: its codes are zeros

// The tensors of one launch: tensor i owns the blocks first[i] .. first[i + 1) of the launch, block b of it the
// state's elements (at[i] + b) BLK ...
struct Table {
    void* p[TENSORS];
    const void* g[TENSORS];
    int64_t n[TENSORS], at[TENSORS];
    int32_t first[TENSORS + 1];
    int32_t count;
};

struct Step {
    float keep, beta1, one1, beta2, one2, root, eps, rate;
    const float* grad_scale;
    void *m, *v;
    float *m_scale, *v_scale;
};

DEV float lane_max_bits(float x) {             // the largest of 64 values >= 0 (or NaN, the largest of all), by bits
    unsigned u = __float_as_uint(x);
    auto up = [&](unsigned o) __attribute__((always_inline)) { u = u > o ? u : o; };
    up((unsigned)__builtin_amdgcn_mov_dpp((int)u, 0x128, 0xf, 0xf, true));
    up((unsigned)__builtin_amdgcn_mov_dpp((int)u, 0x124, 0xf, 0xf, true));
    up((unsigned)__builtin_amdgcn_mov_dpp((int)u, 0x122, 0xf, 0xf, true));
    up((unsigned)__builtin_amdgcn_mov_dpp((int)u, 0x121, 0xf, 0xf, true));
    u32x2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    u = r[0] > r[1] ? r[0] : r[1];
    r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0] > r[1] ? r[0] : r[1]);
}

// A block's scale from its largest value, and what multiplies a value to lie in 0 .. 1
DEV void block_scale(float top, float& scale, float& inv) {
    scale = top < TINY ? 0.0f : top;           // (NaN stays)
    inv = scale > 0.0f ? 1.0f / scale : 0.0f;
}

template <class P, class G, bool Q8>
__global__ __launch_bounds__(256) void k_adamw(Table t, Step s) {
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + threadIdx.x / 64));
    const int all = t.first[t.count];
    int b = wave * PER_WAVE;
    if (b >= all) return;
    const int end = min(all, b + PER_WAVE);
    int i = 0;                                 // the tensor of block b
    for (int lo = 0, hi = t.count; hi - lo > 1;) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= b) lo = mid; else hi = mid;
        i = lo;
    }
    const float gs = s.grad_scale ? *s.grad_scale : 1.0f;
    for (; b < end; ++b) {
        while (b >= t.first[i + 1]) ++i;
        const int64_t in = (int64_t)(b - t.first[i]) * BLK + 4 * lane, st = (t.at[i] + b - t.first[i]) * BLK + 4 * lane;
        const int64_t left = t.n[i] - in;
        const int n = left > 4 ? 4 : left < 0 ? 0 : (int)left;
        P* pp = (P*)t.p[i] + in;
        float p[4], g[4], m[4], v[4];
        load_n<P, 4>(pp, n, p);
        load_n<G, 4>((const G*)t.g[i] + in, n, g);
        uint32_t mc = 0, vc = 0;
        if constexpr (Q8) {
            mc = *((const uint32_t*)((const char*)s.m + st));
            vc = *((const uint32_t*)((const char*)s.v + st));
            const float ms = s.m_scale[st / BLK] * (float)(1.0 / 16129.0), vs = s.v_scale[st / BLK] * (float)(1.0 / 65025.0);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float c = (float)(int8_t)(mc >> (8 * k)), d = (float)((vc >> (8 * k)) & 255), r = d * d * vs;
                m[k] = c * fabsf(c) * ms;
                v[k] = r * r;
            }
        } else {
            load_n<float, 4>((const float*)s.m + st, 4, m);
            load_n<float, 4>((const float*)s.v + st, 4, v);
        }
        float r[4];
        float mtop = 0.0f, rtop = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = s.grad_scale ? g[k] * gs : g[k];
            m[k] = m[k] * s.beta1 + x * s.one1;
            v[k] = v[k] * s.beta2 + x * x * s.one2;
            r[k] = sqrtf(v[k]);
            p[k] = p[k] * s.keep - m[k] / (r[k] * s.root + s.eps) * s.rate;
        }
        store_n<P, 4>(pp, n, p);
        if constexpr (Q8) {
            // (by bits, so that a NaN is the largest and marks its block)
            unsigned mt = 0, rt = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                mt = max(mt, __float_as_uint(fabsf(m[k])));
                rt = max(rt, __float_as_uint(fabsf(r[k])));
            }
            mtop = lane_max_bits(__uint_as_float(mt));
            rtop = lane_max_bits(__uint_as_float(rt));
            float ms, mi, rs, ri;
            block_scale(mtop, ms, mi);
            block_scale(rtop, rs, ri);
            // A code is a square root rounded to a whole number.  The hardware's root is within 2^-22 of the exactly
            // rounded one, so the two give the same code unless the root lies within 2^-13 of a half, which is
            // rare: then the wave rounds all of its block's codes from exact roots.  (The expansion of an exact root
            // is a dozen operations, and the step was bound by its operations: 337 -> 299 us for 98 M elements.)
            float mr[4], vr[4], worst = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float x = __builtin_amdgcn_sqrtf(fabsf(m[k]) * mi) * 127.0f, y = __builtin_amdgcn_sqrtf(r[k] * ri) * 255.0f;
                mr[k] = rintf(x);
                vr[k] = rintf(y);
                worst = fmaxf(worst, fmaxf(fabsf(x - mr[k]), fabsf(y - vr[k])));
            }
            if (__any(!(worst < 0.5f - 0x1p-13f))) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mr[k] = fminf(rintf(sqrtf(fabsf(m[k]) * mi) * 127.0f), 127.0f);
                    vr[k] = fminf(rintf(sqrtf(r[k] * ri) * 255.0f), 255.0f);
                }
            }
            mc = vc = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = (int)copysignf(mr[k], m[k]);
                const int d = (int)(r[k] > 0.0f && rs > 0.0f ? fmaxf(vr[k], 1.0f) : vr[k]);
                mc |= (uint32_t)(c & 255) << (8 * k);
                vc |= (uint32_t)(d & 255) << (8 * k);
            }
            *((uint32_t*)((char*)s.m + st)) = mc;
            *((uint32_t*)((char*)s.v + st)) = vc;
            if (lane == 0) {
                s.m_scale[st / BLK] = ms;
                s.v_scale[st / BLK] = rs;
            }
        } else {
            store_n<float, 4>((float*)s.m + st, 4, m);
            store_n<float, 4>((float*)s.v + st, 4, v);
        }
    }
}

// The values that 8-bit moments stand for
__global__ __launch_bounds__(256) void k_adamw_moments(const uint32_t* mc, const uint32_t* vc, const float* ms,
                                                       const float* vs, float* m, float* v, int64_t words) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const uint32_t a = mc[i], b = vc[i];
        const float sa = ms[i / (BLK / 4)] * (float)(1.0 / 16129.0), sb = vs[i / (BLK / 4)] * (float)(1.0 / 65025.0);
        float x[4], y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float c = (float)(int8_t)(a >> (8 * k)), d = (float)((b >> (8 * k)) & 255), r = d * d * sb;
            x[k] = c * fabsf(c) * sa;
            y[k] = r * r;
        }
        store_n<float, 4>(m + 4 * i, 4, x);
        store_n<float, 4>(v + 4 * i, 4, y);
    }
}

template <class P, class G>
void adamw_launch(const Table& t, const Step& s, bool q8, hipStream_t st) {
    const unsigned grid = (unsigned)((t.first[t.count] + 4 * PER_WAVE - 1) / (4 * PER_WAVE));
    if (q8) hipLaunchKernelGGL((k_adamw<P, G, true>), dim3(grid), dim3(256), 0, st, t, s);
    else hipLaunchKernelGGL((k_adamw<P, G, false>), dim3(grid), dim3(256), 0, st, t, s);
}

void adamw_types(const Table& t, const Step& s, const D8sAdamwArgs* a, hipStream_t st) {
    const bool q8 = a->bits == 8;
    if (a->dtype == D8S_F32) {
        if (a->grad_dtype == D8S_F32) adamw_launch<float, float>(t, s, q8, st);
        else if (a->grad_dtype == D8S_BF16) adamw_launch<float, bf16>(t, s, q8, st);
        else adamw_launch<float, f16>(t, s, q8, st);
    } else if (a->dtype == D8S_BF16) {
        if (a->grad_dtype == D8S_F32) adamw_launch<bf16, float>(t, s, q8, st);
        else adamw_launch<bf16, bf16>(t, s, q8, st);
    } else {
        if (a->grad_dtype == D8S_F32) adamw_launch<f16, float>(t, s, q8, st);
        else adamw_launch<f16, f16>(t, s, q8, st);
    }
}

}  // namespace

extern "C" int d8s_adamw(const D8sAdamwArgs* a, void* stream) {
    const char* what = "d8s_adamw";
    OREQ(a != nullptr, "null arguments");
    OREQ(a->bits == 32 || a->bits == 8, "bits must be 32 or 8");
    OREQ(a->dtype >= D8S_F32 && a->dtype <= D8S_F16 && a->grad_dtype >= D8S_F32 && a->grad_dtype <= D8S_F16,
         "dtype and grad_dtype must be D8S_F32, D8S_BF16 or D8S_F16");
    OREQ(a->dtype == D8S_F32 || a->grad_dtype == D8S_F32 || a->dtype == a->grad_dtype,
         "gradients of 16 bits beside parameters of another type of 16 bits");
    OREQ(a->tensors && a->count >= 1, "no tensors");
    OREQ(a->m && a->v && (a->bits == 32 || (a->m_scale && a->v_scale)), "null state");
    OREQ(((uintptr_t)a->m & 3) == 0 && ((uintptr_t)a->v & 3) == 0, "state not 4-byte aligned");
    OREQ(a->step >= 1, "step must be at least 1");
    OREQ(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1, "betas must be in [0, 1)");
    for (int i = 0; i < a->count; ++i) {
        const D8sAdamwTensor& x = a->tensors[i];
        OREQ(x.n >= 0 && (x.n == 0 || (x.p && x.g)), "null tensor");
        OREQ(x.at >= 0 && x.at % BLK == 0, "a tensor's place in the state must be a multiple of 256");
        OREQ(x.n <= (1ll << 38), "tensor too large");
    }
    Step s;
    s.keep = (float)(1.0 - a->lr * a->weight_decay);
    s.beta1 = (float)a->beta1;
    s.one1 = (float)(1.0 - a->beta1);
    s.beta2 = (float)a->beta2;
    s.one2 = (float)(1.0 - a->beta2);
    s.root = (float)(1.0 / sqrt(1.0 - pow(a->beta2, (double)a->step)));
    s.eps = (float)a->eps;
    s.rate = (float)(a->lr / (1.0 - pow(a->beta1, (double)a->step)));
    s.grad_scale = a->grad_scale;
    s.m = a->m;
    s.v = a->v;
    s.m_scale = a->m_scale;
    s.v_scale = a->v_scale;
    Table t;
    t.count = 0;
    t.first[0] = 0;
    constexpr int64_t MOST = 1 << 28;          // blocks a launch
    for (int i = 0; i < a->count; ++i) {
        const D8sAdamwTensor& x = a->tensors[i];
        for (int64_t done = 0, all = (x.n + BLK - 1) / BLK; done < all;) {
            if (t.count == TENSORS || t.first[t.count] == MOST) {
                adamw_types(t, s, a, (hipStream_t)stream);
                t.count = 0;
            }
            const int64_t take = std::min(all - done, MOST - t.first[t.count]);
            const int k = t.count++;
            t.p[k] = (char*)x.p + done * BLK * (a->dtype == D8S_F32 ? 4 : 2);
            t.g[k] = (const char*)x.g + done * BLK * (a->grad_dtype == D8S_F32 ? 4 : 2);
            t.n[k] = x.n - done * BLK;
            t.at[k] = x.at / BLK + done;
            t.first[k + 1] = t.first[k] + (int32_t)take;
            done += take;
        }
    }
    if (t.count) adamw_types(t, s, a, (hipStream_t)stream);
    return d8s_host_launched(what);
}

extern "C" int d8s_adamw_moments(const void* m_code, const void* v_code, const float* m_scale, const float* v_scale,
                                 int64_t n, float* m, float* v, void* stream) {
    const char* what = "d8s_adamw_moments";
    OREQ(m_code && v_code && m_scale && v_scale && m && v, "null pointer");
    OREQ(n >= BLK && n % BLK == 0, "n must be a positive multiple of 256");
    OREQ(((uintptr_t)m_code & 3) == 0 && ((uintptr_t)v_code & 3) == 0, "state not 4-byte aligned");
    const int64_t blocks = std::min<int64_t>((n / 4 + 255) / 256, 16384);
    hipLaunchKernelGGL(k_adamw_moments, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                       (const uint32_t*)m_code, (const uint32_t*)v_code, m_scale, v_scale, m, v, n / 4);
    return d8s_host_launched(what);
}
