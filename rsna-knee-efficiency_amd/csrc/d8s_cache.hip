// gfx950 kernels of a context layer's cache of keys and values in 8 bits: tokens appended, read back, and attended over by
// new tokens; the C ABI is in include/d8s_hip.h.
//
// Per key head, 64 tokens in a row are a block.  A block that is full is held as codes with one float32 scale: with a its largest
// |x|, int8 codes rint(127 x / a) of unit a / 127, or e4m3 codes of 448 x / a and unit a / 448.  The block that is not full yet
// (the tail) stays in the inputs' 16 bits, so a token is rounded once, with its block's final scale, and a cache does not depend on
// how its tokens were split over calls.
//
// Layout: keys [B][HK][blocks][64][D], values transposed, [B][HK][blocks][D][64], the tails [B][HK][64][D] and [B][HK][D][64]: both
// products of attention then read their operands as they lie in memory, 16 bytes a lane, and nothing is transposed between.
// int8 codes lie in memory as code + 128: one v_perm makes of two bytes the float16 numbers 1024 + byte, one addition the codes.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "d8s_elem.h"
#include "d8s_hip.h"
#include "d8s_host.h"

namespace {

using namespace d8s;

#define CREQ(cond, msg) \
    do { if (!(cond)) return d8s_host_fail((int)hipErrorInvalidValue, std::string(what) + ": " + (msg)); } while (0)

constexpr int NT = 256, BLK = D8S_CACHE_BLOCK;
constexpr float LOG2E = 1.4426950408889634f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x2 __attribute__((ext_vector_type(2)));
template <class T>
using Frag = T __attribute__((ext_vector_type(8)));
typedef Vec<uint16_t, 8> Raw;                  // 8 elements of 16 bits at any element's address

DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's length and how many of its T tokens are there
DEV int length_of(const D8sCache& c, int b) { return max(0, min(c.lengths[b], c.S)); }
DEV int count_of(const int32_t* counts, int b, int T) { return counts ? max(0, min(counts[b], T)) : T; }

// ---- append ----------------------------------------------------------------------------------------
// A workgroup owns one block of a key head's keys and values: it gathers the block's tokens (from the tail and from the input) in
// registers, 8 channels of D / 32 tokens a thread, reduces the largest |x| and writes the codes, values through LDS.  The first
// workgroup of a head, which alone reads the tail, then writes the new one.  The last workgroup of a row to arrive sets its length.
// Bound by memory: 16 studies of up to 6144 tokens, 8 heads of 128, bfloat16, 88 us for 302 MB while 400 MB written before still
// drain (written and read back 170 us for 806 MB, 4.7 TB/s beside a copy's 5.1).  (A tail copied value by value was 16 dependent loads: one
// study of 4 heads 15 us in place of 7.5.)
//
// A code is formed from x times TOP / a, one multiplication, in place of the exact quotient's dozen operations.  The product is within 2^-23
// of the quotient of two numbers of at most 11 bits (times TOP, 7 or 3 bits), which differs from every border between two
// codes by 2^-19 of itself or lies on it: so rounding the product to 20 bits behind its leading one gives a number on the same
// side of, or on, the same border, and the code of the exact quotient.
template <bool E4M3>
constexpr float CODE_TOP = E4M3 ? 448.0f : 127.0f;

DEV float snap(float y) { return __uint_as_float((__float_as_uint(y) + 4u) & ~7u); }

// The codes of four numbers, the first in the lowest byte
template <bool E4M3>
DEV uint32_t codes4(const float* y) {
    if constexpr (E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(snap(y[0]), snap(y[1]), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(snap(y[2]), snap(y[3]), w, true);
    } else {
        // adding 1.5 x 2^23 rounds to a whole number (ties to even) and leaves it in the low bits; 128 more are the bias
        constexpr float MAGIC = 12582912.0f + 128.0f;
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(snap(y[i]) + MAGIC);
        const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0c);
        return lo | hi;
    }
}

// Whether this is the last of a row's `all` workgroups to get here; the counters are zeros again then.  Every workgroup has read its row's
// length by that time: the length was used before, so it was there before the atomic is issued, and nothing else is handed on (an
// order of memory would write the L2 back in every workgroup: the 16 studies took 1076 us, and 300 without).  Additions to one line
// follow each other at 12 ns, so many workgroups count in 16 lines first (300 -> 95 us).
DEV bool last_of_row(int32_t* counters, int id, int all) {
    const auto last = [](int32_t* at, int n) __attribute__((always_inline)) {
        if (__hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != n - 1) return false;
        __hip_atomic_store(at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return true;
    };
    constexpr int LINE = 32, LINES = D8S_CACHE_ARRIVED / LINE - 1;
    if (all < 4 * LINES) return last(counters, all);
    const int line = id % LINES;
    return last(counters + (1 + line) * LINE, (all + LINES - 1 - line) / LINES) && last(counters, LINES);
}

template <class T, bool E4M3, int D>
__global__ __launch_bounds__(NT) void k_cache_append(D8sCacheAppendArgs p, int chunks) {
    constexpr int P = D / 8, N = D / 32;       // threads a token, tokens a thread
    constexpr int PITCH = BLK + 4;             // bytes between channels of the transposed codes
    __shared__ uint32_t tops[2][NT / 64];
    __shared__ uint32_t turned[D * PITCH / 4];
    const D8sCache& c = p.c;
    const int id = blockIdx.x, hk = id % c.HK, i = id / c.HK % chunks, b = id / c.HK / chunks;
    const int n0 = length_of(c, b), n1 = n0 + min(count_of(p.counts, b, p.T), c.S - n0);
    const int j = n0 / BLK + i, nb = c.S / BLK;
    const int64_t head = (int64_t)b * c.HK + hk;
    const T* ks = (const T*)p.k + b * p.k_sb + hk * p.k_sh;
    const T* vs = (const T*)p.v + b * p.v_sb + hk * p.v_sh;
    T* kt = (T*)c.k_tail + head * BLK * D;
    T* vt = (T*)c.v_tail + head * BLK * D;
    if ((j + 1) * BLK <= n1) {
        const int ch = threadIdx.x % P * 8, t0 = threadIdx.x / P * N;
        Vec<T, 8> raw[2][N];
        if (j * BLK >= n0) {                   // (all loads at once)
            const int64_t at = j * BLK + t0 - n0;
#pragma unroll
            for (int t = 0; t < N; ++t) {
                raw[0][t] = *(const Vec<T, 8>*)(ks + (at + t) * p.k_ss + ch);
                raw[1][t] = *(const Vec<T, 8>*)(vs + (at + t) * p.v_ss + ch);
            }
        } else {
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const int at = j * BLK + t0 + t;
                if (at >= n0) {
                    raw[0][t] = *(const Vec<T, 8>*)(ks + (int64_t)(at - n0) * p.k_ss + ch);
                    raw[1][t] = *(const Vec<T, 8>*)(vs + (int64_t)(at - n0) * p.v_ss + ch);
                } else {
                    raw[0][t] = *(const Vec<T, 8>*)(kt + (t0 + t) * D + ch);
#pragma unroll
                    for (int k = 0; k < 8; ++k) raw[1][t][k] = vt[(ch + k) * BLK + t0 + t];
                }
            }
        }
        uint32_t top[2] = {};                  // by bits, so that what is not finite is the largest
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int k = 0; k < 8; ++k) top[x] = max(top[x], __float_as_uint((float)raw[x][t][k]) & 0x7fffffffu);
#pragma unroll
            for (int o = 32; o >= 1; o /= 2) top[x] = max(top[x], (uint32_t)__shfl_xor((int)top[x], o));
            if (threadIdx.x % 64 == 0) tops[x][threadIdx.x / 64] = top[x];
        }
        __syncthreads();
        const int64_t block = head * nb + j;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t most = max(max(tops[x][0], tops[x][1]), max(tops[x][2], tops[x][3]));
            const bool finite = most < 0x7f800000u;
            const float a = __uint_as_float(most);
            const float up = a < 0x1p-64f ? 0x1p64f : 1.0f;              // (the quotient could pass float32)
            const float by = a > 0.0f && finite ? CODE_TOP<E4M3> / (a * up) : 0.0f;
            if (threadIdx.x == 0) (x ? c.v_scale : c.k_scale)[block] = finite ? a / CODE_TOP<E4M3> : __builtin_nanf("");
            uint32_t w[N][2];
#pragma unroll
            for (int t = 0; t < N; ++t) {
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = finite ? (float)raw[x][t][k] * up * by : 0.0f;
                w[t][0] = codes4<E4M3>(y);
                w[t][1] = codes4<E4M3>(y + 4);
            }
            if (x == 0) {
                uint8_t* o = (uint8_t*)c.k_code + block * BLK * D + t0 * D + ch;
#pragma unroll
                for (int t = 0; t < N; ++t) *(u32x2*)(o + t * D) = u32x2{w[t][0], w[t][1]};
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t sel = 0x0c0c0400u + (k % 4) * 0x0101u;
                    uint8_t* o = (uint8_t*)turned + (ch + k) * PITCH + t0;
                    const uint32_t lo = __builtin_amdgcn_perm(w[1][k / 4], w[0][k / 4], sel);
                    if constexpr (N == 4) *(uint32_t*)o = lo | __builtin_amdgcn_perm(w[N - 1][k / 4], w[N - 2][k / 4], sel) << 16;
                    else *(uint16_t*)o = (uint16_t)lo;
                }
                __syncthreads();
                uint8_t* o = (uint8_t*)c.v_code + block * BLK * D;
#pragma unroll
                for (int s = 0; s < D * BLK / 16 / NT; ++s) {
                    const int e = s * NT + threadIdx.x, at = (e / 4 * PITCH + e % 4 * 16) / 4;
                    *(u32x4*)(o + e * 16) = u32x4{turned[at], turned[at + 1], turned[at + 2], turned[at + 3]};
                }
            }
        }
    }
    if (i == 0 && n1 % BLK != 0 && n1 > n0) {
        const int last = n1 / BLK * BLK, ch = threadIdx.x % P * 8, t0 = threadIdx.x / P * N;
        Vec<T, 8> raw[2][N];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int64_t at = min(max(last + t0 + t, n0), n1 - 1) - n0;
            raw[0][t] = *(const Vec<T, 8>*)(ks + at * p.k_ss + ch);
            raw[1][t] = *(const Vec<T, 8>*)(vs + at * p.v_ss + ch);
        }
        __syncthreads();                       // the old tail has been read
#pragma unroll
        for (int t = 0; t < N; ++t)
            if (last + t0 + t >= n0 && last + t0 + t < n1) {
                *(Vec<T, 8>*)(kt + (t0 + t) * D + ch) = raw[0][t];
#pragma unroll
                for (int k = 0; k < 8; ++k) vt[(ch + k) * BLK + t0 + t] = raw[1][t][k];
            }
    }
    __syncthreads();
    if (threadIdx.x == 0 && last_of_row(p.arrived + b * D8S_CACHE_ARRIVED, id % (c.HK * chunks), c.HK * chunks)) {
        const int lost = count_of(p.counts, b, p.T) - (n1 - n0);
        if (lost) p.dropped[b] += lost;
        c.lengths[b] = n1;
    }
}

// ---- reading back ------------------------------------------------------------------------------------
// The values that a code stands for are code * scale, rounded once to float32 and then to the output's type.  The heads of a token are
// neighbours in the output, so neighbouring workgroups run them (88 -> 82 us for the 16 studies' 503 MB, 6.1 TB/s).
template <bool E4M3>
DEV float value_of(uint32_t word, int k) {
    const uint32_t byte = word >> (8 * k) & 255;
    if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
    else return (float)((int)byte - 128);
}

constexpr int READ_WGS = 1 << 23;              // in a row of the grid (one dimension has fewer than 2^32 threads)
template <class T, class O, bool E4M3, int D>
__global__ __launch_bounds__(NT) void k_cache_read(D8sCacheReadArgs p, int blocks) {
    constexpr int P = D / 8, N = D / 32, PITCH = BLK + 4;
    __shared__ uint32_t turned[D * PITCH / 4];
    const D8sCache& c = p.c;
    const int id = blockIdx.y * READ_WGS + blockIdx.x, hk = id % c.HK, values = id / c.HK & 1, j = id / c.HK / 2 % blocks, b = id / c.HK / 2 / blocks;
    if (b >= c.B) return;
    const int n = length_of(c, b), nb = c.S / BLK;
    const int64_t head = (int64_t)b * c.HK + hk, block = head * nb + j;
    const int ch = threadIdx.x % P * 8, t0 = threadIdx.x / P * N;
    const bool full = (j + 1) * BLK <= n;
    float x[N][8] = {};
    if (full) {
        const uint8_t* code = (const uint8_t*)(values ? c.v_code : c.k_code) + block * BLK * D;
        const float scale = (values ? c.v_scale : c.k_scale)[block];
        if (values) {
#pragma unroll
            for (int s = 0; s < D * BLK / 16 / NT; ++s) {
                const int e = s * NT + threadIdx.x, at = (e / 4 * PITCH + e % 4 * 16) / 4;
                const u32x4 w = *(const u32x4*)(code + e * 16);
#pragma unroll
                for (int k = 0; k < 4; ++k) turned[at + k] = w[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint8_t* o = (const uint8_t*)turned + (ch + k) * PITCH + t0;
                uint32_t w;
                if constexpr (N == 4) w = *(const uint32_t*)o;
                else w = *(const uint16_t*)o;
#pragma unroll
                for (int t = 0; t < N; ++t) x[t][k] = value_of<E4M3>(w, t) * scale;
            }
        } else {
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const u32x2 w = *(const u32x2*)(code + (t0 + t) * D + ch);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[t][k] = value_of<E4M3>(w[k / 4], k % 4) * scale;
            }
        }
    } else if (j * BLK < n) {
        const T* tail = (const T*)(values ? c.v_tail : c.k_tail) + head * BLK * D;
#pragma unroll
        for (int t = 0; t < N; ++t)
            if (j * BLK + t0 + t < n)
#pragma unroll
                for (int k = 0; k < 8; ++k) x[t][k] = (float)(values ? tail[(ch + k) * BLK + t0 + t] : tail[(t0 + t) * D + ch + k]);
    }
    O* o = (O*)(values ? p.v : p.k);
#pragma unroll
    for (int t = 0; t < N; ++t) {
        const int at = j * BLK + t0 + t;
        if (at < p.tokens) store_n<O, 8>(o + (((int64_t)b * p.tokens + at) * c.HK + hk) * D + ch, 8, x[t]);
    }
}

// ---- attention, few rows -------------------------------------------------------------------------------
// Row r of a key head is query head r % G of new token r / G (G query heads share the key head).  With s = scale q k over the visible
// keys, P = softmax(s), out = P v.  A block's scale multiplies its scores, and its part of the sum P v, in float32.
//
// A wave runs 16 rows over one block of 64 tokens at a time on v_mfma_f32_16x16x32_f16.  Codes are whole numbers up to 127 or of 4 bits, exact
// in float16; queries in bfloat16 are brought into float16's range by a power of two a row (exact, for what is not 2^-29 of the
// row's largest).  Lane l holds row l % 16 (of queries) or 4 (l / 16) + register (of keys) of a product's result; key row
// 4 g + r of tile u is token 16 g + 4 u + r of the block, so a lane's weights of all four tiles are those of tokens 16 g .. 16 g + 15: what
// it reads of a channel's row of the transposed values, 16 bytes, is in the same order.
// P is rounded to float16 between the products (the matrix unit's full rate takes 16-bit operands; half a step is 2^-11 of each value,
// independent from value to value) after 2^NARROW_UP times (float16 holds little below 2^-14); the running maximum is raised only where a
// tile exceeds it by more than 2^RISE.
// Bound by memory: of a block's 16 KB (D = 128) a wave makes float16 numbers in 256 instructions and forms 32 products, and the next
// block's codes are in flight meanwhile.  64 requests of 8192 tokens, 32 heads on 8 key heads of 128: 176 us, 6.1 TB/s (vector
// instructions in the place of products, as for 16-bit keys, would be bound by them: twice the values a byte).
constexpr float RISE = 6.0f, NARROW_UP = 8.0f;
// Weights are up to 2^(NARROW_UP + RISE), and bfloat16 values up to float32's own limit: once values (of a scale) above 2^64 (HIGH) are met,
// sums are held times LOWER.  Parts of a row are left as means of values, which stay in range, with the sum of their weights.
constexpr float LOWER = 0x1p-64f, HIGH = 0x1p56f;
// Bits 15 and 31: whether the first and the second of two bfloat16 numbers is 2^64 or more, or none
DEV uint32_t high_values(uint32_t two) { return ((two & 0x7fff7fffu) + 0x20802080u) & 0x80008000u; }
// Of four such pairs a bit each, the first in the lowest
DEV uint32_t high_bits(const uint32_t* two) {
    uint32_t bits = 0;
#pragma unroll
    for (int y = 0; y < 4; ++y) bits |= (two[y] >> 15 & 1) << (2 * y) | (two[y] >> 31) << (2 * y + 1);
    return bits;
}

DEV f32x4 mfma(Frag<bf16> a, Frag<bf16> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
DEV f32x4 mfma(Frag<f16> a, Frag<f16> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Eight codes as float16 numbers
template <bool E4M3>
DEV Frag<f16> codes_frag(uint32_t lo, uint32_t hi) {
    f16x2 h[4];
    if constexpr (E4M3) {
        h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
        h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
        h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    } else {
        const f16x2 bias = {(f16)-1152.0f, (f16)-1152.0f};
        h[0] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) + bias;
        h[1] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) + bias;
        h[2] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) + bias;
        h[3] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) + bias;
    }
    return Frag<f16>{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// What a block's scores are times: the scale (with log2(e)), the scale of its keys, and for bfloat16 rows 2^-down.  The powers of two of the
// first and the last are joined and taken by the second, exactly: no product leaves float32 that the result does not.
template <class T>
DEV float unit_of(float scale, float keys, int down) {
    if constexpr (!__is_same(T, bf16)) return scale * keys;
    return ldexpf(keys, __builtin_amdgcn_frexp_expf(scale) - 1 - down) * (2.0f * __builtin_amdgcn_frexp_mantf(scale));
}

// Bits 0 .. 63 below n (any n)
DEV uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : ~(~0ull << n); }

// Max and sum over the four groups of 16 lanes, in every lane
DEV float groups_max(float x) {
    float a, b;
    swap16(x, a, b);
    swap32(fmaxf(a, b), a, b);
    return fmaxf(a, b);
}
DEV float groups_sum(float x) {
    float a, b;
    swap16(x, a, b);
    swap32(a + b, a, b);
    return a + b;
}

// Whether anything is seen, by the sum of the weights: not where it is zero; a sum that is not a number stays one
DEV bool any_weight(float sum) { return sum > 0.0f || sum != sum; }

// Shares of a row joined: their maximum and the sum of weights share by share, and what a share's mean counts
DEV float weight_of(u32x2 stats, float top) {
    const float m = __uint_as_float(stats[0]);
    return __uint_as_float(stats[1]) * (m == -INFINITY ? 0.0f : exp2_(m - top));
}
DEV void add_share(float& top, float& sum, u32x2 stats) {
    const float up = fmaxf(top, __uint_as_float(stats[0]));
    sum = sum * (top == -INFINITY ? 1.0f : exp2_(top - up)) + weight_of(stats, up);
    top = up;
}
// Of K threads' maxima and sums the maximum, and one over the sum (0 where nothing is seen)
template <int K>
DEV float sum_of(const float* sm, const float* ss, float& top) {
    top = sm[0];
#pragma unroll
    for (int x = 1; x < K; ++x) top = fmaxf(top, sm[x]);
    float sum = 0.0f;
#pragma unroll
    for (int x = 0; x < K; ++x) sum += weight_of(u32x2{__float_as_uint(sm[x]), __float_as_uint(ss[x])}, top);
    return any_weight(sum) ? 1.0f / sum : 0.0f;
}

// The blocks that queries at positions i0 .. i1 of a row of n tokens can see: those of the first tokens, then the window's
struct Blocks {
    int first, start, count;
    DEV int at(int i) const { return i < first ? i : start + i - first; }
};
DEV Blocks blocks_of(const D8sCacheAttnArgs& p, int n, int i0, int i1) {
    const int lo = max(0, i0 - p.left), hi = min(n - 1, i1 + p.right);
    if (i1 < 0 || hi < 0) return {0, 0, 0};
    const int start = lo / BLK, first = min((min(p.sinks, n) + BLK - 1) / BLK, start);
    return {first, start, first + max(0, hi / BLK - start + 1)};
}

// Which tile of rows a workgroup runs, of which group (a key head's share of blocks).  Workgroups go to the 8 XCDs in turn: all tiles
// of a group, which read the same blocks, are given to one, and the groups to all in turn.
struct Place {
    int tile, group;
};
DEV Place place_of(int tiles) {
    const int w = blockIdx.x, groups = gridDim.x / tiles, even = groups / 8 * 8 * tiles;
    if (w < even) return {w / 8 % tiles, w / 8 / tiles * 8 + w % 8};
    return {(w - even) % tiles, groups / 8 * 8 + (w - even) / tiles};
}

// What the shares of a row leave where there are several: the mean of its values, and before the means its maximum and the sum of its weights
struct Part {
    float* at;
    int cuts;
    int64_t rows;
    template <int D>
    DEV u32x2* stats(int cut, int64_t row) const { return (u32x2*)at + (cut * rows + row); }
    template <int D>
    DEV float* sums(int cut, int64_t row) const { return at + 2 * (cuts * rows + cuts * rows % 2) + (cut * rows + row) * D; }
};

// A tile of 16 rows of row b: its length and new tokens, the blocks they see; those in codes come first, and the block that is not
// full, if it is seen, is the last one
struct Rows {
    int n, cnt, full, coded;
    Blocks list;
    DEV bool tail() const { return coded < list.count; }
};
DEV Rows rows_of(const D8sCacheAttnArgs& p, int b, int rt) {
    const int G = p.H / p.c.HK, n = length_of(p.c, b), cnt = count_of(p.counts, b, p.T), full = n / BLK;
    const int tlo = rt * 16 / G, thi = min(min(rt * 16 + 15, p.T * G - 1) / G, cnt - 1);
    const Blocks list = tlo < cnt ? blocks_of(p, n, n - cnt + tlo, n - cnt + thi) : Blocks{0, 0, 0};
    return {n, cnt, full, list.count && list.at(list.count - 1) >= full ? list.count - 1 : list.count, list};
}

// The waves of a workgroup over blocks e0 .. e1 - 1 of a tile's rows, and its tail.  part_of(y): where what row y of the tile has is left
// (null statistics: it is all of the row, and goes to the output)
struct Left {
    u32x2* stats;
    float* sums;
};
template <class T, bool E4M3, int D, int W, class F>
DEV void rows_job(const D8sCacheAttnArgs& p, const Rows& a, int rt, int hk, int b, int e0, int e1, bool tail, F part_of) {
    constexpr int KL = D / 16, VL = D / 16, KS = D / 32, PITCH = D + 4;
    __shared__ float sm[W][16], sl[W][16];
    __shared__ float so[W][16][PITCH];
    const D8sCache& c = p.c;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), row = lane % 16, g = lane / 16;
    const int G = p.H / c.HK, rows = p.T * G, n = a.n, nb = c.S / BLK, full = a.full;
    const Blocks& list = a.list;
    const int r = rt * 16 + row, t = min(r, rows - 1) / G, h = hk * G + min(r, rows - 1) % G;
    const int i = n - a.cnt + t;               // the row's position
    const bool on = r < rows && t < a.cnt && i >= 0;
    const int64_t head = (int64_t)b * c.HK + hk;
    const uint16_t* qp = (const uint16_t*)p.q + b * p.q_sb + t * p.q_ss + h * p.q_sh;
    // queries: channels 64 (k / 2) + 16 g + 8 (k % 2) .. of step k
    Frag<f16> q[KS];
    int down = 0;                              // the power of two that a bfloat16 row was multiplied by
    {
        Frag<T> x[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) x[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 64 * (k / 2) + 16 * g + 8 * (k % 2)));
        if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) {
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int d = 0; d < 8; ++d) top = fmaxf(top, fabsf((float)x[k][d]));
            top = groups_max(top);
            down = top > 0.0f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int d = 0; d < 8; ++d) q[k][d] = (f16)ldexpf((float)x[k][d], down);
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k] = __builtin_bit_cast(Frag<f16>, x[k]);
        }
    }
    const float cs = p.scale * LOG2E;
    const int krow = 16 * (row / 4) + row % 4; // the lane's token of tile 0
    float m = -INFINITY, l = 0.0f, low = 1.0f;
    f32x4 acc[VL] = {};
    u32x4 kr[KL], vr[VL];
    float ks = 0.0f, vs = 0.0f;
    const uint8_t* kc = (const uint8_t*)c.k_code + head * nb * BLK * D + krow * D + 16 * g;
    const uint8_t* vc = (const uint8_t*)c.v_code + head * nb * BLK * D + row * BLK + 16 * g;
    const auto load_k = [&](int j) __attribute__((always_inline)) {
        const uint8_t* kp = kc + (int64_t)j * BLK * D;
#pragma unroll
        for (int x = 0; x < KL; ++x) kr[x] = *(const u32x4*)(kp + (x % 4) * 4 * D + x / 4 * 64);
        ks = c.k_scale[head * nb + j];
    };
    const auto load_v = [&](int j) __attribute__((always_inline)) {
        const uint8_t* vp = vc + (int64_t)j * BLK * D;
#pragma unroll
        for (int x = 0; x < VL; ++x) vr[x] = *(const u32x4*)(vp + x * 16 * BLK);
        vs = c.v_scale[head * nb + j];
    };
    // Weights of a block from its scores (times by), and the sums raised to a new maximum; visible bits of the row's 64 tokens
    const auto weights = [&](f32x4* s, float by, uint64_t vis) __attribute__((always_inline)) {
        const uint32_t mine = (uint32_t)(vis >> (16 * g));
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[u][x] = mine >> (4 * u + x) & 1 ? s[u][x] * by : -INFINITY;
                top = fmaxf(top, s[u][x]);
            }
        top = groups_max(top);
        if (__any(top > m + RISE)) {
            const float up = fmaxf(m, top), a = up == -INFINITY ? 1.0f : exp2_(m - up);
            m = up;
            l *= a;
#pragma unroll
            for (int d = 0; d < VL; ++d) acc[d] *= a;
        }
        const float base = (m == -INFINITY ? 0.0f : m) - NARROW_UP;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[u][x] = exp2_(s[u][x] - base);
                l += s[u][x];
            }
    };
    // (a row at a time: one that sees no such values may have ones that would not be left of it)
    const auto lower = [&](bool high) __attribute__((always_inline)) {
        const bool turn = high && low == 1.0f;
        if (!__any(turn)) return;
        low = turn ? LOWER : low;
#pragma unroll
        for (int d = 0; d < VL; ++d) acc[d] *= turn ? LOWER : 1.0f;
    };
    const auto visible = [&](int k0) __attribute__((always_inline)) {
        if (!on) return (uint64_t)0;
        return bits_below(min(i + p.right, n - 1) + 1 - k0) & (~bits_below(i - p.left - k0) | bits_below(p.sinks - k0));
    };
    int e = e0 + wave;
    if (e < e1) {
        load_k(list.at(e));
        load_v(list.at(e));
    }
    for (; e < e1; e += W) {
        const int j = list.at(e), next = list.at(min(e + W, e1 - 1));
        f32x4 s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            s[u] = f32x4{};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const u32x4 w = kr[u + k / 2 * 4];
                s[u] = mfma(codes_frag<E4M3>(w[k % 2 * 2], w[k % 2 * 2 + 1]), q[k], s[u]);
            }
        }
        const float by = unit_of<T>(cs, ks, down);
        load_k(next);
        const uint64_t vis = visible(j * BLK);
        weights(s, by, vis);
        if constexpr (__is_same(T, bf16)) lower(vs > HIGH && vis);
        const float scale = vis ? vs * low : 0.0f;         // (a scale that is not a number is not met by rows that see nothing of the block)
        Frag<f16> w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int x = 0; x < 8; ++x) w[k][x] = (f16)s[2 * k + x / 4][x % 4];
#pragma unroll
        for (int d = 0; d < VL; ++d) {
            f32x4 o = mfma(codes_frag<E4M3>(vr[d][0], vr[d][1]), w[0], f32x4{});
            o = mfma(codes_frag<E4M3>(vr[d][2], vr[d][3]), w[1], o);
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[d][x] = __builtin_fmaf(o[x], scale, acc[d][x]);
        }
        load_v(next);
    }
    if (tail && (e1 - e0) % W == wave) {       // the tail, in its own type
        const uint16_t* kt = (const uint16_t*)c.k_tail + head * BLK * D + krow * D + 16 * g;
        const uint16_t* vt = (const uint16_t*)c.v_tail + head * BLK * D + row * BLK + 16 * g;
        u32x4 kw[4 * KS], vw[2 * VL];          // (all its loads at once)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < KS; ++k) kw[4 * k + u] = *(const u32x4*)(kt + u * 4 * D + 64 * (k / 2) + 8 * (k % 2));
#pragma unroll
        for (int d = 0; d < VL; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) vw[2 * d + k] = *(const u32x4*)(vt + d * 16 * BLK + 8 * k);
        f32x4 s[4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const Frag<T> x = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 64 * (k / 2) + 16 * g + 8 * (k % 2)));
#pragma unroll
            for (int u = 0; u < 4; ++u) s[u] = mfma(__builtin_bit_cast(Frag<T>, kw[4 * k + u]), x, s[u]);
        }
        const uint64_t vis = visible(full * BLK);
        weights(s, cs, vis);
        const int there = n - full * BLK - 16 * g;          // of the lane's 16 tokens; what lies past them is not used
        uint32_t two[8] = {};                  // which of the lane's 16 tokens have high values
#pragma unroll
        for (int d = 0; d < VL; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                Raw v = __builtin_bit_cast(Raw, vw[2 * d + k]);
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = 8 * k + x < there ? v[x] : 0;
                vw[2 * d + k] = __builtin_bit_cast(u32x4, v);
                if constexpr (__is_same(T, bf16))
#pragma unroll
                    for (int x = 0; x < 4; ++x) two[4 * k + x] |= high_values(vw[2 * d + k][x]);
            }
        uint32_t high = high_bits(two) | high_bits(two + 4) << 8;
        if (__any(high)) {
#pragma unroll
            for (int o = 1; o < 16; o *= 2) high |= (uint32_t)__shfl_xor((int)high, o);
            uint64_t all = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) all |= (uint64_t)(uint32_t)__shfl((int)high, 16 * x) << (16 * x);
            lower(all & vis);
        }
        Frag<T> w[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int x = 0; x < 8; ++x) w[k][x] = (T)(s[2 * k + x / 4][x % 4] * low);
#pragma unroll
        for (int d = 0; d < VL; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k) acc[d] = mfma(__builtin_bit_cast(Frag<T>, __builtin_bit_cast(Raw, vw[2 * d + k])), w[k], acc[d]);
    }
    l = groups_sum(l);
    if (g == 0) {
        sm[wave][row] = m;
        sl[wave][row] = l;
    }
#pragma unroll
    for (int d = 0; d < VL; ++d) *(f32x4*)&so[wave][row][16 * d + 4 * g] = acc[d] * (any_weight(l) ? 1.0f / l : 0.0f) * (1.0f / low);
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * D; x += 64 * W) {
        const int y = x / D, d = x % D, ry = rt * 16 + y;
        if (ry >= rows) break;
        float top = sm[0][y];
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, sm[w][y]);
        float a[W], o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            a[w] = sl[w][y] * (sm[w][y] == -INFINITY ? 0.0f : exp2_(sm[w][y] - top));
            sum += a[w];
        }
        const float each = any_weight(sum) ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) o = __builtin_fmaf(so[w][y][d], a[w] * each, o);
        const Left z = part_of(y);
        if (!z.stats) {
            ((T*)p.out)[(((int64_t)b * p.T + ry / G) * p.H + hk * G + ry % G) * D + d] = (T)o;
        } else {
            if (d == 0) *z.stats = u32x2{__float_as_uint(top), __float_as_uint(sum)};
            z.sums[d] = o;
        }
    }
}

// One tile of rows and one share of its blocks a workgroup.  The tail has a workgroup of its own where there are several: in its 16 bits
// it takes as long as two of the others, behind which it would wait (33 requests of 8193 tokens: 32 us, 27 without its token).
template <class T, bool E4M3, int D, int W>
__global__ __launch_bounds__(64 * W) void k_cache_rows(D8sCacheAttnArgs p, int tiles, int split, float* part) {
    const D8sCache& c = p.c;
    const int cuts = split > 1 ? split + 1 : 1, G = p.H / c.HK;
    const Place place = place_of(tiles);
    const int rt = place.tile, cut = place.group % cuts, hk = place.group / cuts % c.HK, b = place.group / cuts / c.HK;
    const Rows a = rows_of(p, b, rt);
    const bool tail = a.tail() && (cut == split || split == 1);
    const int e0 = cut == split ? 0 : (int)((int64_t)a.coded * cut / split), e1 = cut == split ? 0 : (int)((int64_t)a.coded * (cut + 1) / split);
    const Part parts{part, cuts, (int64_t)c.B * p.T * p.H};
    rows_job<T, E4M3, D, W>(p, a, rt, hk, b, e0, e1, tail, [&](int y) {
        if (split == 1) return Left{nullptr, nullptr};
        const int64_t at = ((int64_t)b * p.T + (rt * 16 + y) / G) * p.H + hk * G + (rt * 16 + y) % G;
        return Left{parts.template stats<D>(cut, at), parts.template sums<D>(cut, at)};
    });
}

// Requests of different lengths, one tile of rows each: all their blocks in a row (a request's key heads after each other, a tail as TAIL
// blocks, a request without any as one) are cut into equal shares, one a workgroup, whose lengths the host cannot know.  A share may
// begin and end inside a key head: what it has of the first one is its part 0, of the last one part 1; key heads that lie in one share
// go straight to the output.
constexpr int TAIL = 2, EVEN_ROWS = NT;        // at most a request a thread
DEV int64_t cost_of(const Rows& a) { return max(1, a.coded + (a.tail() ? TAIL : 0)); }
// Shares of `all` blocks: at least one for each wave
DEV int64_t shares_of(int64_t all, int most) { return min((int64_t)most, max((int64_t)1, all / 4)); }
struct Even {
    int64_t* ends;                             // [B]: blocks of all requests up to this one
    float* part;                               // [shares][2][16][4 + D]: statistics and means
    template <int D>
    DEV Left at(int64_t share, int which, int y) const {
        float* z = part + ((share * 2 + which) * 16 + y) * (D + 4);
        return {(u32x2*)z, z + 4};
    }
};

template <class T, bool E4M3, int D>
__global__ __launch_bounds__(NT, 2) void k_cache_even(D8sCacheAttnArgs p, Even even) {
    const D8sCache& c = p.c;
    __shared__ int64_t ends[EVEN_ROWS], waves[NT / 64];
    const int tid = threadIdx.x;
    int64_t sum = tid < c.B ? cost_of(rows_of(p, tid, 0)) * c.HK : 0;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int64_t before = __shfl_up(sum, o);
        sum += tid % 64 >= o ? before : 0;
    }
    if (tid % 64 == 63) waves[tid / 64] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64 - 1; ++w) sum += w < tid / 64 ? waves[w] : 0;
    ends[tid] = sum;
    __syncthreads();
    if (blockIdx.x == 0 && tid < c.B) even.ends[tid] = sum;
    const int64_t all = ends[EVEN_ROWS - 1], shares = shares_of(all, gridDim.x), me = blockIdx.x;
    if (me >= shares) return;
    const int64_t u1 = all * (me + 1) / shares;
    int64_t u = all * me / shares;
    while (u < u1) {
        int b = 0;                             // the first request that ends behind u
        for (int step = EVEN_ROWS / 2; step >= 1; step /= 2)
            if (b + step <= c.B - 1 && ends[b + step - 1] <= u) b += step;
        b = __builtin_amdgcn_readfirstlane(b);
        const Rows a = rows_of(p, b, 0);
        const int64_t cost = cost_of(a), off = u - (b ? ends[b - 1] : 0);
        const int hk = __builtin_amdgcn_readfirstlane((int)(off / cost)), from = __builtin_amdgcn_readfirstlane((int)(off % cost));
        const int to = __builtin_amdgcn_readfirstlane((int)min(cost, from + (u1 - u)));
        const bool whole = from == 0 && to == cost;
        rows_job<T, E4M3, D, 4>(p, a, 0, hk, b, min(from, a.coded), min(to, a.coded), a.tail() && from <= a.coded && to > a.coded,
                                [&](int y) { return whole ? Left{nullptr, nullptr} : even.template at<D>(me, from == 0, y); });
        u += to - from;
        __syncthreads();                       // (the waves' sums have been read)
    }
}

// A row of a key head that lies in several shares, joined: four channels a thread, the shares over eight groups of threads
template <class T, int D>
__global__ __launch_bounds__(NT) void k_cache_even_join(D8sCacheAttnArgs p, Even even, int most) {
    constexpr int EACH = D / 4, K = NT / EACH;
    __shared__ f32x4 so[NT];
    __shared__ float ss[K], sm[K];
    const D8sCache& c = p.c;
    const int G = p.H / c.HK, rows = p.T * G, y = blockIdx.x % rows, hk = blockIdx.x / rows % c.HK, b = blockIdx.x / rows / c.HK;
    const int64_t all = even.ends[c.B - 1], shares = shares_of(all, most), before = b ? even.ends[b - 1] : 0;
    const int64_t cost = (even.ends[b] - before) / c.HK, from = before + hk * cost, to = from + cost;
    // share s holds blocks all s / shares .. all (s + 1) / shares - 1
    const int64_t s0 = ((from + 1) * shares - 1) / all, s1 = (to * shares - 1) / all;
    if (s0 == s1) return;
    const int d = threadIdx.x % EACH * 4, k = threadIdx.x / EACH;
    float top = -INFINITY, sum = 0.0f;
    f32x4 o = {};
    for (int64_t s = s0 + k; s <= s1; s += K) add_share(top, sum, *even.template at<D>(s, s == s0, y).stats);
    if (d == 0) {
        sm[k] = top;
        ss[k] = sum;
    }
    __syncthreads();
    const float each = sum_of<K>(sm, ss, top);
#pragma unroll 4
    for (int64_t s = s0 + k; s <= s1; s += K) {
        const Left z = even.template at<D>(s, s == s0, y);
        const float w = weight_of(*z.stats, top) * each;
        const f32x4 v = *(const f32x4*)(z.sums + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(v[e], w, o[e]);
    }
    so[threadIdx.x] = o;
    __syncthreads();
    if (k != 0) return;
#pragma unroll
    for (int x = 1; x < K; ++x) o += so[threadIdx.x + x * EACH];
    const float f[4] = {o[0], o[1], o[2], o[3]};
    store_n<T, 4>((T*)p.out + (((int64_t)b * p.T + y / G) * p.H + hk * G + y % G) * D + d, 4, f);
}

// ---- attention, many rows ------------------------------------------------------------------------------
// A workgroup runs 128 or 256 rows of a key head, 32 a wave, over the blocks they can see, on v_mfma_f32_32x32x16_f16.  Codes are made
// float16 once for all waves, on their way to LDS (two buffers; the next block's codes are in flight while one is computed).
// Lane l of a product's result holds row l % 32 (of queries) and the key rows r % 4 + 8 (r / 4) + 4 (l / 32) of its 16 registers
// r; a block's token lies in the key tile's row with bits 2 and 3 of its number exchanged, so that a lane's weights are those of 8
// neighbouring tokens at a time, as the transposed values have them.
// The scale of a block's values is in the exponent that its weights are formed from, relative to a reference that all sums are in units
// of: the weights are float16 numbers, so the reference follows the scales where they fall VSPAN times below it or rise above (the sums are then
// scaled).  It is one for all rows, also for those that do not see the block, so float32 keeps every row's sums only where the scales of the
// workgroup's blocks are within SPREAD of each other and below HIGH.  Where they are not (only bfloat16 values can be such), blocks are run one by
// one, their products formed by themselves and added times the scale, in units of 1, or, a row at a time, of 1 / LOWER, as with few rows.
// (2 x 256 queries over 8192 tokens of 8 key heads of 128: 89 us, and 91 where the scales are apart.  Looking at them first costs a bfloat16
// call a load and some shuffles: 8192 queries over themselves 566 -> 570, 4096 of 64 channels 105 -> 106.)
//
// Bound by its instructions: per 32 x 64 scores a wave issues 32 products of 32 cycles (D = 128) beside 218 vector instructions (32 of
// them its share of the codes' conversion, at 128 rows 64), and two waves a SIMD hardly overlap them: 2 x 256 queries of 32 heads over 22528
// tokens of 8 key heads 198 .. 206 us, 0.92 .. 0.95 PFLOP/s (a large library product 1.36), the matrix unit 0.45 busy, the vector unit 0.50, LDS
// 0.28, at 2.0 GHz.
// Tried, no better: crews of four waves a barrier apart, one at its products while the other forms weights (219 us: a lone wave's
// weights wait for themselves); reads of LDS six products ahead by scheduling groups (204); a barrier for two blocks (192 .. 200).
constexpr float VSPAN = 16.0f, SPREAD = 0x1p60f;
// A block that is full and followed by others, the block that is not full, and one whose scale is too far from the others'
enum Kind { CODED, RAW, APART };

typedef float f32x16 __attribute__((ext_vector_type(16)));
DEV f32x16 mfma(Frag<bf16> a, Frag<bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
DEV f32x16 mfma(Frag<f16> a, Frag<f16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Where piece c (16 bytes) of row r of a tile of W 16-bit values a row lies: c ^ swizzle<W>(r).  Reads of one piece of 32 rows and writes
// of whole rows then touch every bank once.
template <int W>
DEV int swizzle(int r) {
    static_assert(W == 64 || W == 128, "rows of 8 or 16 pieces");
    if constexpr (W == 64) return (r >> 1) & 7;            // two rows fill the banks once: it goes by pairs
    else return r & 15;
}
// The byte of piece `half` of the lane's row; with bits 5 .. flipped that of piece 2 k + half
template <int W>
DEV uint32_t piece_at(int r, int c) { return r * 2 * W + ((c ^ swizzle<W>(r)) << 4); }
DEV u32x4& at_byte(u32x4* tile, uint32_t at) { return *(u32x4*)((char*)tile + at); }
// Keeps the addresses derived from this one from being formed ahead of the loop and held in registers
DEV uint32_t fresh(uint32_t at) {
    asm volatile("" : "+v"(at));
    return at;
}
// Nothing but reads of LDS is moved over this by the compiler
DEV void fence() { __builtin_amdgcn_sched_barrier(0x100); }
// The key tile's row of a block's token, and back
DEV int key_row(int t) { return (t & 0x33) | (t & 4) << 1 | (t & 8) >> 1; }

// With more tiles than run at once: every group's last tile first, then those before it, and tiles behind a request's count at the end.
// Queries that see all before them see most in their last tile, and what is started last should be short (8192 queries over themselves, 32
// heads on 8: 561 us, 645 the other way).  An XCD runs the same groups all the time, for its L2, unless those could be of some requests
// only, whose lengths differ: then the requests go round, four tiles of neighbours at a time, which share most of what they see in a window
// (1024 queries each over 1024 .. 4096 tokens of one key head: 184 us, 228 without; 8 prompts of 30 .. 2048 tokens 53, and 79).
DEV Place late_first(const D8sCache& c, int tiles) {
    const int w = blockIdx.x, groups = gridDim.x / tiles, i = w / groups;
    return {i, c.B > 1 && c.HK % 8 ? (w + i / 4 % c.B * c.HK) % groups : w % groups};
}

template <class T, bool E4M3, int D, int W>
__global__ __launch_bounds__(64 * W, D == 128 ? 2 : W == 4 ? 3 : 4) void k_cache_tile(D8sCacheAttnArgs p, int tiles, int split, float* part) {
    constexpr int THREADS = 64 * W, ROWS = 32 * W, ND = D / 32, KS = D / 16, N = BLK * D / 8, PER = N / THREADS;       // pieces of a tile, and of a thread
    __shared__ u32x4 lk0[N], lk1[N], lv0[N], lv1[N];
    const D8sCache& c = p.c;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), half = lane / 32;
    const int G = p.H / c.HK, rows = p.T * G;
    const Place place = split == 1 ? late_first(c, tiles) : place_of(tiles);
    const int cut = place.group % split, hk = place.group / split % c.HK, b = place.group / split / c.HK;
    const int n = length_of(c, b), cnt = count_of(p.counts, b, p.T), nb = c.S / BLK;
    const int busy = (int)(((int64_t)cnt * G + ROWS - 1) / ROWS), rt = split == 1 && place.tile < busy ? busy - 1 - place.tile : place.tile;
    const int r0 = rt * ROWS + 32 * wave, r = r0 + lane % 32, t = min(r, rows - 1) / G, h = hk * G + min(r, rows - 1) % G;
    const int i = n - cnt + t;                 // the row's position
    const bool on = r < rows && t < cnt && i >= 0;
    const int64_t head = (int64_t)b * c.HK + hk;
    const uint16_t* qp = (const uint16_t*)p.q + b * p.q_sb + t * p.q_ss + h * p.q_sh;
    const int tlo = rt * ROWS / G, thi = min(min(rt * ROWS + ROWS - 1, rows - 1) / G, cnt - 1);
    const Blocks list = tlo < cnt ? blocks_of(p, n, n - cnt + tlo, n - cnt + thi) : Blocks{0, 0, 0};
    const int e0 = (int)((int64_t)list.count * cut / split), e1 = (int)((int64_t)list.count * (cut + 1) / split);
    // positions of the wave's first and last row: what all of them see, or none
    const int wlo = n - cnt + r0 / G, whi = n - cnt + min(min(r0 + 31, rows - 1) / G, cnt - 1);
    Frag<f16> q[KS];
    int down = 0;                              // the power of two that a bfloat16 row was multiplied by
    {
        Frag<T> x[KS];
#pragma unroll
        for (int k = 0; k < KS; ++k) x[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 16 * k + 8 * half));
        if constexpr (__is_same(T, bf16)) {
            float top = 0.0f, a, z;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int d = 0; d < 8; ++d) top = fmaxf(top, fabsf((float)x[k][d]));
            swap32(top, a, z);
            top = fmaxf(a, z);
            down = top > 0.0f && top < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int d = 0; d < 8; ++d) q[k][d] = (f16)ldexpf((float)x[k][d], down);
        } else {
#pragma unroll
            for (int k = 0; k < KS; ++k) q[k] = __builtin_bit_cast(Frag<f16>, x[k]);
        }
    }
    const float cs = p.scale * LOG2E;
    // the block that is not full is the last one, if it is among the share's
    const int full = n / BLK;
    const int coded = e1 > e0 && list.at(e1 - 1) >= full ? e1 - 1 : e1;
    constexpr bool WIDE = __is_same(T, bf16);
    bool apart = false;                        // the scales of the values are too far from each other
    if constexpr (WIDE) {
        float least = INFINITY, most = 0.0f;
        for (int e = e0 + lane; e < coded; e += 64) {
            const float vs = c.v_scale[head * nb + list.at(e)];
            least = vs > 0.0f ? fminf(least, vs) : least;
            most = fmaxf(most, vs);
        }
#pragma unroll
        for (int o = 8; o >= 1; o /= 2) least = fminf(least, __shfl_xor(least, o));
        float x, y;
        swap16(least, x, y);
        swap32(fminf(x, y), x, y);
        least = fminf(x, y);
        apart = __any(most > HIGH || most > least * SPREAD);
    }
    const auto job = [&](auto far) __attribute__((always_inline)) {
        constexpr bool FAR = decltype(far)::value;
        float m = -INFINITY, l = 0.0f, vref = FAR ? 1.0f : 0.0f, vinv = 0.0f, low = 1.0f;          // (sums are in units of vref / low, low a row's own)
        f32x16 acc[ND] = {};
        // the thread's pieces: piece x of the key tile is channels 8 (e % (D / 8)) of token e / (D / 8), of the value tile tokens
        // 8 (e % 8) of channel e / 8, with e = x * THREADS + threadIdx.x: 8 codes each, as they lie in memory
        u32x2 kr[PER], vr[PER];
        const auto load = [&](int j) __attribute__((always_inline)) {
            const u32x2* kc = (const u32x2*)((const uint8_t*)c.k_code + (head * nb + j) * BLK * D) + threadIdx.x;
            const u32x2* vc = (const u32x2*)((const uint8_t*)c.v_code + (head * nb + j) * BLK * D) + threadIdx.x;
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                kr[x] = kc[x * THREADS];
                vr[x] = vc[x * THREADS];
            }
        };
        // (a thread's pieces lie whole tiles of 16 or 32 rows apart, at one place of the swizzle)
        constexpr int STEP = THREADS * 16;
        const uint32_t kput = piece_at<D>(key_row(threadIdx.x / (D / 8)), threadIdx.x % (D / 8)), vput = piece_at<64>(threadIdx.x / 8, threadIdx.x % 8);
        const auto put1 = [&](u32x4* tile, uint32_t at, const u32x2* codes, int x) __attribute__((always_inline)) {
            at_byte(tile, at + x * STEP) = __builtin_bit_cast(u32x4, codes_frag<E4M3>(codes[x][0], codes[x][1]));
        };
        const auto put = [&](u32x4* tile, uint32_t at, const u32x2* codes) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < PER; ++x) put1(tile, at, codes, x);
        };
        // One block in LDS: scores times by, the values' scale vs; `high`: which tokens have values above 1 / LOWER.  Of CODED ones
        // the next block's codes go to nk and nv on the way, their conversions between the products, which leave most of the issue slots.
        // (Waves whose rows see nothing of a block run it all the same: a way round it cost copies of the sums in every block.)
        const auto turn = [&](auto kind, const auto& qf, u32x4* tk, u32x4* tv, u32x4* nk, u32x4* nv, int k0, float by, float vs,
                              uint64_t high) __attribute__((always_inline)) {
            constexpr Kind KIND = decltype(kind)::value;
            typedef std::conditional_t<KIND == RAW, T, f16> C;
            constexpr bool NEXT = KIND == CODED;
            const uint32_t ka = fresh(piece_at<D>(lane % 32, half)), va = fresh(piece_at<64>(lane % 32, half));
            f32x16 s[2];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    s[u] = mfma(__builtin_bit_cast(Frag<C>, at_byte(tk, (ka ^ (k << 5)) + u * 64 * D)), qf[k], k == 0 ? f32x16{} : s[u]);
                if constexpr (NEXT)
                    if (k % (KS / PER) == KS / PER - 1) {
                        fence();
                        put1(nk, kput, kr, k / (KS / PER));
                        fence();
                    }
            }
            by = by == 0.0f ? 0x1p-126f : by;      // (scores of a block of zeros are zeros; masked ones stay -infinity)
            // the reference of the values' scales (0 at first; a block of zeros needs none), 1 for blocks that need none of these
            float turned = 1.0f, ratio = 1.0f;
            if constexpr (KIND == CODED || !WIDE) {
                if ((vs > 0.0f) & ((vs > vref * 2.0f) | (vs * VSPAN < vref))) {
                    const float to = fmaxf(vs, 0x1p-126f);
                    turned = vref / to;
                    vref = to;
                    vinv = 1.0f / to;
                }
                ratio = vs == 0.0f ? 1.0f : vs * vinv;
            } else if (!FAR) {
                turned = vref;
                vref = 1.0f;
            }
            float lift = __builtin_amdgcn_logf(ratio) + NARROW_UP, weigh = __builtin_amdgcn_rcpf(ratio);
            uint64_t seen = on ? ~0ull : 0;        // tokens of the block that the row sees
            if (!(k0 + BLK <= n && k0 + BLK - 1 <= wlo + p.right && (k0 >= whi - p.left || k0 + BLK <= p.sinks))) {
                uint64_t vis = 0;
                if (on) vis = bits_below(min(i + p.right, n - 1) + 1 - k0) & (~bits_below(i - p.left - k0) | bits_below(p.sinks - k0));
                // (rows that see nothing of the block do not meet a scale of it that is not a number)
                by = vis ? by : 1.0f;
                lift = vis ? lift : 0.0f;
                weigh = vis ? weigh : 1.0f;
                seen = vis;
                const uint32_t mine[2] = {(uint32_t)(vis >> (8 * half)), (uint32_t)(vis >> (32 + 8 * half))};
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        // (register x of s[u] is token 32 u + 16 (x / 8) + 8 half + x % 8)
                        const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)mine[u], 16 * (x / 8) + x % 8, 1);
                        s[u][x] = __uint_as_float((__float_as_uint(s[u][x]) & keep) | (0xff800000u & ~keep));
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int x = 0; x < 16; ++x) top = fmaxf(top, s[u][x]);
            float t0, t1;
            swap32(top, t0, t1);
            top = fmaxf(t0, t1) * by;
            if constexpr (KIND != CODED && WIDE) {
                // (a row at a time: one that does not see such values may have ones that would not be left of it)
                const bool lower = (high & seen) && low == 1.0f;
                turned *= lower ? LOWER : 1.0f;
                low = lower ? LOWER : low;
                if (KIND == RAW) {                 // bfloat16 weights take the unit themselves
                    lift = low == 1.0f ? NARROW_UP : NARROW_UP - 64.0f;
                    weigh = 1.0f / low;
                }
            }
            if (__any((top > m + RISE) | (turned != 1.0f))) {
                const float up = fmaxf(m, top), a = up == -INFINITY ? 1.0f : exp2_(m - up);
                m = up;
                l *= a;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int x = 0; x < 16; ++x) acc[d][x] *= a * turned;
            }
            const float base = (m == -INFINITY ? 0.0f : m) - lift;
            float sum = 0.0f;
            const auto weight = [&](int u, int x) __attribute__((always_inline)) {
                s[u][x] = exp2_(__builtin_fmaf(s[u][x], by, -base));
            };
            const auto summed = [&](int u, int x) __attribute__((always_inline)) {
                float z[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) z[y] = s[u][x + y] + s[u][x + 4 + y];
                sum += (z[0] + z[1]) + (z[2] + z[3]);
            };
            const auto weights = [&](int k) __attribute__((always_inline)) {
                Frag<C> w;
#pragma unroll
                for (int x = 0; x < 8; ++x) w[x] = (C)s[k / 2][8 * (k % 2) + x];
                return w;
            };
            const auto values = [&](int k, int d) __attribute__((always_inline)) {
                return __builtin_bit_cast(Frag<C>, at_byte(tv, (va ^ (k << 5)) + d * 32 * 2 * BLK));
            };
            if constexpr (KIND == APART) {
                Frag<C> w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) weight(k / 2, 8 * (k % 2) + x);
                    summed(k / 2, 8 * (k % 2));
                    w[k] = weights(k);
                }
                const float scale = seen ? vs * low : 0.0f;    // (also one that is not a number)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    f32x16 o = {};
#pragma unroll
                    for (int k = 0; k < 4; ++k) o = mfma(values(k, d), w[k], o);
#pragma unroll
                    for (int x = 0; x < 16; ++x) acc[d][x] = __builtin_fmaf(o[x], scale, acc[d][x]);
                }
            } else {
#pragma unroll
                for (int x = 0; x < 8; ++x) weight(0, x);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    fence();
                    const Frag<C> w = weights(k);
#pragma unroll
                    for (int d = 0; d < ND; ++d) acc[d] = mfma(values(k, d), w, acc[d]);
                    fence();
                    summed(k / 2, 8 * (k % 2));
                    if (k < 3) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) weight((k + 1) / 2, 8 * ((k + 1) % 2) + x);
                    }
                    if constexpr (NEXT)
                        if (k % (4 / PER) == 4 / PER - 1) put1(nv, vput, vr, k / (4 / PER));
                }
            }
            l = __builtin_fmaf(sum, weigh, l);
        };
        const auto by_of = [&](int j) __attribute__((always_inline)) { return unit_of<T>(cs, c.k_scale[head * nb + j], down); };
        if constexpr (FAR) {
#pragma unroll 1
            for (int e = e0; e < coded; ++e) {
                const int j = list.at(e);
                const float vs = c.v_scale[head * nb + j];
                load(j);
                __syncthreads();                   // the tiles are no longer read
                put(lk0, kput, kr);
                put(lv0, vput, vr);
                __syncthreads();
                turn(std::integral_constant<Kind, APART>(), q, lk0, lv0, lk0, lv0, j * BLK, by_of(j), vs, vs > HIGH ? ~0ull : 0);
            }
        } else {
            if (e0 < coded) {
                load(list.at(e0));
                put(lk0, kput, kr);
                put(lv0, vput, vr);
                load(list.at(min(e0 + 1, coded - 1)));
            }
            const auto step = [&](int e, u32x4* tk, u32x4* tv, u32x4* nk, u32x4* nv) __attribute__((always_inline)) {
                const int j = list.at(e);
                __syncthreads();                   // the block is there, and the other one is no longer read
                turn(std::integral_constant<Kind, CODED>(), q, tk, tv, nk, nv, j * BLK, by_of(j), c.v_scale[head * nb + j], 0);
                load(list.at(min(e + 2, coded - 1)));          // (past the last block the same again, into the buffer that is not read)
            };
            for (int e = e0; e < coded; e += 2) {
                step(e, lk0, lv0, lk1, lv1);
                if (e + 1 < coded) step(e + 1, lk1, lv1, lk0, lv0);
            }
        }
        if (coded < e1) {                          // the tail, in its own type
            __syncthreads();
            uint32_t two[4] = {};                  // which of the thread's 8 tokens have high values
            const Raw* kt = (const Raw*)((const uint16_t*)c.k_tail + head * BLK * D);
            const Raw* vt = (const Raw*)((const uint16_t*)c.v_tail + head * BLK * D);
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int e = x * THREADS + threadIdx.x, there = n - full * BLK - 8 * (e % 8);     // of the piece's 8 tokens; the others are not used
                at_byte(lk0, kput + x * STEP) = __builtin_bit_cast(u32x4, kt[e]);
                Raw v = vt[e];
#pragma unroll
                for (int y = 0; y < 8; ++y) v[y] = y < there ? v[y] : 0;
                const u32x4 words = at_byte(lv0, vput + x * STEP) = __builtin_bit_cast(u32x4, v);
                if constexpr (__is_same(T, bf16))
#pragma unroll
                    for (int y = 0; y < 4; ++y) two[y] |= high_values(words[y]);
            }
            uint64_t high = 0;
            if constexpr (WIDE) {
                // (lanes l and l + 8 have the same tokens)
                uint32_t bits = high_bits(two);
#pragma unroll
                for (int o = 8; o < 64; o *= 2) bits |= (uint32_t)__shfl_xor((int)bits, o);
                if (lane < 8) ((uint8_t*)lk1)[8 * wave + lane] = (uint8_t)bits;        // (not read any more)
            }
            __syncthreads();
            if constexpr (WIDE)
#pragma unroll
                for (int x = 0; x < W; ++x) high |= ((const uint64_t*)lk1)[x];
            Frag<T> x[KS];
#pragma unroll
            for (int k = 0; k < KS; ++k) x[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 16 * k + 8 * half));
            turn(std::integral_constant<Kind, RAW>(), x, lk0, lv0, lk0, lv0, full * BLK, cs, 1.0f, high);
        }
        float l0, l1;
        swap32(l, l0, l1);
        l = l0 + l1;
        if (r >= rows) return;
        const int64_t at = ((int64_t)b * p.T + t) * p.H + h;
        const bool any = on && any_weight(l);
        const float each = 1.0f / l, unit = vref * (1.0f / low);
        if (split == 1) {
            T* o = (T*)p.out + at * D + 4 * half;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    float f[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) f[y] = any ? acc[d][x + y] * each * unit : 0.0f;
                    store_n<T, 4>(o + 32 * d + 2 * x, 4, f);
                }
        } else {
            const Part z{part, split, (int64_t)c.B * p.T * p.H};
            if (half == 0) *z.template stats<D>(cut, at) = u32x2{__float_as_uint(on ? m : -INFINITY), __float_as_uint(on ? l : 0.0f)};
            float* o = z.template sums<D>(cut, at) + 4 * half;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int x = 0; x < 16; x += 4) {
                    f32x4 f;
#pragma unroll
                    for (int y = 0; y < 4; ++y) f[y] = any ? acc[d][x + y] * each * unit : 0.0f;
                    *(f32x4*)(o + 32 * d + 2 * x) = f;
                }
        }
    };
    // (a loop of its own: a way between the two in one loop cost copies of the sums in every block)
    if (WIDE && apart) job(std::true_type());
    else job(std::false_type());
}

// A row's shares joined, four channels a thread.  With few rows K threads share its channels, each some of the shares.
template <class T, int D, int K>
__global__ __launch_bounds__(NT) void k_cache_join(Part part, T* out) {
    constexpr int EACH = D / 4, RW = NT / (EACH * K);                  // threads a share, rows a workgroup
    __shared__ f32x4 so[K > 1 ? NT : 1];
    __shared__ float ss[K > 1 ? RW * K : 1], sm[K > 1 ? RW * K : 1];
    const int d = threadIdx.x % EACH * 4, k = threadIdx.x / EACH % K, own = threadIdx.x / (EACH * K);
    const int64_t row = (int64_t)blockIdx.x * RW + own;
    const bool on = row < part.rows;
    float top = -INFINITY;
    f32x4 o = {};
    float sum = 0.0f;
    if (on)
        for (int s = k; s < part.cuts; s += K) add_share(top, sum, *part.template stats<D>(s, row));
    float each = any_weight(sum) ? 1.0f / sum : 0.0f;
    if constexpr (K > 1) {
        if (d == 0) {
            sm[own * K + k] = top;
            ss[own * K + k] = sum;
        }
        __syncthreads();
        each = sum_of<K>(sm + own * K, ss + own * K, top);
    }
    if (on) {
#pragma unroll 4
        for (int s = k; s < part.cuts; s += K) {
            const float a = weight_of(*part.template stats<D>(s, row), top) * each;
            const f32x4 z = *(const f32x4*)(part.template sums<D>(s, row) + d);
#pragma unroll
            for (int y = 0; y < 4; ++y) o[y] = __builtin_fmaf(z[y], a, o[y]);
        }
    }
    if constexpr (K > 1) {
        so[threadIdx.x] = o;
        __syncthreads();
        if (k != 0) return;
#pragma unroll
        for (int x = 1; x < K; ++x) o += so[threadIdx.x + x * EACH];
    }
    if (!on) return;
    const float f[4] = {o[0], o[1], o[2], o[3]};
    store_n<T, 4>(out + row * D + d, 4, f);
}

// How a call is run, by sizes that the host knows (lengths it does not); each side measured, in us:
// - 128 or 256 rows a workgroup where a key head has 64 and more, and all of them enough blocks: 256 queries of 8 heads over 22528
//   tokens 48 (16 rows a workgroup: 94); 32 rows a key head, 16 requests of 8000 tokens 80 (16 rows: 53, the memory's time); 1000
//   queries of 4 requests that see 200 tokens 20 (13).  256 rows halve what a row takes of the conversions (256 queries of 32 heads over
//   2 x 22528 tokens: 198, and 218 by 128), but a few blocks end in a longer last round (prompts of 2048 within 1024: 91, and 87).
// - Else 16 rows.  Where they see few blocks, one workgroup of many waves (SMALL) takes them all: one launch, for a caller whose host is the
//   limit (one token over 2048: 11.6 call by call, 16.0 in shares; in a graph 10.5 and 7.6), and no slower in a graph up to a
//   block a wave (500 tokens: 6.4 and 7.1).
// - One tile of rows a request and several requests: their blocks in equal shares (64 requests of 1 .. 16384 tokens 204, in one share a
//   key head 231; all of 8192 tokens 187, and 176), unless the window makes them alike anyway (33 requests, 8192 tokens seen of 22528:
//   28, and 23) or there are few blocks.
// - Else every tile's blocks in as many shares as fill the GPU once (33 x 8192 tokens of one key head: 18.6, twice 23, four times 25;
//   a few workgroups more than fit cost a round).
// Lengths far below the capacity are run as if they filled it: 81 tokens over 1458 10.6 in a cache of 1458 tokens, 12.1 in one of 22528; calls
// that the memory or the products bound take the same time in both (33 requests of 2048 tokens 17.4).
template <int D>
constexpr int SMALL = D == 64 ? 16 : 8;        // (registers for two or four waves a SIMD)
struct Plan {
    bool small, even;
    int rows, tiles, split;                    // rows of a workgroup
    int cuts() const { return split == 1 || rows > 16 ? split : split + 1; }     // workgroups a tile of rows, and parts to join
};
Plan plan_of(const D8sCacheAttnArgs* a) {
    const int64_t rows = (int64_t)a->T * (a->H / a->c.HK), heads = (int64_t)a->c.B * a->c.HK, cus = d8s_host_cu_count();
    const auto seen = [&](int64_t each) {      // about how many blocks a tile of so many rows sees in a full cache (one or two more where
                                               // its window and the first tokens do not begin and end with a block)
        const int64_t tokens = (each - 1) / (a->H / a->c.HK) + 1;
        const int64_t wide = std::min<int64_t>(a->c.S, (int64_t)a->left + a->right + std::min<int64_t>(a->T, tokens));
        return (std::min<int64_t>(a->c.S, wide + a->sinks) + BLK - 1) / BLK;
    };
    const bool tile = rows >= 64 && heads * ((rows + 15) / 16) * seen(16) > 12000;
    const int64_t each = !tile ? 16 : rows <= 128 || seen(128) < 32 ? 128 : 256, tiles = (rows + each - 1) / each, problems = heads * tiles, blocks = seen(each);
    const bool small = !tile && problems <= cus / 2 && blocks <= (a->c.D == 64 ? 3 * SMALL<64> : 2 * SMALL<128>);
    const bool joined = (int64_t)a->c.B * a->T * a->H < (1 << 24);           // (a workgroup a row: fewer than 2^32 threads)
    if (!tile && !small && tiles == 1 && a->c.B > 1 && a->c.B <= EVEN_ROWS && joined && blocks >= 16 && 4 * blocks > 3 * (a->c.S / BLK))
        return {false, true, 16, 1, (int)std::max<int64_t>(1, std::min(2 * cus, problems * blocks / 4))};
    const int64_t slots = each == 256 ? (a->c.D == 64 ? 2 * cus : cus) : 2 * cus;
    const int64_t split = small ? 1 : tile ? std::min(slots / problems, blocks / 8) : std::min(slots / problems - 1, blocks / 4);
    return {small, false, (int)each, (int)tiles, (int)std::max<int64_t>(1, split)};
}

uint64_t ends_bytes(const D8sCacheAttnArgs* a) { return ((uint64_t)a->c.B * 8 + 15) / 16 * 16; }

int cache_check(const D8sCache* c, const char* what) {
    CREQ(c->dtype == D8S_BF16 || c->dtype == D8S_F16, "dtype must be D8S_BF16 or D8S_F16");
    CREQ(c->codes == D8S_INT8 || c->codes == D8S_E4M3, "codes must be D8S_INT8 or D8S_E4M3");
    CREQ(c->D == 64 || c->D == 128, "D must be 64 or 128");
    CREQ(c->B >= 1 && c->S >= 1 && c->HK >= 1, "bad sizes");
    CREQ(c->S <= (1 << 29), "more than 2^29 tokens");
    CREQ((int64_t)c->B * c->HK < (1 << 22), "too many heads");
    CREQ(c->k_tail && c->v_tail && c->lengths, "null cache");
    CREQ(c->S < BLK || (c->k_code && c->v_code && c->k_scale && c->v_scale), "null cache");
    CREQ((((uintptr_t)c->k_code | (uintptr_t)c->v_code | (uintptr_t)c->k_tail | (uintptr_t)c->v_tail) & 15) == 0,
         "cache not 16-byte aligned");
    return 0;
}

template <class T, bool E4M3, int D>
void append_run(const D8sCacheAppendArgs& a, hipStream_t st) {
    const int chunks = (a.T + 2 * BLK - 2) / BLK;
    hipLaunchKernelGGL((k_cache_append<T, E4M3, D>), dim3((unsigned)((int64_t)a.c.B * a.c.HK * chunks)), dim3(NT), 0, st, a, chunks);
}
template <class T, bool E4M3, int D>
void read_run(const D8sCacheReadArgs& a, hipStream_t st) {
    const int blocks = (a.tokens + BLK - 1) / BLK;
    const int64_t all = (int64_t)a.c.B * a.c.HK * 2 * blocks;
    const dim3 grid((unsigned)std::min<int64_t>(all, READ_WGS), (unsigned)((all + READ_WGS - 1) / READ_WGS));
    if (a.out_dtype == D8S_F32) hipLaunchKernelGGL((k_cache_read<T, float, E4M3, D>), grid, dim3(NT), 0, st, a, blocks);
    else hipLaunchKernelGGL((k_cache_read<T, T, E4M3, D>), grid, dim3(NT), 0, st, a, blocks);
}
template <class T, bool E4M3, int D>
void attn_run(const D8sCacheAttnArgs& a, hipStream_t st) {
    const Plan x = plan_of(&a);
    if (x.even) {
        const Even even{(int64_t*)a.workspace, (float*)((char*)a.workspace + ends_bytes(&a))};
        hipLaunchKernelGGL((k_cache_even<T, E4M3, D>), dim3((unsigned)x.split), dim3(NT), 0, st, a, even);
        hipLaunchKernelGGL((k_cache_even_join<T, D>), dim3((unsigned)((int64_t)a.c.B * a.T * a.H)), dim3(NT), 0, st, a, even, x.split);
        return;
    }
    const int64_t all = (int64_t)a.c.B * a.T * a.H;
    const dim3 grid((unsigned)((int64_t)a.c.B * a.c.HK * x.tiles * x.cuts()));
    float* part = (float*)a.workspace;
    if (x.rows == 256) hipLaunchKernelGGL((k_cache_tile<T, E4M3, D, 8>), grid, dim3(512), 0, st, a, x.tiles, x.split, part);
    else if (x.rows == 128) hipLaunchKernelGGL((k_cache_tile<T, E4M3, D, 4>), grid, dim3(256), 0, st, a, x.tiles, x.split, part);
    else if (x.small) hipLaunchKernelGGL((k_cache_rows<T, E4M3, D, SMALL<D>>), grid, dim3(64 * SMALL<D>), 0, st, a, x.tiles, x.split, part);
    else hipLaunchKernelGGL((k_cache_rows<T, E4M3, D, 4>), grid, dim3(NT), 0, st, a, x.tiles, x.split, part);
    if (x.split == 1) return;
    const Part parts{part, x.cuts(), all};
    constexpr int K = 8, FEW = NT * 4 / (D * K), MANY = NT * 4 / D;              // rows a workgroup
    if (all < 4096) hipLaunchKernelGGL((k_cache_join<T, D, K>), dim3((unsigned)((all + FEW - 1) / FEW)), dim3(NT), 0, st, parts, (T*)a.out);
    else hipLaunchKernelGGL((k_cache_join<T, D, 1>), dim3((unsigned)((all + MANY - 1) / MANY)), dim3(NT), 0, st, parts, (T*)a.out);
}

#define BY_KIND(run, a, st)                                                                                            \
    do {                                                                                                               \
        const bool e = (a).c.codes == D8S_E4M3, d = (a).c.D == 64;                                                     \
        if ((a).c.dtype == D8S_BF16) {                                                                                 \
            if (e) d ? run<bf16, true, 64>((a), st) : run<bf16, true, 128>((a), st);                                   \
            else d ? run<bf16, false, 64>((a), st) : run<bf16, false, 128>((a), st);                                   \
        } else {                                                                                                       \
            if (e) d ? run<f16, true, 64>((a), st) : run<f16, true, 128>((a), st);                                     \
            else d ? run<f16, false, 64>((a), st) : run<f16, false, 128>((a), st);                                     \
        }                                                                                                              \
    } while (0)

int attn_check(const D8sCacheAttnArgs* a, const char* what) {
    CREQ(a != nullptr, "null arguments");
    if (int rc = cache_check(&a->c, what)) return rc;
    CREQ(a->T >= 1 && a->T <= (1 << 29) && a->H >= 1 && a->H % a->c.HK == 0, "bad sizes (H a multiple of HK)");
    CREQ((int64_t)a->T * a->H <= (1 << 30) && (int64_t)a->c.B * a->T * a->H < (1 << 27), "too many heads and tokens");
    CREQ(a->left >= 0 && a->right >= 0 && a->sinks >= 0, "left, right and sinks must not be negative");
    CREQ(a->scale >= 0x1p-100f && a->scale <= 0x1p100f, "scale must be 2^-100 .. 2^100");
    return 0;
}

// The arguments with a window no wider than the cache (the kernel adds its sides to positions)
D8sCacheAttnArgs clipped(const D8sCacheAttnArgs* a) {
    D8sCacheAttnArgs c = *a;
    c.left = std::min(a->left, a->c.S);
    c.right = std::min(a->right, a->c.S);
    c.sinks = std::min(a->sinks, a->c.S);
    return c;
}

}  // namespace

extern "C" int d8s_cache_append(const D8sCacheAppendArgs* a, void* stream) {
    const char* what = "d8s_cache_append";
    CREQ(a != nullptr, "null arguments");
    if (int rc = cache_check(&a->c, what)) return rc;
    CREQ(a->T >= 1 && a->T <= (1 << 29), "bad number of tokens");
    CREQ((int64_t)a->c.B * a->c.HK * ((a->T + 2 * BLK - 2) / BLK) < (1 << 24), "too many heads and tokens");
    CREQ(a->k && a->v && a->arrived && a->dropped, "null pointer");
    BY_KIND(append_run, *a, (hipStream_t)stream);
    return d8s_host_launched(what);
}

extern "C" int d8s_cache_read(const D8sCacheReadArgs* a, void* stream) {
    const char* what = "d8s_cache_read";
    CREQ(a != nullptr, "null arguments");
    if (int rc = cache_check(&a->c, what)) return rc;
    CREQ(a->tokens >= 1 && a->tokens <= a->c.S, "tokens must be 1 .. S");
    CREQ(a->out_dtype == D8S_F32 || a->out_dtype == a->c.dtype, "out_dtype must be D8S_F32 or dtype");
    CREQ((int64_t)a->c.B * a->c.HK * 2 * ((a->tokens + BLK - 1) / BLK) < (1ll << 31) - READ_WGS, "too many heads and tokens");
    CREQ(a->k && a->v, "null pointer");
    BY_KIND(read_run, *a, (hipStream_t)stream);
    return d8s_host_launched(what);
}

extern "C" int d8s_cache_attention_workspace(const D8sCacheAttnArgs* a, uint64_t* bytes) {
    const char* what = "d8s_cache_attention_workspace";
    if (int rc = attn_check(a, what)) return rc;
    CREQ(bytes != nullptr, "null arguments");
    const Plan x = plan_of(a);
    if (x.even) {
        *bytes = ends_bytes(a) + (uint64_t)x.split * 2 * 16 * (a->c.D + 4) * 4;
        return 0;
    }
    const int cuts = x.cuts();
    const uint64_t parts = (uint64_t)cuts * a->c.B * a->T * a->H;
    *bytes = cuts > 1 ? parts * (a->c.D + 2) * 4 + parts % 2 * 8 : 0;
    return 0;
}

extern "C" int d8s_cache_attention(const D8sCacheAttnArgs* a, void* stream) {
    const char* what = "d8s_cache_attention";
    if (int rc = attn_check(a, what)) return rc;
    CREQ(a->q && a->out, "null pointer");
    uint64_t need = 0;
    if (int rc = d8s_cache_attention_workspace(a, &need)) return rc;
    CREQ(need == 0 || (a->workspace && a->ws_bytes >= need && ((uintptr_t)a->workspace & 15) == 0),
         "workspace smaller than d8s_cache_attention_workspace() or not 16-byte aligned");
    const D8sCacheAttnArgs c = clipped(a);
    BY_KIND(attn_run, c, (hipStream_t)stream);
    return d8s_host_launched(what);
}
