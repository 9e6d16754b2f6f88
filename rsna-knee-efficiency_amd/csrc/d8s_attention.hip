// gfx950 kernels of attention within a window of neighbouring tokens and a few first tokens that stay visible, for a
// context layer over all the tokens of a study: forward, backward, and one new token against a cache; the C ABI is in
// include/d8s_hip.h.
//
// Key j is visible to query i iff j <= i + right, (j >= i - left or j < sinks) and mask[j].  With s = scale q k,
//   P = softmax over the visible keys (nothing visible: zeros),  o = P v,  lse = log sum exp s (-inf);
//   dv = P^T do,  dP = do v^T,  dS = P (dP - rowsum(do o)),  dq = scale dS k,  dk = scale dS^T q.
//
// The products run on v_mfma_f32_32x32x16 (bf16 or f16, float32 sums), arranged so that what comes out of one product
// goes into the next from the registers it is in: lane l of a 32 x 32 result holds column l % 32 and the rows
// r % 4 + 8 (r / 4) + 4 (l / 32) of its 16 registers r, and an operand's lane holds row (or column) l % 32 and eight of
// the 16 values that are summed over.  Which eight is free as long as both operands agree, so the eight registers
// 8 s .. 8 s + 7 of a result are an operand as they are, and the other one is read with
// the same order: rows 16 s + 4 (l / 32) + (0 .. 3) and 8 more, by ds_read_b64_tr_b16, which hands each lane a column
// of a row-major tile.  So nothing is transposed or exchanged between lanes.
// Tiles of rows lie in LDS in 16-byte pieces, piece c of row r at c ^ swizzle(r): both ways of reading them (16
// lanes at one piece of 16 rows; 32 lanes at 4 neighbouring pieces of 4 rows) then touch every bank once.
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

#define AREQ(cond, msg) \
    do { if (!(cond)) return d8s_host_fail((int)hipErrorInvalidValue, std::string(what) + ": " + (msg)); } while (0)

constexpr int NT = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <class T>
using Frag = T __attribute__((ext_vector_type(8)));
template <class T>
constexpr bool NARROW = false;                 // whether P and dS have to be brought into T's range
template <>
constexpr bool NARROW<f16> = true;
typedef Vec<uint16_t, 8> Raw;                  // 8 elements as they lie in memory

DEV f32x16 mfma(Frag<bf16> a, Frag<bf16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
DEV f32x16 mfma(Frag<f16> a, Frag<f16> b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Where piece c (16 bytes) of row r of a tile lies: c ^ swizzle<D>(r).  The swizzle repeats every 16 rows.
template <int D>
DEV int swizzle(int r) {
    static_assert(D == 64 || D == 128, "rows of 8 or 16 pieces");
    if constexpr (D == 64) {
        const int k = (r >> 1) & 7;            // two rows fill the banks once: it goes by pairs
        return (k & 1) << 2 | (k & 2) | k >> 2;
    } else {
        return (r & 3) << 2 | (r >> 2 & 3);
    }
}

// Every address of a tile's operands is the lane's first one with some bits flipped (the piece) and a constant added
// (the rows), so two registers serve all of them.
// A tile's two buffers are shared arrays of their own, and a loop's turn names them: so the compiler sees that reads of
// one do not wait for the copies into the other (through one array, or addresses as numbers, it waits for every copy
// in flight before the first read: the copies of the next tile would be waited for at once).
// The lane's first address for rows_frag, and for cols_frag, relative to a tile
template <int D>
DEV uint32_t rows_at(int lane) {
    const int r = lane % 32;
    return r * 2 * D + ((lane / 32 ^ swizzle<D>(r)) << 4);
}
template <int D>
DEV uint32_t cols_at(int lane) {
    const int i = lane % 16, r = 4 * (lane / 32) + i / 4, c = 2 * (lane / 16 & 1) + (i % 4) / 2;
    return r * 2 * D + ((c ^ swizzle<D>(r)) << 4) + 8 * (i & 1);
}
// Keeps the addresses derived from this one from being formed ahead of the loop and held in registers
DEV uint32_t fresh(uint32_t at) {
    asm volatile("" : "+v"(at));
    return at;
}

// Operand of rows r0 .. r0 + 31 (r0 a multiple of 16), values 16 k .. 16 k + 15 of each
template <class T, int D>
DEV Frag<T> rows_frag(const u32x4* tile, uint32_t at, int r0, int k) {
    return __builtin_bit_cast(Frag<T>, *(const u32x4*)((const char*)tile + ((at ^ (uint32_t)(k << 5)) + r0 * 2 * D)));
}

// Operand of columns 32 d .. 32 d + 31, summed over the tile's rows r0 .. r0 + 15 in the order of a result's registers
template <class T, int D>
DEV Frag<T> cols_frag(const u32x4* tile, uint32_t at, int r0, int d) {
    typedef __attribute__((address_space(3))) s16x4* lds;
    const uint32_t lo = at ^ (uint32_t)(d << 6), hi = lo ^ (D == 64 ? 16u : 32u);    // (8 rows on, the swizzle differs in one bit)
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)((const char*)tile + (lo + r0 * 2 * D)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)((const char*)tile + (hi + (r0 + 8) * 2 * D)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<T>, v);
}

// Registers 8 s .. of a result as the next product's operand.  P and dS are rounded to T here because the matrix unit's
// full rate takes 16-bit operands (float32 ones a sixteenth of it): at most 2^-8 (bf16) or 2^-11 (f16, above 2^-14) of
// each value, independent from value to value, about what the results' own rounding to T adds; P's sum and the
// statistics stay float32.  The gradients bring P and dS into the range where that holds for f16 (see backward).
template <class T>
DEV Frag<T> round_frag(const f32x16& x, int s) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)x[8 * s + j];
    return f;
}

// Consecutive problems on one XCD's L2: workgroup w runs problem (w % 8) (n / 8) + w / 8 (as far as 8 divides n)
DEV int xcd_order(int w, int n) {
    const int per = n / 8;
    return w < 8 * per ? (w % 8) * per + w / 8 : w;
}

// The tiles of 64 keys a run of queries i0 .. i1 can see: the first tokens' ones, then the window's
constexpr int TILE = 64;
struct Tiles {
    int first, start, count;
    DEV int at(int i) const { return i < first ? i : start + i - first; }
};
DEV Tiles tiles_of(const D8sAttnArgs& p, int i0, int i1) {
    const int lo = max(0, i0 - p.left) / TILE, hi = min(p.S - 1, i1 + p.right) / TILE;
    const int first = min((p.sinks + TILE - 1) / TILE, lo);
    return {first, lo, first + hi - lo + 1};
}

// Whether queries i0 .. i0 + 31 see none, or all, of keys k0 .. k1 (left, right and sinks are at most S, and S at
// most 2^29: no sum of them overflows)
DEV bool none_seen(const D8sAttnArgs& p, int i0, int k0, int k1) {
    return k0 > i0 + 31 + p.right || (k1 < i0 - p.left && k0 >= p.sinks);
}
DEV bool all_seen(const D8sAttnArgs& p, int i0, int k0, int k1) {
    return k1 <= i0 + p.right && (k0 >= i0 + 31 - p.left || k1 < p.sinks);
}

// Bits 0 .. 63 below n, or from n on (any n)
DEV uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : ~(~0ull << n); }
DEV uint64_t bits_from(int n) { return ~bits_below(n); }

// What a lane keeps of its 16 registers of a 32 x 32 result whose row r is kept iff bit r of `rows` is set: the bits
// moved so that register r's is at r % 4 + 8 (r / 4)
DEV uint32_t lane_rows(uint32_t rows, int lane) { return rows >> (4 * (lane / 32)); }
DEV uint32_t keep_mask(uint32_t lane_bits, int r) {       // all ones where register r is kept (one v_bfe_i32)
    return (uint32_t)__builtin_amdgcn_sbfe((int)lane_bits, r % 4 + 8 * (r / 4), 1);
}

// Copies a tile of ROWS rows of a matrix (rows `stride` elements apart, those past `last` replaced by it) to LDS
// without registers: each lane of a wave's copy brings the 16 bytes that belong at its place of the swizzled tile.
template <int D, int ROWS>
struct Copy {
    static constexpr int P = D / 8, N = ROWS * P / NT, STEP = NT / P;   // rows between a thread's pieces
    int row, col;                              // of the thread's first piece
    DEV Copy() {
        row = threadIdx.x / P;
        col = 8 * (threadIdx.x % P ^ swizzle<D>(row));
        static_assert(STEP % 16 == 0, "the same swizzle for all of a thread's pieces");
    }
    DEV void operator()(const uint16_t* p, int64_t stride, int r0, int last, u32x4* tile, int wave) const {
        typedef const __attribute__((address_space(1))) void* global;
        typedef __attribute__((address_space(3))) void* lds;
        if (r0 + ROWS - 1 <= last) {
            const uint16_t* q = p + r0 * stride + (row * stride + col);
#pragma unroll
            for (int n = 0; n < N; ++n)
                __builtin_amdgcn_global_load_lds((global)(q + n * STEP * stride), (lds)(tile + n * NT + wave * 64), 16, 0, 0);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n)
                __builtin_amdgcn_global_load_lds((global)(p + min(r0 + row + n * STEP, last) * stride + col),
                                                 (lds)(tile + n * NT + wave * 64), 16, 0, 0);
        }
    }
    // zeros in the thread's own pieces of rows whose bit is not set (its copies have arrived)
    DEV void clear(u32x4* tile, uint64_t rows) const {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (!(rows >> (row + n * STEP) & 1)) tile[n * NT + threadIdx.x] = u32x4{0, 0, 0, 0};
    }
};
// The same for a loop that seldom needs it: nothing of it is held in registers from turn to turn
template <int D>
DEV void clear_rows(u32x4* a, u32x4* b, uint64_t rows) {
    int at = threadIdx.x;
    asm volatile("" : "+v"(at));
#pragma unroll 1
    for (; at < TILE * D / 8; at += NT)
        if (!(rows >> (at / (D / 8)) & 1)) a[at] = b[at] = u32x4{0, 0, 0, 0};
}
DEV void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Which of the tile's keys exist and are not masked, from the byte a lane read for its key
struct KeyBits {
    const uint8_t* mask;
    int S;
    uint32_t byte;
    DEV void load(int k0, int lane) { byte = mask ? mask[min(k0 + lane, S - 1)] : 1; }
    DEV uint64_t bits(int k0) {
        const uint64_t in = bits_below(S - k0);
        asm volatile("" : "+v"(byte));         // (compared here and not at the load, which would wait for it there)
        return mask ? __ballot(byte != 0) & in : in;
    }
};

// Rows of results held by lane columns (column l % 32, rows as in lane_rows): values 32 d + ... of row `o`, scaled,
// rounded, and joined between the wave's halves into 16-byte stores.
template <class T, int ND>
DEV void store_rows(T* o, const f32x16* acc, float scale, bool on, int lane) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
            typedef T half4 __attribute__((ext_vector_type(4)));
            u32x2 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                half4 h;
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = (T)(acc[d][4 * (g + k) + j] * scale);
                w[k] = __builtin_bit_cast(u32x2, h);
            }
            const u32x2 a = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            const u32x2 b = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            // lower lanes: values 8 g .. 8 g + 7; upper lanes: the eight after them
            const Vec<uint32_t, 4> v = {a[0], b[0], a[1], b[1]};
            typedef Vec<uint16_t, 8> out8;
            if (on) *(out8*)(o + 32 * d + 8 * (g + lane / 32)) = __builtin_bit_cast(out8, v);
        }
}

// Whether anything is seen, by the sum of the weights: not where it is zero (no key, or every score is -infinity); a sum that
// is not a number stays one
DEV bool any_weight(float sum) { return sum > 0.0f || sum != sum; }

// ---- forward --------------------------------------------------------------------------------------
// Bound by its instructions: a wave's tile of 32 x 64 scores is 162 vector operations (32 exponentials among them) beside 16
// (D = 64) or 32 (D = 128) products of 32 cycles, and the two overlap only between waves.  Measured: 22528 tokens of 4
// heads of 64, 1024 neighbours each, two keys in eight masked, 38 us (0.47 PFLOP/s; 32 heads without a mask 0.68); 2 x 8199
// tokens of 16 heads of 128, 1024 before each, 182 us (0.72 PFLOP/s).  (In a long row of passes: after a pause the card's
// clock is lower, 47 us for the first.)  Tiles of 32 keys and more waves: 49 and 216 us where these were 43 and 185.
//
// A workgroup runs 128 queries of a head, 32 a wave, over the tiles of 64 keys they can see; keys and values go
// through two LDS buffers, the next tile's copies in flight while one is computed.  A wave forms s transposed (keys x
// queries), so a query's statistics are one value a lane, and P goes from registers into the second product.
// The running maximum m is raised, and the sums scaled, only where a tile exceeds it by more than 2^RISE (P stays below
// 2^RISE, harmless in float32 and in both types), which after a row's first tiles is rare.
// float16 holds nothing below 2^-25 and little below 2^-14, and P next to one key that outweighs each of many others is
// that small: it is formed times 2^NARROW_UP (in its exponent, so at no cost), which leaves the sums' quotient as it is.
constexpr float RISE = 6.0f, NARROW_UP = 8.0f;

template <class T, int D>
__global__ __launch_bounds__(NT, (D == 64 ? 3 : 2)) void k_attn(D8sAttnArgs p) {
    constexpr int ND = D / 32;
    constexpr int N = TILE * D / 8;
    __shared__ u32x4 lk0[N], lk1[N], lv0[N], lv1[N];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int nq = (p.S + 127) / 128, id = xcd_order(blockIdx.x, gridDim.x);
    const int b = id / (nq * p.H), h = id / nq % p.H, i00 = id % nq * 128, i0 = i00 + 32 * wave;
    const int hk = h / (p.H / p.HK);
    const uint16_t* kp = (const uint16_t*)p.k + b * p.k_sb + hk * p.k_sh;
    const uint16_t* vp = (const uint16_t*)p.v + b * p.v_sb + hk * p.v_sh;
    const int i = i0 + lane % 32;
    Frag<T> q[D / 16];
    {
        const uint16_t* qp = (const uint16_t*)p.q + b * p.q_sb + h * p.q_sh + (int64_t)min(i, p.S - 1) * p.q_ss;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
            q[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 16 * k + 8 * (lane / 32)));
    }
    const float c = p.scale * LOG2E;
    float m = -INFINITY, l = 0.0f;
    f32x16 acc[ND] = {};
    const Tiles tiles = tiles_of(p, i00, min(i00 + 127, p.S - 1));
    const Copy<D, TILE> copy;
    KeyBits keys{p.mask ? p.mask + b * p.mask_sb : nullptr, p.S, 1};
    int k0 = tiles.at(0) * TILE;
    copy(kp, p.k_ss, k0, p.S - 1, lk0, wave);
    copy(vp, p.v_ss, k0, p.S - 1, lv0, wave);
    keys.load(k0, lane);
    // tile t from tk and tv, the next one's copies into nk and nv
    const auto turn = [&](int t, u32x4* tk, u32x4* tv, u32x4* nk, u32x4* nv) __attribute__((always_inline)) {
        arrived();
        const uint64_t bits = keys.bits(k0);
        if (bits != ~0ull) {                   // whatever memory holds of a masked key is not used
            copy.clear(tk, bits);
            copy.clear(tv, bits);
        }
        __syncthreads();                       // the tile is there, and the other one is no longer read
        const int now = k0;
        if (t + 1 < tiles.count) {
            k0 = tiles.at(t + 1) * TILE;
            copy(kp, p.k_ss, k0, p.S - 1, nk, wave);
            copy(vp, p.v_ss, k0, p.S - 1, nv, wave);
            keys.load(k0, lane);
        }
        if (bits == 0 || i0 >= p.S || none_seen(p, i0, now, now + TILE - 1)) return;
        const uint32_t ra = fresh(rows_at<D>(lane)), ca = fresh(cols_at<D>(lane));
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = mfma(rows_frag<T, D>(tk, ra, 32 * u, 0), q[0], f32x16{});
#pragma unroll
            for (int k = 1; k < D / 16; ++k) s[u] = mfma(rows_frag<T, D>(tk, ra, 32 * u, k), q[k], s[u]);
        }
        Frag<T> early[ND];                     // the first values, read while the exponentials are formed
#pragma unroll
        for (int d = 0; d < ND; ++d) early[d] = cols_frag<T, D>(tv, ca, 0, d);
        if (bits != ~0ull || !all_seen(p, i0, now, now + TILE - 1)) {
            const uint64_t vis = bits & bits_below(i + p.right + 1 - now) & (bits_from(i - p.left - now) | bits_below(p.sinks - now));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if ((uint32_t)(bits >> (32 * u)) == ~0u && all_seen(p, i0, now + 32 * u, now + 32 * u + 31)) continue;
                const uint32_t mine = lane_rows((uint32_t)(vis >> (32 * u)), lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t keep = keep_mask(mine, r);
                    s[u][r] = __uint_as_float((__float_as_uint(s[u][r]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
        float t0, t1;
        swap32(top, t0, t1);
        top = fmaxf(t0, t1);
        if (__any(top * c > m * c + RISE)) {
            const float up = fmaxf(m, top), a = up == -INFINITY ? 1.0f : exp2_((m - up) * c);
            m = up;
            l *= a;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= a;
        }
        const float mc = (m == -INFINITY ? 0.0f : m * c) - (NARROW<T> ? NARROW_UP : 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[u][r] = exp2_(__builtin_fmaf(s[u][r], c, -mc));
                sum += s[u][r];
            }
        l += sum;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const Frag<T> w = round_frag<T>(s[u / 2], u % 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] = mfma(u == 0 ? early[d] : cols_frag<T, D>(tv, ca, 16 * u, d), w, acc[d]);
        }
    };
    for (int t = 0; t < tiles.count; t += 2) {
        turn(t, lk0, lv0, lk1, lv1);
        if (t + 1 < tiles.count) turn(t + 1, lk1, lv1, lk0, lv0);
    }
    float l0, l1;
    swap32(l, l0, l1);
    l = l0 + l1;
    const bool any = any_weight(l);
    if (p.lse && lane < 32 && i < p.S) p.lse[((int64_t)b * p.H + h) * p.S + i] = any ? (m * c + (log2f(l) - (NARROW<T> ? NARROW_UP : 0.0f))) * LN2 : -INFINITY;
    store_rows<T, ND>((T*)p.out + (((int64_t)b * p.S + i) * p.H + h) * D, acc, any ? 1.0f / l : 0.0f, i < p.S, lane);
}

// ---- backward ----------------------------------------------------------------------------------------
// float16 holds values of 2^-14 .. 2^16 in full, and dS = P (dP - rowsum(do o)) is a share of 1 / (keys seen) of a
// gradient that may itself be small, or multiplied by a large loss scale.  So there dS is formed times a power of two,
// which the results are divided by (exact): |dP - rowsum| <= |do||v| + |rowsum|, so from the largest |do| and |rowsum| of
// the queries that a workgroup runs over (dk; of a lane's own query for dq) and the largest |v| of the keys follows a power
// that keeps |dS| below 2^15 (P is 1 at most, 2 with its rounding), and nothing above 2^-28 of that bound is
// held in fewer bits.  It is in the exponent that P is formed from (for dk partly in v), so a tile costs no operation
// more: 2 x 8199 tokens of 16 heads of 128, 541 us with it and 535 without.  bfloat16 has float32's range and needs none.
// The largest norms of every tile of 64 queries and of 64 keys are left by k_attn_delta; queries that see nothing, keys
// that are masked and rows that are not finite are left out of them, so that they do not cost the others their bits.
//
// k_attn_delta leaves rowsum(do o) of every query.  One launch then runs both kinds of workgroups beside each other:
// first those of the keys (dk and dv, the longer ones), then those of the queries (dq), which fill the compute units
// that the keys leave; what either writes the other does not read.  Both form s and dP: two products of seven more
// than sums shared through atomics would take, for results that do not depend on an order.
// Bound as the forward pass, with the matrix unit busy 0.44 of the time: 2 x 8199 tokens of 16 heads of 128 (4 key heads),
// 1024 before each, in 507 .. 539 us from card to card, float16 (0.6 PFLOP/s with the products formed twice; two launches
// after each other took 700).
// Of each tile of 64 rows: the largest |do| and |rowsum(do o)| [B][H][tiles], the largest |v| [B][HK][tiles]
struct Tops {
    float *g, *r, *v;
};
DEV float wave_max(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o /= 2) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
// The power of two (its exponent) that brings values of at most `bound` below 2^14
DEV int shift_of(float bound) {
    return bound > 0.0f && bound < INFINITY ? min(max(14 - __builtin_amdgcn_frexp_expf(bound), -64), 64) : 0;
}
// A value that is the same in all lanes, in a scalar register
DEV float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }
DEV float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The sum of squares of a row whose other half is held by the lane 32 away
template <class T, int N>
DEV float row_square(const Frag<T>* f) {
    float x = 0.0f, a, b;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) x = __builtin_fmaf((float)f[k][j], (float)f[k][j], x);
    swap32(x, a, b);
    return a + b;
}

template <class T, int D>
__global__ __launch_bounds__(NT) void k_attn_delta(D8sAttnArgs p, float* delta, Tops tops) {
    constexpr int L = D / 8, ROWS = NT / L;    // lanes a row, rows at a time
    constexpr int TURNS = NARROW<T> ? TILE / ROWS : 1;
    const int run_rows = ROWS * TURNS, runs = (p.S + run_rows - 1) / run_rows, of_queries = p.B * p.H * runs;
    const bool keys = NARROW<T> && (int)blockIdx.x >= of_queries;
    const int id = keys ? blockIdx.x - of_queries : blockIdx.x, heads = keys ? p.HK : p.H;
    const int run = id % runs, h = id / runs % heads, b = id / runs / heads, d = threadIdx.x % L * 8;
    float first = 0.0f, second = 0.0f;         // the largest squares; rowsums
#pragma unroll
    for (int n = 0; n < TURNS; ++n) {
        const int i = run * run_rows + n * ROWS + threadIdx.x / L;
        const int64_t ic = min(i, p.S - 1);
        if (NARROW<T> && keys) {
            float v[8], x = 0.0f;
            load_n<T, 8>((const T*)p.v + b * p.v_sb + h * p.v_sh + ic * p.v_ss + d, 8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) x = __builtin_fmaf(v[k], v[k], x);
            x = lanes_sum<L>(x);
            const bool on = p.mask == nullptr || p.mask[b * p.mask_sb + ic] != 0;
            first = fmaxf(first, on && x < INFINITY ? x : 0.0f);
            continue;
        }
        float g[8], o[8], x = 0.0f, y = 0.0f;
        load_n<T, 8>((const T*)p.dout + b * p.do_sb + h * p.do_sh + ic * p.do_ss + d, 8, g);
        load_n<T, 8>((const T*)p.out + (((int64_t)b * p.S + ic) * p.H + h) * D + d, 8, o);
#pragma unroll
        for (int k = 0; k < 8; ++k) x = __builtin_fmaf(g[k], o[k], x);
        x = lanes_sum<L>(x);
        const int64_t at = ((int64_t)b * p.H + h) * p.S;
        if (d == 0 && i < p.S) delta[at + i] = x;
        if constexpr (NARROW<T>) {
#pragma unroll
            for (int k = 0; k < 8; ++k) y = __builtin_fmaf(g[k], g[k], y);
            y = lanes_sum<L>(y);
            const bool on = p.lse[at + ic] != -INFINITY && y < INFINITY && fabsf(x) < INFINITY;
            first = fmaxf(first, on ? y : 0.0f);
            second = fmaxf(second, on ? fabsf(x) : 0.0f);
        }
    }
    if constexpr (NARROW<T>) {
        __shared__ float red[2][NT / 64];
        first = wave_max(first);
        second = wave_max(second);
        if (threadIdx.x % 64 == 0) {
            red[0][threadIdx.x / 64] = first;
            red[1][threadIdx.x / 64] = second;
        }
        __syncthreads();
        if (threadIdx.x != 0) return;
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) {
            first = fmaxf(first, red[0][w]);
            second = fmaxf(second, red[1][w]);
        }
        (keys ? tops.v : tops.g)[id] = sqrtf(first);
        if (!keys) tops.r[id] = second;
    }
}

// Queries: as the forward pass, with do beside q: P from lse, dP = do v^T transposed, dS, dq += dS k.
DEV float lse2_of(float lse) { return lse == -INFINITY ? INFINITY : lse * LOG2E; }   // (empty row: every P is 0)

template <class T, int D>
DEV void dq_body(const D8sAttnArgs& p, const float* delta, const Tops& tops, int id, u32x4* lk0, u32x4* lk1, u32x4* lv0, u32x4* lv1) {
    constexpr int ND = D / 32;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int nq = (p.S + 127) / 128;
    const int b = id / (nq * p.H), h = id / nq % p.H, i00 = id % nq * 128, i0 = i00 + 32 * wave;
    const int hk = h / (p.H / p.HK);
    const uint16_t* kp = (const uint16_t*)p.k + b * p.k_sb + hk * p.k_sh;
    const uint16_t* vp = (const uint16_t*)p.v + b * p.v_sb + hk * p.v_sh;
    const int i = i0 + lane % 32;
    const int64_t ic = min(i, p.S - 1);
    Frag<T> q[D / 16], g[D / 16];
    {
        const int64_t at = 8 * (lane / 32);
        const uint16_t* qp = (const uint16_t*)p.q + b * p.q_sb + h * p.q_sh + ic * p.q_ss + at;
        const uint16_t* gp = (const uint16_t*)p.dout + b * p.do_sb + h * p.do_sh + ic * p.do_ss + at;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            q[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(qp + 16 * k));
            g[k] = __builtin_bit_cast(Frag<T>, *(const Raw*)(gp + 16 * k));
        }
    }
    const int64_t stat = ((int64_t)b * p.H + h) * p.S + ic;
    const float c = p.scale * LOG2E, dl = delta[stat];
    float lse2 = lse2_of(p.lse[stat]), unscale = p.scale;
    f32x16 acc[ND] = {};
    const Tiles tiles = tiles_of(p, i00, min(i00 + 127, p.S - 1));
    const Copy<D, TILE> copy;
    KeyBits keys{p.mask ? p.mask + b * p.mask_sb : nullptr, p.S, 1};
    int k0 = tiles.at(0) * TILE;
    copy(kp, p.k_ss, k0, p.S - 1, lk0, wave);
    copy(vp, p.v_ss, k0, p.S - 1, lv0, wave);
    keys.load(k0, lane);
    // tile t from tk and tv, the next one's copies into nk and nv
    if constexpr (NARROW<T>) {                 // P, and so dS, times a power of two of the query's own
        const int nt = (p.S + TILE - 1) / TILE;
        float top = 0.0f;
        for (int t = lane; t < tiles.count; t += 64) top = fmaxf(top, tops.v[((int64_t)b * p.HK + hk) * nt + tiles.at(t)]);
        const int e = shift_of(__builtin_fmaf(sqrtf(row_square<T, D / 16>(g)), wave_max(top), fabsf(dl)));
        lse2 -= (float)e;
        unscale *= power_of_two(-e);
    }
    const auto turn = [&](int t, u32x4* tk, u32x4* tv, u32x4* nk, u32x4* nv) __attribute__((always_inline)) {
        arrived();
        const uint64_t bits = keys.bits(k0);
        if (bits != ~0ull) {
            copy.clear(tk, bits);
            copy.clear(tv, bits);
        }
        __syncthreads();
        const int now = k0;
        if (t + 1 < tiles.count) {
            k0 = tiles.at(t + 1) * TILE;
            copy(kp, p.k_ss, k0, p.S - 1, nk, wave);
            copy(vp, p.v_ss, k0, p.S - 1, nv, wave);
            keys.load(k0, lane);
        }
        if (bits == 0 || i0 >= p.S || none_seen(p, i0, now, now + TILE - 1)) return;
        const uint32_t ra = fresh(rows_at<D>(lane)), ca = fresh(cols_at<D>(lane));
        const uint64_t vis = bits & bits_below(i + p.right + 1 - now) & (bits_from(i - p.left - now) | bits_below(p.sinks - now));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if ((uint32_t)(bits >> (32 * u)) == 0 || none_seen(p, i0, now + 32 * u, now + 32 * u + 31)) continue;
            f32x16 s = mfma(rows_frag<T, D>(tk, ra, 32 * u, 0), q[0], f32x16{});
            f32x16 dp = mfma(rows_frag<T, D>(tv, ra, 32 * u, 0), g[0], f32x16{});
#pragma unroll
            for (int k = 1; k < D / 16; ++k) {
                s = mfma(rows_frag<T, D>(tk, ra, 32 * u, k), q[k], s);
                dp = mfma(rows_frag<T, D>(tv, ra, 32 * u, k), g[k], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = exp2_(__builtin_fmaf(s[r], c, -lse2)) * (dp[r] - dl);
            if ((uint32_t)(bits >> (32 * u)) != ~0u || !all_seen(p, i0, now + 32 * u, now + 32 * u + 31)) {
                const uint32_t mine = lane_rows((uint32_t)(vis >> (32 * u)), lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __uint_as_float(__float_as_uint(s[r]) & keep_mask(mine, r));
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const Frag<T> ds = round_frag<T>(s, w);
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    acc[d] = mfma(cols_frag<T, D>(tk, ca, 32 * u + 16 * w, d), ds, acc[d]);
            }
        }
    };
    for (int t = 0; t < tiles.count; t += 2) {
        turn(t, lk0, lv0, lk1, lv1);
        if (t + 1 < tiles.count) turn(t + 1, lk1, lv1, lk0, lv0);
    }
    store_rows<T, ND>((T*)p.dq + (((int64_t)b * p.S + i) * p.H + h) * D, acc, unscale, i < p.S, lane);
}

// Keys: a workgroup runs 128 keys of a key head, 32 a wave, over the tiles of 64 queries that see them, one query head of
// the group after the other, so that dk and dv of shared heads are sums within one workgroup, in a fixed order.  The
// tiles of the first tokens are seen by every query: their queries are split over `sink_split` workgroups (and all
// tiles' over `split` where there are fewer tiles than compute units), whose float32 sums k_attn_join adds.
// The products start from -lse / scale and -rowsum(do o) in place of zero, so P and dS are an exponential and a product.
struct KeySplit {
    int sink_tiles, sink_split, split;
};
constexpr int KEYS = 128;
// Operands of v that lie in LDS, each lane's own, and are read again for every product: with all of k, v, dk and dv in
// registers nine of a lane's are spilled at D = 128 (four at D = 64 in float16, whose powers of two take some), and a
// read back from scratch memory waits for the copies in flight before it.
template <class T, int D>
constexpr int PARKED = NARROW<T> && D == 64 ? 4 : 3;

template <class T, int D>
DEV void dkv_body(const D8sAttnArgs& p, const float* delta, const Tops& tops, float* part, KeySplit ks, int id, u32x4* lq0, u32x4* lq1, u32x4* lg0,
                  u32x4* lg1, float (*ls)[2 * TILE], u32x4* parked) {
    constexpr int ND = D / 32;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int nk = (p.S + KEYS - 1) / KEYS, G = p.H / p.HK;
    const int items = ks.sink_tiles * ks.sink_split + (nk - ks.sink_tiles) * ks.split;
    const int item = id % items, bh = id / items, b = bh / p.HK, hk = bh % p.HK;
    const bool sink = item < ks.sink_tiles * ks.sink_split;
    const int rest = sink ? item : item - ks.sink_tiles * ks.sink_split, n = sink ? ks.sink_split : ks.split;
    const int kt = (sink ? 0 : ks.sink_tiles) + rest / n, cut = rest % n;
    const int j0 = kt * KEYS, jw = j0 + 32 * wave, j = jw + lane % 32;
    const uint8_t* mask = p.mask ? p.mask + b * p.mask_sb : nullptr;
    const int64_t jc = min(j, p.S - 1);
    const bool on = j < p.S && (mask == nullptr || mask[jc] != 0), any = __any(on);
    Frag<T> k[D / 16], v[D / 16];
    {
        const uint16_t* kp = (const uint16_t*)p.k + b * p.k_sb + hk * p.k_sh + jc * p.k_ss + 8 * (lane / 32);
        const uint16_t* vp = (const uint16_t*)p.v + b * p.v_sb + hk * p.v_sh + jc * p.v_ss + 8 * (lane / 32);
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
            k[u] = __builtin_bit_cast(Frag<T>, *(const Raw*)(kp + 16 * u));
            v[u] = __builtin_bit_cast(Frag<T>, *(const Raw*)(vp + 16 * u));
        }
    }
    // queries that see any of the keys: from j0 - right, to left past the last key or the end for a first token
    const int lo = max(0, j0 - p.right) / TILE;
    const int hi = (j0 < p.sinks ? p.S - 1 : min(p.S - 1, j0 + KEYS - 1 + p.left)) / TILE;
    const int per = hi - lo + 1;
    const int t0 = (int)((int64_t)G * per * cut / n), t1 = (int)((int64_t)G * per * (cut + 1) / n);
    const float c = p.scale * LOG2E, c1 = 1.0f / p.scale;
    f32x16 dk[ND] = {}, dv[ND] = {};
    const Copy<D, TILE> copy;
    float se = 0.0f, sd = 0.0f;                // as they come from memory: used a turn later
    int si = 0;
    int h = hk * G + t0 / per, qt = lo + t0 % per;         // of the tile whose copies are on their way
    const auto load = [&](u32x4* nq, u32x4* ng) __attribute__((always_inline)) {
        copy((const uint16_t*)p.q + b * p.q_sb + h * p.q_sh, p.q_ss, qt * TILE, p.S - 1, nq, wave);
        copy((const uint16_t*)p.dout + b * p.do_sb + h * p.do_sh, p.do_ss, qt * TILE, p.S - 1, ng, wave);
        const int i = qt * TILE + lane;
        const int64_t at = ((int64_t)b * p.H + h) * p.S + min(i, p.S - 1);
        se = p.lse[at];
        if (wave == 0) sd = delta[at];
        si = i;
    };
    if (t0 < t1) load(lq0, lg0);
    // The powers of two (exponents) of P and of v, which dS then has both of: P's between 0 and 14 as far as v can take the
    // rest (raised as far as float16 goes, which costs it no bits, or lowered by 2^10 at most, which costs it what lies
    // below 2^-15)
    int of_p = 0, of_v = 0;
    if constexpr (NARROW<T>) {
        const int nt = (p.S + TILE - 1) / TILE;
        float tops_of[3] = {};                 // |do|, |rowsum(do o)| of the queries, |v| of the keys
        for (int t = t0 + (int)threadIdx.x; t < t1; t += NT) {
            const int64_t at = ((int64_t)b * p.H + hk * G + t / per) * nt + lo + t % per;
            tops_of[0] = fmaxf(tops_of[0], tops.g[at]);
            tops_of[1] = fmaxf(tops_of[1], tops.r[at]);
        }
        if (threadIdx.x < KEYS / TILE) tops_of[2] = tops.v[((int64_t)b * p.HK + hk) * nt + min(j0 / TILE + (int)threadIdx.x, nt - 1)];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            tops_of[k] = wave_max(tops_of[k]);
            if (lane == 0) ls[1][4 * k + wave] = tops_of[k];       // (written again behind the first turn's barrier)
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) tops_of[k] = fmaxf(fmaxf(ls[1][4 * k], ls[1][4 * k + 1]), fmaxf(ls[1][4 * k + 2], ls[1][4 * k + 3]));
        const int e = __builtin_amdgcn_readfirstlane(shift_of(__builtin_fmaf(tops_of[0], tops_of[2], tops_of[1])));
        // (2^15 is the largest power that float16 itself holds)
        const int room = __builtin_amdgcn_readfirstlane(min(max(0, 15 - __builtin_amdgcn_frexp_expf(tops_of[2])), 15));
        of_p = min(max(e, 0), 14);
        of_v = min(max(e - of_p, -10), room);
        of_p = min(of_p, e - of_v);
        const T by = (T)power_of_two(of_v);
#pragma unroll
        for (int u = 0; u < D / 16; ++u) v[u] *= by;
    }
    const float p_add = uniform(of_p * LN2), v_by = power_of_two(of_v);
    parked += threadIdx.x;
#pragma unroll
    for (int x = 0; x < PARKED<T, D>; ++x) parked[x * NT] = __builtin_bit_cast(u32x4, v[x]);
    // tile t from tq and tg, its -lse / scale and -rowsum(do o) (with the powers of two) in `stats`, the next one's copies into nq and ng
    const auto turn = [&](int t, u32x4* tq, u32x4* tg, float* stats, u32x4* nq, u32x4* ng) __attribute__((always_inline)) {
        const int qn = qt * TILE;
        arrived();
        asm volatile("" : "+v"(se), "+v"(sd));
        // a row past the end, or that sees nothing: every P is 0, and whatever memory holds of it is not used
        const bool sees = si < p.S && se != -INFINITY;
        if (mask) {                            // (without one, a query sees itself)
            const uint64_t rows = __ballot(sees);
            if (rows != ~0ull) clear_rows<D>(tq, tg, rows);
        }
        if (wave == 0) {
            stats[lane] = sees ? (NARROW<T> ? p_add - se : -se) * c1 : -INFINITY;
            stats[TILE + lane] = sees ? (NARROW<T> ? -sd * v_by : -sd) : 0.0f;
        }
        __syncthreads();                       // the tile is there, and the other one is no longer read
        if (t + 1 < t1) {
            if (++qt > hi) {
                qt = lo;
                ++h;
            }
            load(nq, ng);
        }
        if (!any) return;
        const uint32_t ra = fresh(rows_at<D>(lane)), ca = fresh(cols_at<D>(lane));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int q0 = qn + 32 * u;
            if (q0 >= p.S || none_seen(p, q0, jw, jw + 31)) continue;
            f32x16 s, dp;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 e = *(const f32x4*)&stats[32 * u + 8 * g + 4 * (lane / 32)];
                const f32x4 d = *(const f32x4*)&stats[TILE + 32 * u + 8 * g + 4 * (lane / 32)];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[4 * g + r] = e[r];
                    dp[4 * g + r] = d[r];
                }
            }
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                s = mfma(rows_frag<T, D>(tq, ra, 32 * u, x), k[x], s);
                dp = mfma(rows_frag<T, D>(tg, ra, 32 * u, x), x < PARKED<T, D> ? __builtin_bit_cast(Frag<T>, parked[fresh(x * NT)]) : v[x], dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = exp2_(s[r] * c);
                dp[r] *= s[r];
            }
            if (!all_seen(p, q0, jw, jw + 31)) {
                // query q0 + r sees key j: r >= j - right - q0, and r <= j + left - q0 or j is a first token
                const uint64_t vis = bits_from(j - p.right - q0) & (j < p.sinks ? ~0ull : bits_below(j + p.left + 1 - q0));
                const uint32_t mine = lane_rows((uint32_t)vis, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t keep = keep_mask(mine, r);
                    s[r] = __uint_as_float(__float_as_uint(s[r]) & keep);
                    dp[r] = __uint_as_float(__float_as_uint(dp[r]) & keep);
                }
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const Frag<T> pf = round_frag<T>(s, w), df = round_frag<T>(dp, w);
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    dv[d] = mfma(cols_frag<T, D>(tg, ca, 32 * u + 16 * w, d), pf, dv[d]);
                    dk[d] = mfma(cols_frag<T, D>(tq, ca, 32 * u + 16 * w, d), df, dk[d]);
                }
            }
        }
    };
    for (int t = t0; t < t1; t += 2) {
        turn(t, lq0, lg0, ls[0], lq1, lg1);
        if (t + 1 < t1) turn(t + 1, lq1, lg1, ls[1], lq0, lg0);
    }
    const float dk_by = NARROW<T> ? p.scale * power_of_two(-of_p - of_v) : p.scale, dv_by = NARROW<T> ? power_of_two(-of_p) : 1.0f;
    if (!on) {                                 // a masked key's column may hold anything: it has no gradient
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
    }
    if (n > 1) {                               // part[problem and item][dk, dv][key][D]
        if (j >= p.S) return;
        float* o = part + (int64_t)id * 2 * KEYS * D + (int64_t)(j - j0) * D + 4 * (lane / 32);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 x, z;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = dk[d][4 * g + r] * dk_by;
                    z[r] = dv[d][4 * g + r] * dv_by;
                }
                *(f32x4*)(o + 32 * d + 8 * g) = x;
                *(f32x4*)(o + KEYS * D + 32 * d + 8 * g) = z;
            }
        return;
    }
    const int64_t at = (((int64_t)b * p.S + j) * p.HK + hk) * D;
    store_rows<T, ND>((T*)p.dk + at, dk, dk_by, j < p.S, lane);
    store_rows<T, ND>((T*)p.dv + at, dv, dv_by, j < p.S, lane);
}

// The first `of_keys` workgroups run keys, the others queries
template <class T, int D>
__global__ __launch_bounds__(NT, (D == 64 ? 3 : 2)) void k_attn_back(D8sAttnArgs p, const float* delta, Tops tops,
                                                                     float* part, KeySplit ks, int of_keys) {
    constexpr int N = TILE * D / 8;
    __shared__ u32x4 a0[N], a1[N], b0[N], b1[N];
    __shared__ float stats[2][2 * TILE];
    __shared__ u32x4 parked[PARKED<T, D> * NT];
    const int w = blockIdx.x;
    if (w < of_keys) dkv_body<T, D>(p, delta, tops, part, ks, xcd_order(w, of_keys), a0, a1, b0, b1, stats, parked);
    else dq_body<T, D>(p, delta, tops, xcd_order(w - of_keys, gridDim.x - of_keys), a0, a1, b0, b1);
}

// dk and dv of the split tiles: the float32 parts summed in order, four values a thread
template <class T, int D>
__global__ __launch_bounds__(NT) void k_attn_join(D8sAttnArgs p, const float* part, KeySplit ks) {
    const int nk = (p.S + KEYS - 1) / KEYS, items = ks.sink_tiles * ks.sink_split + (nk - ks.sink_tiles) * ks.split;
    const int joined = ks.split > 1 ? nk : ks.sink_tiles;          // tiles per problem, the first ones
    const int kt = blockIdx.x % joined, bh = blockIdx.x / joined, b = bh / p.HK, hk = bh % p.HK;
    const bool sink = kt < ks.sink_tiles;
    const int n = sink ? ks.sink_split : ks.split;
    const int first = sink ? kt * n : ks.sink_tiles * ks.sink_split + (kt - ks.sink_tiles) * n;
    const float* src = part + ((int64_t)bh * items + first) * 2 * KEYS * D;
    if (n == 1) return;                        // (written by its one workgroup)
    const int e = (blockIdx.y * NT + threadIdx.x) * 4, which = e / (KEYS * D), j = kt * KEYS + e % (KEYS * D) / D;
    if (j >= p.S) return;
    f32x4 s = {};
    for (int i = 0; i < n; ++i) s += *(const f32x4*)(src + (int64_t)i * 2 * KEYS * D + e);
    T* o = (T*)(which ? p.dv : p.dk) + (((int64_t)b * p.S + j) * p.HK + hk) * D + e % D;
    const float f[4] = {s[0], s[1], s[2], s[3]};
    store_n<T, 4>(o, 4, f);
}

// Into how many workgroups a key tile's queries are split.  In units of one tile of 64 queries for one wave of keys (a
// tile of queries for dq counts the same), a workgroup gets at most its share of all work on the slots of the GPU, at
// least twelve units (a shorter one is mostly beginning and end) and, unless its keys are first tokens, whole tiles
// where there are enough of them.  Tiles of first tokens are split into two workgroups a slot altogether at most: every
// share leaves 2 x 128 x D float32 values, and many first tokens fill the GPU without (1 x 22528 tokens, 32 heads on 8 of
// 128, 255 before each and 4096 first ones: 6.1 -> 5.0 ms, 2.4 -> 0.57 GB).
KeySplit key_split(const D8sAttnArgs* a) {
    const int64_t S = a->S, nk = (S + KEYS - 1) / KEYS, nq = (S + TILE - 1) / TILE, G = a->H / a->HK;
    const int64_t wide = std::min<int64_t>(a->left, S) + std::min<int64_t>(a->right, S);
    const int64_t seen = std::min(nq, (wide + KEYS) / TILE + 1), problems = (int64_t)a->B * a->HK;
    const int64_t slots = (int64_t)d8s_host_cu_count() * (a->D == 64 ? 3 : 2);
    const int64_t all = problems * nk * G * seen * 2;
    const int64_t most = std::max<int64_t>(12, std::min(G * seen, all / slots));
    KeySplit k;
    k.split = (int)((G * seen + most - 1) / most);
    k.sink_tiles = (int)std::min(nk, ((int64_t)a->sinks + KEYS - 1) / KEYS);
    const int64_t sinks = std::max<int64_t>(1, problems * k.sink_tiles), few = (2 * slots + sinks - 1) / sinks;
    k.sink_split = (int)std::min(few, (G * nq + most - 1) / most);
    return k;
}
int64_t key_items(const D8sAttnArgs* a, const KeySplit& k) {
    const int64_t nk = (a->S + KEYS - 1) / KEYS;
    return (int64_t)k.sink_tiles * k.sink_split + (nk - k.sink_tiles) * k.split;
}
uint64_t delta_bytes(const D8sAttnArgs* a) { return ((uint64_t)a->B * a->H * a->S * 4 + 255) / 256 * 256; }
// The tiles' largest norms, where dS is brought into its type's range
uint64_t tops_bytes(const D8sAttnArgs* a) {
    if (a->dtype != D8S_F16) return 0;
    return ((uint64_t)a->B * (2 * a->H + a->HK) * ((a->S + TILE - 1) / TILE) * 4 + 255) / 256 * 256;
}

// ---- one new token against a cache ------------------------------------------------------------------
// A workgroup runs GM query heads of a key head over a share of the keys their token sees.  A key's row is read 16
// bytes a lane by D / 8 lanes, so a wave reads 8 (D = 64) or 4 rows at a time; each group of lanes keeps the softmax
// statistics and the sums of its own keys, and they are joined at the end, across the groups, the waves, and (k_join)
// the shares.  Bound by memory: every key and value is read once for all the heads that share it (up to 8).  Measured:
// 64 requests of 1 .. 8192 tokens, 4096 visible, 32 heads on 8 key heads of 128: 170 us (4.7 TB/s).
template <class T, int D, int GM>
__global__ __launch_bounds__(NT) void k_token(D8sTokenArgs p, int split, float* part) {
    constexpr int LK = D / 8, KW = 64 / LK, U = 4;
    __shared__ float sm[4][GM], sl[4][GM];
    __shared__ float so[4][GM][D];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, gl = lane / LK, dl = lane % LK * 8;
    const int G = p.H / p.HK, ng = (G + GM - 1) / GM;
    const int cut = blockIdx.x % split, pr = blockIdx.x / split, g0 = pr % ng * GM, hk = pr / ng % p.HK, b = pr / ng / p.HK;
    const int gn = min(GM, G - g0);
    const int len = max(0, min(p.lengths[b], p.S)), lo = max(0, len - 1 - p.left), first = min(p.sinks, lo);
    const int seen = first + len - lo;         // visible keys, the first tokens before the window's
    const int e0 = (int)((int64_t)seen * cut / split), e1 = (int)((int64_t)seen * (cut + 1) / split);
    const float c = p.scale * LOG2E;
    float q[GM][8], acc[GM][8], m[GM], l[GM];
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        const int h = hk * G + g0 + min(g, gn - 1);
        load_n<T, 8>((const T*)p.q + b * p.q_sb + h * p.q_sh + dl, 8, q[g]);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            q[g][d] *= c;
            acc[g][d] = 0.0f;
        }
        m[g] = -INFINITY;
        l[g] = 0.0f;
    }
    const T* kp = (const T*)p.k + b * p.k_sb + hk * p.k_sh + dl;
    const T* vp = (const T*)p.v + b * p.v_sb + hk * p.v_sh + dl;
    for (int e = e0 + wave * U * KW; e < e1; e += 4 * U * KW) {
        Vec<T, 8> k[U], v[U];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int x = e + u * KW + gl, xc = min(x, e1 - 1);
            on[u] = x < e1;
            const int64_t j = xc < first ? xc : lo + xc - first;
            k[u] = *(const Vec<T, 8>*)(kp + j * p.k_ss);
            v[u] = *(const Vec<T, 8>*)(vp + j * p.v_ss);
        }
#pragma unroll
        for (int g = 0; g < GM; ++g) {
            float s[U], top = m[g];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x = 0.0f;
#pragma unroll
                for (int d = 0; d < 8; ++d) x = __builtin_fmaf(q[g][d], (float)k[u][d], x);
                x = lanes_sum<LK>(x);
                s[u] = on[u] ? x : -INFINITY;
                top = fmaxf(top, s[u]);
            }
            const float base = top == -INFINITY ? 0.0f : top, a = exp2_(m[g] - base);
            m[g] = top;
            l[g] *= a;
#pragma unroll
            for (int d = 0; d < 8; ++d) acc[g][d] *= a;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float w = exp2_(s[u] - base);
                l[g] += w;
                // (the row read in place of one past the end is a visible key's: its weight is 0, its values may not be)
#pragma unroll
                for (int d = 0; d < 8; ++d) acc[g][d] = on[u] ? __builtin_fmaf(w, (float)v[u][d], acc[g][d]) : acc[g][d];
            }
        }
    }
#pragma unroll
    for (int g = 0; g < GM; ++g) {
        float top = m[g], x, y;
        if constexpr (LK == 8) top = fmaxf(top, dpp<0x128>(top));
        swap16(top, x, y);
        top = fmaxf(x, y);
        swap32(top, x, y);
        top = fmaxf(x, y);
        const float a = top == -INFINITY ? 0.0f : exp2_(m[g] - top);
        const auto join = [&](float f) __attribute__((always_inline)) {
            f *= a;
            if constexpr (LK == 8) f += dpp<0x128>(f);
            swap16(f, x, y);
            f = x + y;
            swap32(f, x, y);
            return x + y;
        };
        l[g] = join(l[g]);
#pragma unroll
        for (int d = 0; d < 8; ++d) acc[g][d] = join(acc[g][d]);
        if (gl == 0) {
            if (dl == 0) {
                sm[wave][g] = top;
                sl[wave][g] = l[g];
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) so[wave][g][dl + d] = acc[g][d];
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < gn * D; x += NT) {
        const int g = x / D, d = x % D;
        const float top = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g]));
        float o = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float a = sm[w][g] == -INFINITY ? 0.0f : exp2_(sm[w][g] - top);
            o = __builtin_fmaf(so[w][g][d], a, o);
            sum = __builtin_fmaf(sl[w][g], a, sum);
        }
        const int64_t head = (int64_t)b * p.H + hk * G + g0 + g;
        if (split == 1) {
            ((T*)p.out)[head * D + d] = (T)(any_weight(sum) ? o / sum : 0.0f);
        } else {                               // part[share][head][m, l, o ...]
            float* t = part + ((int64_t)cut * p.B * p.H + head) * (D + 2);
            if (d == 0) {
                t[0] = top;
                t[1] = sum;
            }
            t[2 + d] = o;
        }
    }
}

// A head's shares joined: their statistics by every wave, their sums by 256 / D groups of threads
template <class T, int D>
__global__ __launch_bounds__(NT) void k_join(const float* part, T* out, int split, int heads) {
    constexpr int GROUPS = NT / D;
    __shared__ float so[GROUPS][D], ss[GROUPS];
    const int head = blockIdx.x, d = threadIdx.x % D, g = threadIdx.x / D, lane = threadIdx.x % 64;
    const float* p = part + (int64_t)head * (D + 2);
    const int64_t step = (int64_t)heads * (D + 2);
    float top = -INFINITY;
    for (int s = lane; s < split; s += 64) top = fmaxf(top, p[s * step]);
#pragma unroll
    for (int x = 32; x >= 1; x /= 2) top = fmaxf(top, __shfl_xor(top, x));
    float o = 0.0f, sum = 0.0f;
#pragma unroll 8
    for (int s = g; s < split; s += GROUPS) {
        const float m = p[s * step], a = m == -INFINITY ? 0.0f : exp2_(m - top);
        sum = __builtin_fmaf(p[s * step + 1], a, sum);
        o = __builtin_fmaf(p[s * step + 2 + d], a, o);
    }
    so[g][d] = o;
    if (d == 0) ss[g] = sum;
    __syncthreads();
    if (g != 0) return;
    sum = ss[0];
#pragma unroll
    for (int x = 1; x < GROUPS; ++x) {
        o += so[x][d];
        sum += ss[x];
    }
    out[(int64_t)head * D + d] = (T)(any_weight(sum) ? o / sum : 0.0f);
}

// Shares of a token's keys: enough workgroups for TOKEN_WGS a compute unit, so that long and short rows even out (the 64
// requests above: 170 us; with 8 a compute unit 176, with 4 186), at least the keys of one turn of a workgroup's waves each
constexpr int TOKEN_WGS = 16;
int token_split(const D8sTokenArgs* a) {
    const int G = a->H / a->HK, gm = G > 4 ? 8 : G > 2 ? 4 : G;
    const int64_t problems = (int64_t)a->B * a->HK * ((G + gm - 1) / gm);
    const int64_t seen = std::min<int64_t>(a->S, (int64_t)a->left + 1 + a->sinks);
    return (int)std::max<int64_t>(1, std::min((TOKEN_WGS * d8s_host_cu_count() + problems - 1) / problems, seen / (a->D == 64 ? 128 : 64)));
}

template <class T, int D>
void token_run(const D8sTokenArgs& a, hipStream_t st) {
    const int G = a.H / a.HK, split = token_split(&a);
    float* part = (float*)a.workspace;
    const auto go = [&](auto kernel, int gm) {
        const int64_t blocks = (int64_t)a.B * a.HK * ((G + gm - 1) / gm) * split;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(NT), 0, st, a, split, part);
    };
    if (G == 1) go(k_token<T, D, 1>, 1);
    else if (G == 2) go(k_token<T, D, 2>, 2);
    else if (G <= 4) go(k_token<T, D, 4>, 4);
    else go(k_token<T, D, 8>, 8);
    if (split > 1)
        hipLaunchKernelGGL((k_join<T, D>), dim3((unsigned)(a.B * a.H)), dim3(NT), 0, st, part, (T*)a.out, split, a.B * a.H);
}

// The arguments with a window no wider than the tokens (the kernels add its sides to positions)
D8sAttnArgs clipped(const D8sAttnArgs* a) {
    D8sAttnArgs c = *a;
    c.left = std::min(a->left, a->S);
    c.right = std::min(a->right, a->S);
    c.sinks = std::min(a->sinks, a->S);
    return c;
}

template <class T, int D>
void attn_run(const D8sAttnArgs& a, hipStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.B * a.H * ((a.S + 127) / 128));
    hipLaunchKernelGGL((k_attn<T, D>), dim3(grid), dim3(NT), 0, st, a);
}

template <class T, int D>
void attn_back_run(const D8sAttnArgs& a, hipStream_t st) {
    float* delta = (float*)a.workspace;
    float* top = (float*)((char*)a.workspace + delta_bytes(&a));
    float* part = (float*)((char*)top + tops_bytes(&a));
    const int64_t tiles = (a.S + TILE - 1) / TILE;
    const Tops tops = {top, top + a.B * a.H * tiles, top + 2 * a.B * a.H * tiles};
    const KeySplit ks = key_split(&a);
    const int problems = a.B * a.HK, nk = (a.S + KEYS - 1) / KEYS;
    const int joined = ks.split > 1 ? nk : ks.sink_split > 1 ? ks.sink_tiles : 0;
    const int of_keys = problems * (int)key_items(&a, ks), of_queries = a.B * a.H * ((a.S + 127) / 128);
    constexpr int ROWS = NARROW<T> ? TILE : NT / (D / 8);
    const unsigned deltas = (unsigned)(a.B * (a.H + (NARROW<T> ? a.HK : 0)) * ((a.S + ROWS - 1) / ROWS));
    hipLaunchKernelGGL((k_attn_delta<T, D>), dim3(deltas), dim3(NT), 0, st, a, delta, tops);
    hipLaunchKernelGGL((k_attn_back<T, D>), dim3((unsigned)(of_keys + of_queries)), dim3(NT), 0, st, a, delta, tops, part, ks, of_keys);
    if (joined)
        hipLaunchKernelGGL((k_attn_join<T, D>), dim3((unsigned)(problems * joined), 2 * KEYS * D / (4 * NT)), dim3(NT), 0, st,
                           a, part, ks);
}

#define BY_TYPE(run, a, st)                                                                            \
    do {                                                                                               \
        if ((a).dtype == D8S_BF16) (a).D == 64 ? run<bf16, 64>((a), st) : run<bf16, 128>((a), st);     \
        else (a).D == 64 ? run<f16, 64>((a), st) : run<f16, 128>((a), st);                             \
    } while (0)

int attn_check(const D8sAttnArgs* a, const char* what) {
    AREQ(a != nullptr, "null arguments");
    AREQ(a->dtype == D8S_BF16 || a->dtype == D8S_F16, "dtype must be D8S_BF16 or D8S_F16");
    AREQ(a->D == 64 || a->D == 128, "D must be 64 or 128");
    AREQ(a->B >= 1 && a->S >= 1 && a->H >= 1 && a->HK >= 1 && a->H % a->HK == 0, "bad sizes (H a multiple of HK)");
    AREQ(a->S <= (1 << 29), "more than 2^29 tokens");
    AREQ((int64_t)a->B * a->H * ((a->S + 127) / 128) < (1 << 24), "too many heads and tokens");
    AREQ(a->left >= 0 && a->right >= 0 && a->sinks >= 0, "left, right and sinks must not be negative");
    AREQ(a->scale >= 0x1p-100f && a->scale <= 0x1p100f, "scale must be 2^-100 .. 2^100 (lse / scale and scale log2(e) are float32)");
    AREQ(a->q && a->k && a->v && a->out, "null pointer");
    return 0;
}

}  // namespace

extern "C" int d8s_attention(const D8sAttnArgs* a, void* stream) {
    const char* what = "d8s_attention";
    if (int rc = attn_check(a, what)) return rc;
    BY_TYPE(attn_run, clipped(a), (hipStream_t)stream);
    return d8s_host_launched(what);
}

extern "C" int d8s_attention_workspace(const D8sAttnArgs* a, uint64_t* bytes) {
    const char* what = "d8s_attention_workspace";
    if (int rc = attn_check(a, what)) return rc;
    AREQ(bytes != nullptr, "null arguments");
    const KeySplit k = key_split(a);
    const bool parts = k.split > 1 || (k.sink_tiles > 0 && k.sink_split > 1);
    *bytes = delta_bytes(a) + tops_bytes(a) + (parts ? (uint64_t)a->B * a->HK * key_items(a, k) * 2 * KEYS * a->D * 4 : 0);
    return 0;
}

extern "C" int d8s_attention_backward(const D8sAttnArgs* a, void* stream) {
    const char* what = "d8s_attention_backward";
    if (int rc = attn_check(a, what)) return rc;
    AREQ(a->lse && a->dout && a->dq && a->dk && a->dv && a->workspace, "null pointer");
    uint64_t need = 0;
    if (int rc = d8s_attention_workspace(a, &need)) return rc;
    AREQ(a->ws_bytes >= need && ((uintptr_t)a->workspace & 15) == 0,
         "workspace smaller than d8s_attention_workspace() or not 16-byte aligned");
    AREQ((int64_t)a->B * a->H * ((a->S + 15) / 16) + (int64_t)a->B * a->HK * key_items(a, key_split(a)) < (1 << 24),
         "too many heads and tokens");
    BY_TYPE(attn_back_run, clipped(a), (hipStream_t)stream);
    return d8s_host_launched(what);
}

static int token_check(const D8sTokenArgs* a, const char* what) {
    AREQ(a != nullptr, "null arguments");
    AREQ(a->dtype == D8S_BF16 || a->dtype == D8S_F16, "dtype must be D8S_BF16 or D8S_F16");
    AREQ(a->D == 64 || a->D == 128, "D must be 64 or 128");
    AREQ(a->B >= 1 && a->S >= 1 && a->H >= 1 && a->HK >= 1 && a->H % a->HK == 0, "bad sizes (H a multiple of HK)");
    AREQ((int64_t)a->B * a->H < (1 << 22), "too many heads");
    AREQ(a->left >= 0 && a->sinks >= 0, "left and sinks must not be negative");
    AREQ(a->scale >= 0x1p-100f && a->scale <= 0x1p100f, "scale must be 2^-100 .. 2^100 (lse / scale and scale log2(e) are float32)");
    return 0;
}

extern "C" int d8s_attention_token_workspace(const D8sTokenArgs* a, uint64_t* bytes) {
    const char* what = "d8s_attention_token_workspace";
    if (int rc = token_check(a, what)) return rc;
    AREQ(bytes != nullptr, "null arguments");
    const int split = token_split(a);
    *bytes = split > 1 ? (uint64_t)split * a->B * a->H * (a->D + 2) * 4 : 0;
    return 0;
}

extern "C" int d8s_attention_token(const D8sTokenArgs* a, void* stream) {
    const char* what = "d8s_attention_token";
    if (int rc = token_check(a, what)) return rc;
    AREQ(a->q && a->k && a->v && a->out && a->lengths, "null pointer");
    uint64_t need = 0;
    if (int rc = d8s_attention_token_workspace(a, &need)) return rc;
    AREQ(need == 0 || (a->workspace && a->ws_bytes >= need), "workspace smaller than d8s_attention_token_workspace()");
    BY_TYPE(token_run, *a, (hipStream_t)stream);
    return d8s_host_launched(what);
}
