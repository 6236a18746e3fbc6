// Rotary positions (with the norm of each head in the same pass, and the gradient of both) and the
// drawing of tokens, on gfx950.  Interfaces: drhip_rotary_t and drhip_sample_t in include/drhip.h.
#include "../../include/drhip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

constexpr int kThreads = 256;

// ---- rotary positions -------------------------------------------------------------------------
//
//   y = R(position) (w * x * r),  r = (mean x^2 + eps)^-1/2      (without a weight: y = R x)
//   R turns the pair (a, b) with number i by position * frequency_i / stretch; pairs are elements
//   (i, i + dims/2) or (2i, 2i + 1); elements from `dims` on are left as they are
//   gradient: g = R^T dy,  dx = r (w g - xhat mean(w g xhat)),  dw = sum over rows of g xhat,  xhat = r x
//
// Bound by memory: a row is read and written once (4 sequences of 4096, 40 heads of 128: 671 MB in 123 us,
// 5.5 TB/s; in float64 1342 MB in 244).  A row belongs to a group of 2^k lanes, eight elements
// each (the halves of four pairs); a group takes two heads of one token, so that the angles, which need 64 bits
// (positions of a million turn by a million radians), are computed once for them.

typedef drhip_rotary_t Rot;

template <typename T> struct Vec4 { T v[4]; };

template <typename T> __device__ __forceinline__ void load_quad(T (&x)[4], const T* p) {
    *(Vec4<T>*)x = *(const Vec4<T>*)__builtin_assume_aligned(p, 16);
}
template <typename T> __device__ __forceinline__ void store_quad(T* p, const T (&x)[4]) {
    *(Vec4<T>*)__builtin_assume_aligned(p, 16) = *(const Vec4<T>*)x;
}

__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }

// A lane's share of a row: pairs (a[n], b[n]) with number idx[n], and elements behind `dims`
template <typename T, bool WIDE> struct Row {
    T a[4], b[4], rest[8];
    // number of the lane's pair n
    __device__ __forceinline__ static int pair(const Rot& p, int lane, int lanes, int n) {
        if (!WIDE) return lane + n * lanes;
        const int half = p.dims / 2;
        if (!p.interleaved) return 4 * lane + n;
        return n < 2 ? 2 * lane + n : half / 2 + 2 * lane + n - 2;
    }
    // which element at(n) is; -1 for none
    __device__ __forceinline__ static int element(const Rot& p, int lane, int lanes, int n) {
        const int half = p.dims / 2;
        if (n >= 8) {
            const int i = WIDE ? 4 * (lane + (n >= 12 ? lanes : 0)) + (n & 3) : lane + (n - 8) * lanes;
            return i < p.d - p.dims ? p.dims + i : -1;
        }
        const bool second = n >= 4;
        const int i = pair(p, lane, lanes, n & 3);
        if ((WIDE ? 4 * lane : i) >= half) return -1;
        return p.interleaved ? 2 * i + second : i + (second ? half : 0);
    }
    __device__ __forceinline__ void load(const Rot& p, const T* row, int lane, int lanes, bool ok) {
        const int half = p.dims / 2, behind = p.d - p.dims;
        if constexpr (WIDE) {
            T u[4] = {}, v[4] = {};
            if (ok && 4 * lane < half) {
                load_quad(u, row + 4 * lane);
                load_quad(v, row + half + 4 * lane);
            }
            spread(p, u, v);
            T s[4] = {}, t[4] = {};
            if (behind) {
                if (ok && 4 * lane < behind) load_quad(s, row + p.dims + 4 * lane);
                if (ok && 4 * (lane + lanes) < behind) load_quad(t, row + p.dims + 4 * (lane + lanes));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) rest[n] = s[n], rest[4 + n] = t[n];
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = lane + n * lanes;
                const bool in = ok && i < half;
                a[n] = in ? row[p.interleaved ? 2 * i : i] : T(0);
                b[n] = in ? row[p.interleaved ? 2 * i + 1 : half + i] : T(0);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int i = lane + n * lanes;
                rest[n] = ok && i < behind ? row[p.dims + i] : T(0);
            }
        }
    }
    __device__ __forceinline__ void spread(const Rot& p, const T (&u)[4], const T (&v)[4]) {
        if (p.interleaved) {
            a[0] = u[0], b[0] = u[1], a[1] = u[2], b[1] = u[3];
            a[2] = v[0], b[2] = v[1], a[3] = v[2], b[3] = v[3];
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) a[n] = u[n], b[n] = v[n];
        }
    }
    __device__ __forceinline__ void store(const Rot& p, T* row, int lane, int lanes) const {
        const int half = p.dims / 2, behind = p.d - p.dims;
        if constexpr (WIDE) {
            if (4 * lane < half) {
                T u[4], v[4];
                if (p.interleaved) {
                    u[0] = a[0], u[1] = b[0], u[2] = a[1], u[3] = b[1];
                    v[0] = a[2], v[1] = b[2], v[2] = a[3], v[3] = b[3];
                } else {
#pragma unroll
                    for (int n = 0; n < 4; ++n) u[n] = a[n], v[n] = b[n];
                }
                store_quad(row + 4 * lane, u);
                store_quad(row + half + 4 * lane, v);
            }
            if (behind) {
                T s[4], t[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) s[n] = rest[n], t[n] = rest[4 + n];
                if (4 * lane < behind) store_quad(row + p.dims + 4 * lane, s);
                if (4 * (lane + lanes) < behind) store_quad(row + p.dims + 4 * (lane + lanes), t);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int i = lane + n * lanes;
                if (i < half) {
                    row[p.interleaved ? 2 * i : i] = a[n];
                    row[p.interleaved ? 2 * i + 1 : half + i] = b[n];
                }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int i = lane + n * lanes;
                if (i < behind) row[p.dims + i] = rest[n];
            }
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int n = 0; n < 4; ++n) f(a[n], n), f(b[n], 4 + n);
#pragma unroll
        for (int n = 0; n < 8; ++n) f(rest[n], 8 + n);
    }
    __device__ __forceinline__ T& at(int n) { return n < 4 ? a[n] : n < 8 ? b[n - 4] : rest[n - 8]; }
    __device__ __forceinline__ const T& at(int n) const { return n < 4 ? a[n] : n < 8 ? b[n - 4] : rest[n - 8]; }
    __device__ __forceinline__ void turn(const T (&c)[4], const T (&s)[4]) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const T x = a[n], y = b[n];
            a[n] = fused(x, c[n], -y * s[n]);
            b[n] = fused(y, c[n], x * s[n]);
        }
    }
};

__device__ __forceinline__ float root(float x) { return sqrtf(x); }
__device__ __forceinline__ double root(double x) { return sqrt(x); }

template <typename T> __device__ __forceinline__ T group_sum(T x, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// Frequencies of the lane's pairs: from the table, or base^(-2i / dims)
template <typename T, bool WIDE>
__device__ __forceinline__ void frequencies(const Rot& p, int lane, int lanes, double (&f)[4]) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int i = Row<T, WIDE>::pair(p, lane, lanes, n);
        const bool in = i < p.dims / 2;
        f[n] = p.frequencies ? (in ? p.frequencies[i] : 0.0) : exp2(i * p.step);
        f[n] *= p.squeeze;
    }
}

// cos and sin of position * f.  In float32 the angle is reduced to half turns between -1 and 1 in 64 bits first; what
// rounding that takes away, up to 9e-8, is put back (cos(x + e) = cos x - e sin x).
template <typename T>
__device__ __forceinline__ void angles(const Rot& p, double position, const double (&f)[4], T (&c)[4], T (&s)[4]) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const double angle = position * f[n];
        double x, y;
        if constexpr (sizeof(T) == 4) {
            const double turns = angle * 0.15915494309189533577, half = 2.0 * (turns - rint(turns));
            const float near = (float)half, rest = (float)((half - (double)near) * 3.14159265358979323846);
            float u, v;
            sincospif(near, &u, &v);
            const float cosine = fmaf(-u, rest, v), sine = fmaf(v, rest, u);
            c[n] = cosine * (float)p.magnitude, s[n] = sine * (float)(p.sign * p.magnitude);
        } else {
            sincos(angle, &x, &y);
            c[n] = y * p.magnitude, s[n] = x * p.sign * p.magnitude;
        }
    }
}

__device__ __forceinline__ double position_of(const Rot& p, int b, int l) {
    if (!p.positions) return (double)(p.first + l);
    const int64_t at = b * p.positions_stride + l;
    return p.positions_wide ? (double)((const int64_t*)p.positions)[at] : (double)((const int32_t*)p.positions)[at];
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Rot p, int lanes_log, int slots, int64_t groups) {
    const int lanes = 1 << lanes_log;
    const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> lanes_log;
    const int lane = threadIdx.x & (lanes - 1);
    const bool live = id < groups;
    const int64_t g = live ? id : 0;
    // a token's heads are taken by `slots` groups in turn, which are neighbours
    const int slot = (int)(g % slots);
    const int64_t token = g / slots;
    const int b = (int)(token / p.rows), l = (int)(token % p.rows);
    double f[4];
    T c[4], s[4];
    frequencies<T, WIDE>(p, lane, lanes, f);
    angles<T>(p, position_of(p, b, l), f, c, s);
    for (int h = slot; h < p.heads; h += slots) {
        Row<T, WIDE> x;
        x.load(p, (const T*)p.x + b * p.x_stride[0] + h * p.x_stride[1] + l * p.x_stride[2], lane, lanes, live);
        if (p.weight) {
            T sum = 0;
            x.each([&](T& v, int) { sum = fused(v, v, sum); });
            sum = group_sum(sum, lanes);
            const T r = T(1) / root(sum / T(p.d) + T(p.eps));
            Row<T, WIDE> w;
            w.load(p, (const T*)p.weight + h * p.weight_stride, lane, lanes, true);
            x.each([&](T& v, int n) { v = v * r * w.at(n); });
        }
        x.turn(c, s);
        if (live) x.store(p, (T*)p.y + b * p.y_stride[0] + h * p.y_stride[1] + l * p.y_stride[2], lane, lanes);
    }
}

// Gradient with a norm.  A block owns a head and every `slots`-th run of tokens, its groups one token each; a lane keeps
// the sums of its elements of dw, the groups meet in LDS, the blocks in `rotary_dw`.  A group has one or a few
// tokens, so it waits for memory more than it computes: one head for a block, whose registers leave room for four
// waves on a SIMD (20 heads of 128, 3554 tokens: 25 us, 4.4 TB/s; in float64 39, 5.6), not two, which share the angles
// but leave room for two (8 us more), and the loads ahead of the angles.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void rotary_grad_kernel(Rot p, int lanes_log, int slots) {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const int lanes = 1 << lanes_log, groups = kThreads >> lanes_log;
    const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> lanes_log;
    const int slot = blockIdx.x % slots, h = blockIdx.x / slots;
    const int64_t tokens = (int64_t)p.batch * p.rows;
    double f[4];
    frequencies<T, WIDE>(p, lane, lanes, f);
    Row<T, WIDE> w;
    T sums[16];
    w.load(p, (const T*)p.weight + h * p.weight_stride, lane, lanes, true);
#pragma unroll
    for (int n = 0; n < 16; ++n) sums[n] = 0;
    for (int64_t t0 = (int64_t)slot * groups; t0 < tokens; t0 += (int64_t)slots * groups) {
        const int64_t token = t0 + group;
        const bool live = token < tokens;
        const int b = live ? (int)(token / p.rows) : 0, l = live ? (int)(token % p.rows) : 0;
        Row<T, WIDE> x, g;
        x.load(p, (const T*)p.x + b * p.x_stride[0] + h * p.x_stride[1] + l * p.x_stride[2], lane, lanes, live);
        g.load(p, (const T*)p.dy + b * p.dy_stride[0] + h * p.dy_stride[1] + l * p.dy_stride[2], lane, lanes, live);
        T c[4], s[4];
        angles<T>(p, position_of(p, b, l), f, c, s);
        g.turn(c, s);
        T square = 0, dot = 0;
        x.each([&](T& v, int n) {
            square = fused(v, v, square);
            dot = fused(v, g.at(n) * w.at(n), dot);
        });
        square = group_sum(square, lanes);
        dot = group_sum(dot, lanes);
        const T r = T(1) / root(square / T(p.d) + T(p.eps));
        const T mean = dot * r * r / T(p.d);            // mean(w g xhat) r
        Row<T, WIDE> out;
        out.each([&](T& v, int n) {
            const T hat = x.at(n) * r;
            sums[n] = live ? fused(g.at(n), hat, sums[n]) : sums[n];
            v = r * fused(-x.at(n), mean, g.at(n) * w.at(n));
        });
        if (live) out.store(p, (T*)p.y + b * p.y_stride[0] + h * p.y_stride[1] + l * p.y_stride[2], lane, lanes);
    }
    // [n][lane] summed over the groups in their order, in 64 bits (in 32 their roundings were half of dw's error)
    T* lds = (T*)shared;
#pragma unroll
    for (int n = 0; n < 16; ++n) lds[n * kThreads + threadIdx.x] = sums[n];
    __syncthreads();
    for (int o = threadIdx.x; o < 16 << lanes_log; o += kThreads) {
        const int n = o >> lanes_log, i = Row<T, WIDE>::element(p, o & (lanes - 1), lanes, n);
        double total = 0.0;
#pragma unroll 8
        for (int j = 0; j < groups; ++j) total += (double)lds[n * kThreads + j * lanes + (o & (lanes - 1))];
        if (i >= 0) ((T*)p.work)[((int64_t)slot * p.heads + h) * p.d_pad + i] = (T)total;
    }
}

// dw from the blocks' parts, in their order; a weight shared by the heads takes all of theirs.  A few
// hundred KB: 5 us for 20 heads of 128 from 56 blocks each, the loads' way and the launch.
template <typename T> __global__ __launch_bounds__(kThreads) void rotary_dw(Rot p, int slots) {
    __shared__ double lds[4][64];
    const int d = (int)blockIdx.x % ((p.d + 63) / 64) * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    const int head = blockIdx.x / ((p.d + 63) / 64);
    const bool shared_weight = p.weight_stride == 0;
    const int64_t count = shared_weight ? (int64_t)slots * p.heads : slots;
    double sum = 0.0;
    if (d < p.d)
#pragma unroll 8
        for (int64_t n = part; n < count; n += 4)
            sum += (double)((const T*)p.work)[(shared_weight ? n : n * p.heads + head) * p.d_pad + d];
    lds[part][threadIdx.x & 63] = sum;
    __syncthreads();
    if (part == 0 && d < p.d) {
        const int k = threadIdx.x & 63;
        ((T*)p.dweight)[(int64_t)head * p.d + d] = (T)(((lds[0][k] + lds[1][k]) + lds[2][k]) + lds[3][k]);
    }
}

int lanes_log_of(const Rot& p) {
    const int half = p.dims / 2, behind = p.d - p.dims;
    int lanes = (half + 3) / 4;
    if ((behind + 7) / 8 > lanes) lanes = (behind + 7) / 8;
    int log = 0;
    while ((1 << log) < lanes) ++log;
    return log;
}

bool quads(const void* p, const int64_t* stride, int n, int item) {
    if (!p) return true;
    if ((uintptr_t)p % 16) return false;
    for (int i = 0; i < n; ++i)
        if (stride[i] * item % 16) return false;
    return true;
}

bool wide_of(const Rot& p) {
    const int item = p.is_double ? 8 : 4, half = p.dims / 2;
    return half % 4 == 0 && (p.d - p.dims) % 4 == 0 && quads(p.x, p.x_stride, 3, item) && quads(p.y, p.y_stride, 3, item) &&
           quads(p.dy, p.dy_stride, 3, item) && quads(p.weight, &p.weight_stride, 1, item);
}

// Blocks for each head in the gradient: up to 2048 in all (8 for a compute unit), and two tokens for each group:
// with one the parts of dw, a row for each block, are twice as many and their sum takes twice as long (10 us for 5)
int grad_slots(const Rot& p) {
    const int64_t groups = kThreads >> lanes_log_of(p);
    const int64_t runs = ((int64_t)p.batch * p.rows + groups - 1) / groups;
    int64_t slots = 2048 / (p.heads ? p.heads : 1);
    if (slots > (runs + 1) / 2) slots = (runs + 1) / 2;
    return slots < 1 ? 1 : (int)slots;
}

// Groups for each token's heads.  Two heads share the angles (4 x 4096 tokens of 40 heads of 128: 124 us; four heads
// 129, eight 137), one where the rows would not fill the device
int rotary_slots(const Rot& p) {
    const int64_t tokens = (int64_t)p.batch * p.rows;
    return tokens * ((p.heads + 1) / 2) << lanes_log_of(p) < 256 * 2048 ? p.heads : (p.heads + 1) / 2;
}

int64_t rotary_blocks(const Rot& p) {
    return (((int64_t)p.batch * p.rows * rotary_slots(p) << lanes_log_of(p)) + kThreads - 1) / kThreads;
}

template <typename T> void launch_rotary(const Rot& p, hipStream_t s) {
    const int log = lanes_log_of(p), slots = rotary_slots(p);
    const int64_t groups = (int64_t)p.batch * p.rows * slots;
    const unsigned blocks = (unsigned)rotary_blocks(p);
    if (wide_of(p))
        rotary_kernel<T, true><<<blocks, kThreads, 0, s>>>(p, log, slots, groups);
    else
        rotary_kernel<T, false><<<blocks, kThreads, 0, s>>>(p, log, slots, groups);
}

template <typename T> void launch_rotary_grad(const Rot& p, hipStream_t s) {
    const int log = lanes_log_of(p), slots = grad_slots(p);
    const unsigned blocks = (unsigned)(p.heads * slots);
    const unsigned lds = 16 * kThreads * sizeof(T);
    if (!blocks) {      // no heads: a weight for all of them has a gradient of zeros
    } else if (wide_of(p))
        rotary_grad_kernel<T, true><<<blocks, kThreads, lds, s>>>(p, log, slots);
    else
        rotary_grad_kernel<T, false><<<blocks, kThreads, lds, s>>>(p, log, slots);
    const unsigned parts = (unsigned)((p.d + 63) / 64 * (p.weight_stride ? p.heads : 1));
    if (parts) rotary_dw<T><<<parts, kThreads, 0, s>>>(p, slots);
}

// ---- drawing tokens ---------------------------------------------------------------------------
//
// Tokens in the order (logit falling, number rising); weights exp((logit - largest) / temperature).  top-k
// keeps the first k, top-p the first ones until their weight reaches p of what is left, min-p those of at
// least min_p of the largest weight: all three are beginnings of that order.  The token is the first one,
// by number, at which the kept weight summed from token 0 exceeds u times all kept weight.
//
// A block for each row.  The row is not sorted: one pass finds the largest logit and counts those of each beginning
// of 13 bits (for top-k), or a second one sums the weights in steps of their logarithm (for top-p); only the tokens
// of the digit or step where a beginning ends, or the few kept ones themselves, go to LDS and are ordered there.
// Where more share a step than LDS holds (many equal logits) the end is found digit by digit over the whole row
// instead.  Weights are 64-bit whole numbers (the largest 2^s, s such that all fit, computed in float64), so that
// sums do not depend on their order; what is below 2^-(s + 1) of the largest is none (s = 45 for 128000 tokens).
//
// 256 rows of 128000 with top-k 50: 39 us, more than half of it the first pass at memory's rate (131 MB).  One row of 32000
// with top-p: 33 us on one compute unit, of which 9 are the weights of all tokens (float64, 13 operations each), 7 the
// kept ones' sums, 12 barriers and scans between the steps.

typedef drhip_sample_t Smp;
typedef unsigned long long u64;
constexpr int kDraw = 1024;          // threads of a block
constexpr int kBins = 2048;          // of a digit of 11 bits
constexpr int kCoarse = 8192;        // of the first 13 bits
constexpr int kChunks = 2048;        // parts of a row whose weights are kept for the last search
constexpr int kList = 2048;          // tokens that LDS holds
constexpr int kHead = 16384;
constexpr int kFew = 128;            // of which so many are ordered by comparing all

__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0;                                    // a NaN is below everything and never drawn
    const unsigned u = __float_as_uint(x + 0.0f);            // (-0 and 0 are equal)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// Position in the order as one number: larger is earlier
__device__ __forceinline__ u64 rank_of(float x, int i) { return (u64)key_of(x) << 32 | (unsigned)~i; }

struct Weigher {
    float least;          // smaller ones have no weight: -inf, NaN, and finite ones where the largest is infinite
    float floor, high;    // for the arithmetic logits lie between: weights of about 2^-400 are nothing
    double zero, by, one; // the largest logit, log2(e) / temperature, 2^s
    const double* roots;  // 2^(j/64)
    // log2 of a weight in 64ths, and the rest: t = k / 64 + rest.  Rises with the logit, is 0 for the largest.
    struct Power {
        int k;
        double rest;
    };
    __device__ __forceinline__ Weigher(float top, double rate, double one, const double* roots) : one(one), roots(roots) {
        constexpr float far = 3.40282347e38f;
        high = fminf(top, far), zero = high, least = top > far ? top : -far;
        const float below = fmaxf(nextafterf(high, -__builtin_inff()), -far);
        // (at the highest rate the next smaller logit has no weight; the floor's rounding moves t by 400 at most, and powers
        // of two down to 2^-1022 can be told apart)
        by = below < high ? fmin(rate, 400.0 / (zero - (double)below)) : 1.0;
        floor = fminf(below, (float)fmax(zero - 400.0 / by, -(double)far));
    }
    __device__ __forceinline__ Power power(float x) const {
        const double t = ((double)__builtin_amdgcn_fmed3f(x, floor, high) - zero) * by;
        const double shift = 105553116266496.0, u = t + shift;            // 1.5 * 2^46, whose last bit is 1/64 ...
        return {x >= least ? (int)(unsigned)__double_as_longlong(u) : -25600, t - (u - shift)};
    }
    // 2^rest: |rest| <= 1/128, a polynomial of degree 4 (own fit, relative error 5e-15).  No conversions to integers, which
    // take four times as long as a product.
    __device__ __forceinline__ static double part(double f) {
        double p = 0.009618138509201629;
        p = fma(p, f, 0.05550419004645178);
        p = fma(p, f, 0.24022650695902897);
        p = fma(p, f, 0.6931471805593244);
        return fma(p, f, 1.0);
    }
    __device__ __forceinline__ double whole_part(int k) const {
        return __longlong_as_double(__double_as_longlong(roots[k & 63]) + ((long long)(k >> 6) << 52));
    }
    __device__ __forceinline__ double real(float x) const {
        const Power t = power(x);
        return part(t.rest) * whole_part(t.k);
    }
    // nearest whole number of 2^t * 2^s <= 2^52: the low bits of its sum with 2^52
    __device__ __forceinline__ u64 whole_of(const Power& t) const {
        const double x = fma(part(t.rest), whole_part(t.k) * one, 4503599627370496.0);
        return (u64)__double_as_longlong(x) - 0x4330000000000000ull;
    }
    __device__ __forceinline__ u64 whole(float x) const { return whole_of(power(x)); }
    __device__ __forceinline__ u64 whole_from(float x, double min_p) const {      // 0 below min_p of the largest
        const Power t = power(x);
        return part(t.rest) * whole_part(t.k) >= min_p ? whole_of(t) : 0;
    }
};

// f(number, logit) for the tokens from `first` to `v`, eight loads at a time under way
template <typename F> __device__ __forceinline__ void each_token(const float* row, int first, int v, F f) {
    int i = first + threadIdx.x;
    for (; i + 7 * kDraw < v; i += 8 * kDraw) {
        float x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = row[i + n * kDraw];
#pragma unroll
        for (int n = 0; n < 8; ++n) f(i + n * kDraw, x[n]);
    }
    for (; i < v; i += kDraw) f(i, row[i]);
}

// f(logit) for one part of the row by one wave, from number `first` to `end`, with NaN for what the last turn has too much
template <typename F> __device__ __forceinline__ void each_of_part(const float* row, int first, int end, F f) {
    for (int i0 = first + (threadIdx.x & 63); i0 < end; i0 += 512) {
        float x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = row[min(i0 + 64 * n, end - 1)];
#pragma unroll
        for (int n = 0; n < 8; ++n) f(i0 + 64 * n < end ? x[n] : __builtin_nanf(""));
    }
}

// x of another lane of the same 16 (or, with CTRL 0x142 and 0x143, of the last lane of the 16 or 32 before) without
// LDS; 0 where there is none and in rows of 16 that ROWS leaves out
template <int CTRL, int ROWS = 15> __device__ __forceinline__ u64 moved(u64 x) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, CTRL, ROWS, 15, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), CTRL, ROWS, 15, false);
    return (u64)hi << 32 | lo;
}

__device__ __forceinline__ u64 of_lane(u64 x, int lane) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, lane);
}

// f over the wave's values, in every lane: neighbours, pairs, fours and eights of 16 lanes, then the four rows
template <typename F> __device__ __forceinline__ u64 of_wave(u64 x, F f) {
    x = f(x, moved<0xb1>(x));
    x = f(x, moved<0x4e>(x));
    x = f(x, moved<0x141>(x));
    x = f(x, moved<0x140>(x));
    return f(f(of_lane(x, 0), of_lane(x, 16)), f(of_lane(x, 32), of_lane(x, 48)));
}
__device__ __forceinline__ u64 wave_sum(u64 x) {
    return of_wave(x, [](u64 a, u64 b) { return a + b; });
}

// Lanes before this one in a mask, and `more`
__device__ __forceinline__ int lanes_before(u64 mask, int more) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, more));
}

// Sum over the wave's lanes up to this one
__device__ __forceinline__ u64 wave_scan(u64 x) {
    x += moved<0x111>(x);
    x += moved<0x112>(x);
    x += moved<0x114>(x);
    x += moved<0x118>(x);
    x += moved<0x142, 10>(x);
    return x + moved<0x143, 12>(x);
}

// Sum over the threads before this one, and over all (`lds`: 17 words)
__device__ __forceinline__ u64 scan(u64 x, u64* lds, u64& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 sum = wave_scan(x);
    __syncthreads();
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    u64 before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kDraw / 64; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    all = total;
    return before + sum - x;
}

struct Found {
    unsigned bin;
    u64 before, inside;       // of the bins above it, and its own
};

// The highest bins first: the one in which the running sum first reaches `want(all)`, between 1 and all
template <int BINS, typename T, typename W> __device__ __forceinline__ Found reach(const T* hist, W want_of, u64* lds, Found* out) {
    constexpr int PER = BINS / kDraw;
    const int first = BINS - 1 - PER * threadIdx.x;
    u64 sum = 0;
#pragma unroll
    for (int n = 0; n < PER; ++n) sum += hist[first - n];
    u64 all, before = scan(sum, lds, all);
    const u64 want = want_of(all);
    if (before < want && want <= before + sum) {
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const u64 x = hist[first - n];
            if (before < want && want <= before + x) *out = {(unsigned)(first - n), before, x};
            before += x;
        }
    }
    __syncthreads();
    return *out;
}

// The key at which the running sum (of counts, or of weights) over falling keys first reaches `want`, over the
// tokens with keys of at least `least` and, in place of those with `tie_key`, `ties` of them; before: the sum of the larger ones
template <bool COUNT>
__device__ unsigned select(const float* row, int v, unsigned least, u64 ties, unsigned tie_key, u64 want, const Weigher& weigh,
                           u64* hist, u64* lds, Found* found, u64& before) {
    unsigned prefix = 0;
    before = 0;
#pragma unroll
    for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
        const int bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kBins; i += kDraw) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < v; i += kDraw) {
            const float x = row[i];
            const unsigned key = key_of(x);
            if (key < least || key == tie_key) continue;
            if (level && key >> (shift + bits) != prefix) continue;
            atomicAdd(&hist[key >> shift & ((1u << bits) - 1)], COUNT ? 1 : weigh.whole(x));
        }
        if (!COUNT && threadIdx.x == 0 && ties && (!level || tie_key >> (shift + bits) == prefix))
            atomicAdd(&hist[tie_key >> shift & ((1u << bits) - 1)], ties * weigh.whole(value_of(tie_key)));
        __syncthreads();
        const u64 rest = want - before;
        const Found f = reach<kBins>(hist, [&](u64) { return rest; }, lds, found);
        before += f.before;
        prefix = prefix << bits | f.bin;
        __syncthreads();
    }
    return prefix;
}

// Sorts n entries, largest first, in place (a bitonic network over the next power of two)
__device__ __forceinline__ void sort_down(u64* list, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kDraw) list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            for (int t = threadIdx.x; t < size >> 1; t += kDraw) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;      // pairs j apart
                const u64 x = list[a], y = list[b];
                if ((x < y) == !(a & k)) list[a] = y, list[b] = x;
            }
            __syncthreads();
        }
}

__global__ __launch_bounds__(kDraw) void sample_kernel(Smp p) {
    __shared__ u64 coarse[kCoarse];            // weights of the first 13 bits, or counts, or the digits of `select`
    __shared__ u64 list[kList], weights[kFew], parts[kChunks], lds[kDraw / 64 + 1];
    __shared__ unsigned marks[kChunks];
    __shared__ double roots[64];
    __shared__ Found found;
    __shared__ int listed, chunk_at;
    __shared__ u64 chunk_before, chunk_tied, cut_rank;
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float* row = p.logits + b * p.logits_stride;
    const int v = p.vocabulary;
    const double temperature = p.temperature ? p.temperature[b] : p.temperature_all;
    const int64_t k = p.top_k ? p.top_k[b] : p.top_k_all;
    const double top_p = fmax(p.top_p ? p.top_p[b] : p.top_p_all, 0.0);      // (conversions of negative numbers below have no defined result)
    const bool counted = k > 0 && k < v && temperature > 0.0, cut_p = top_p < 1.0;
    double min_p = p.min_p ? p.min_p[b] : p.min_p_all;
    if (!(min_p > 0.0)) min_p = 0.0;
    if (min_p > 1.0) min_p = 1.0;
    const double u = p.uniforms_wide ? ((const double*)p.uniforms)[b] : (double)((const float*)p.uniforms)[b];

    // largest logit, lowest number first, and how many tokens have each beginning of 13 bits
    unsigned* counts = (unsigned*)coarse;
    if (counted)
        for (int i = threadIdx.x; i < kCoarse; i += kDraw) counts[i] = 0;
    if (threadIdx.x == 0) listed = 0, chunk_at = 0, chunk_before = 0, chunk_tied = 0, cut_rank = 0, found = {0, 0, 0};
    __syncthreads();
    float most = -__builtin_inff();
    int where = 0;
    auto larger = [&](int i, float x) {
        where = x > most ? i : where;
        most = x > most ? x : most;
    };
    // Of a long row the first kHead tokens say from which digit on a token can be one of the first k, so that the others
    // that are go to the list at once, and only kHead are read again
    const int head = v >= 4 * kHead && k * (v / kHead) <= kList / 2 ? kHead : v;
    if (counted) {
        each_token(row, 0, head, [&](int i, float x) {
            larger(i, x);
            atomicAdd(&counts[key_of(x) >> 19], 1u);
        });
        if (head < v) {
            __syncthreads();
            const unsigned least = reach<kCoarse>(counts, [&](u64) { return (u64)k; }, lds, &found).bin;
            each_token(row, head, v, [&](int i, float x) {
                larger(i, x);
                const unsigned digit = key_of(x) >> 19;
                atomicAdd(&counts[digit], 1u);
                if (digit >= least) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < kList) list[at] = rank_of(x, i);
                }
            });
        }
    } else
        each_token(row, 0, v, larger);
    u64 best = rank_of(most, where);
    best = of_wave(best, [](u64 a, u64 b) { return a > b ? a : b; });
    if (lane == 0) lds[wave] = best;
    __syncthreads();
    best = 0;
#pragma unroll
    for (int w = 0; w < kDraw / 64; ++w) best = lds[w] > best ? lds[w] : best;
    __syncthreads();
    const unsigned top_key = (unsigned)(best >> 32);
    const bool none = top_key <= key_of(-__builtin_inff());
    if (none || !(temperature > 0.0)) {
        if (threadIdx.x == 0) p.tokens[b] = none ? -1 : (int64_t)(int)~(unsigned)best;
        return;
    }
    if (threadIdx.x < 64) roots[threadIdx.x] = exp2(threadIdx.x / 64.0);
    __syncthreads();
    const Weigher weigh{value_of(top_key), 1.4426950408889634074 / temperature, p.one, roots};

    // end of what is kept: ranks of at least `cut`; where that is not known, keys above `cut_key`, and the first
    // `ties` tokens whose key it is
    const unsigned no_key = ~0u;       // (of no number)
    u64 cut = 0, ties = ~0ull;
    unsigned cut_key = 0;
    bool by_key = false;
    u64 before;

    // the draw as a part of all kept weight
    auto target_of = [&](u64 weight) {
        const double goal = u * (double)weight;
        const u64 target = goal > 0.0 ? (goal >= (double)weight ? weight - 1 : (u64)goal) : 0;
        return target >= weight ? weight - 1 : target;
    };
    // weights of the parts of the row, of tokens that are known to be kept
    const int chunk = max(512, ((v + kChunks - 1) / kChunks + 63) & ~63), chunks = (v + chunk - 1) / chunk;
    bool done = false;
    // The list's n tokens, of which the first `most` in the order count and of these the ones before whose weight,
    // with `ahead` of others, stays below want(their weight): added to the parts, the last one is the end of what is kept.
    // Up to kFew tokens, each
    // compares itself with all (n reads of LDS for each), more are sorted: 50 tokens take 3 us less so, 270 take 3 us more.
    // (With `alone` no other token is kept: few ones are drawn from at once, each knows what those of lower number weigh.
    // True if that is done: 3 us less than the way over the parts.)
    auto keep_listed = [&](int n, int most, u64 ahead, auto want_of, bool alone) {
        const int keep = most < n ? most : n;
        const bool few = n <= kFew;
        u64 rank[2] = {0, 0}, x[2] = {0, 0}, sum = 0, all;
        double w[2] = {0.0, 0.0};
        int place = 2 * threadIdx.x;
        if (few) {
            const int me = threadIdx.x;
            if (me < n) {
                rank[0] = list[me];
                w[0] = weigh.real(value_of((unsigned)(rank[0] >> 32)));
                weights[me] = x[0] = weigh.whole(value_of((unsigned)(rank[0] >> 32)));
            } else if (me < n + 8) {
                list[me] = 0;                // (the loop below goes to a multiple of eight)
            }
            __syncthreads();
            if (me < n) {
                place = 0;
                for (int j = 0; j < n; j += 8) {
                    u64 r[8], y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) r[e] = list[j + e], y[e] = weights[j + e];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        sum += r[e] > rank[0] ? y[e] : 0;
                        place += r[e] > rank[0];
                    }
                }
                if (place >= keep) x[0] = 0;
            } else {
                place = keep;
            }
            scan(x[0], lds, all);
        } else {
            sort_down(list, n);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (place + e < keep) {
                    rank[e] = list[place + e];
                    w[e] = weigh.real(value_of((unsigned)(rank[e] >> 32)));
                    x[e] = weigh.whole(value_of((unsigned)(rank[e] >> 32)));
                }
            sum = scan(x[0] + x[1], lds, all);
        }
        const u64 want = want_of(all);
        sum += ahead;
        if (few && alone) {
            const int me = threadIdx.x, number = (int)~(unsigned)rank[0];
            const u64 mine = place < keep && sum < want && w[0] >= min_p ? x[0] : 0;
            if (me < kFew) weights[me] = me < n ? mine : 0;              // (they are read before the scan's barriers)
            __syncthreads();
            if (me >= n) return true;
            u64 below = 0, weight = 0;
            for (int j = 0; j < n; j += 8) {
                u64 r[8], y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = list[j + e], y[e] = weights[j + e];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    weight += y[e];
                    below += (int)~(unsigned)r[e] < number ? y[e] : 0;
                }
            }
            const u64 target = target_of(weight);
            if (below <= target && target < below + mine) p.tokens[b] = number;
            return true;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (few && e) break;
            const bool in = place + e < keep && sum < want;
            sum += x[e];
            if (!in) continue;
            if (sum >= want || place + e == keep - 1) cut_rank = rank[e];
            if (w[e] >= min_p) atomicAdd(&parts[(int)~(unsigned)rank[e] / chunk], x[e]);
        }
        __syncthreads();
        cut = cut_rank;
        done = true;
        return false;
    };
    auto part_of = [&](u64 all) {            // top-p of a weight, at least the first token
        const double goal = top_p * (double)all;
        const u64 want = !cut_p || goal >= (double)all ? all : (u64)ceil(goal);
        return want < 1 ? (u64)1 : want;
    };

    if (counted) {
        const Found f = reach<kCoarse>(counts, [&](u64) { return (u64)k; }, lds, &found);
        const unsigned from = f.bin;
        if (f.before + f.inside <= kList) {
            for (int c = threadIdx.x; c < chunks; c += kDraw) parts[c] = 0;
            // of what is there already, the ones that the whole row's digit leaves; then the tokens not looked at
            const int there = listed;
            const bool ready = there <= kList;
            u64 old[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (ready && (int)threadIdx.x + e * kDraw < there) old[e] = list[threadIdx.x + e * kDraw];
            __syncthreads();
            if (threadIdx.x == 0) listed = 0;
            __syncthreads();
            auto take = [&](u64 r) {
                if (r >> 51 >= from) list[atomicAdd(&listed, 1)] = r;
            };
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (ready && (int)threadIdx.x + e * kDraw < there) take(old[e]);
            each_token(row, 0, ready ? head : v, [&](int i, float x) { take(rank_of(x, i)); });
            __syncthreads();
            if (keep_listed((int)(f.before + f.inside), (int)k, 0, part_of, true)) return;
        }
    }
    if (counted && !done) {
        __syncthreads();
        cut_key = select<true>(row, v, 0, 0, no_key, (u64)k, weigh, coarse, lds, &found, before);
        ties = (u64)k - before;
        by_key = true;
    }
    if (done) {
    } else if (cut_p && !by_key) {
        // The weights by their logarithm in 64ths, of which 2^-s of the largest has less than kCoarse: a step holds few
        // tokens, in the logits' own bits hundreds (sorting those took 8 us of 50)
        auto step_of = [&](const Weigher::Power& t) { return kCoarse - 1 + max(t.k, 1 - kCoarse); };
        for (int i = threadIdx.x; i < kCoarse; i += kDraw) coarse[i] = 0;
        __syncthreads();
        float x[4];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int first = i0 + n * kDraw;
                if (first + kDraw <= v) x[n] = (row + first)[threadIdx.x];
                else x[n] = row[min(first + (int)threadIdx.x, v - 1)];
            }
        };
        fetch(0);
        for (int i0 = 0; i0 < v; i0 += 4 * kDraw) {           // (four at a time: one waits for its own products)
            u64 w[4];
            int at[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const Weigher::Power t = weigh.power(x[n]);
                const u64 whole = weigh.whole_of(t);          // (ahead of the choice: a read of LDS inside it would be a branch)
                w[n] = i0 + n * kDraw + (int)threadIdx.x < v ? whole : 0;
                at[n] = step_of(t);
            }
            if (i0 + 4 * kDraw < v) fetch(i0 + 4 * kDraw);
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (w[n]) atomicAdd(&coarse[at[n]], w[n]);
        }
        __syncthreads();
        u64 want = 0;
        const Found f = reach<kCoarse>(coarse, [&](u64 all) { return want = part_of(all); }, lds, &found);
        // the logits from which on a token's step is at least `step`, as the first key, 64 keys at a time
        auto first_of = [&](int step) {
            u64 base = 0;
            int c = 0;
#pragma unroll
            for (int shift = 26; shift >= -4; shift -= 6) {
                const int by = max(shift, 0);
                const u64 key = base + ((u64)lane << by);
                const bool below = key < top_key && step_of(weigh.power(value_of((unsigned)key))) < step;
                c = __popcll(__ballot(below));
                base += (u64)(shift > 0 && c ? c - 1 : c) << by;
            }
            return max((unsigned)base, key_of(-__builtin_inff()));
        };
        const bool above = (int)f.bin < kCoarse - 1;
        const float from_ending = value_of(first_of((int)f.bin)), from_kept = above ? value_of(first_of((int)f.bin + 1)) : __builtin_nanf("");
        // The tokens of the step in which the beginning ends go to the list, if there is room; those of larger ones are
        // kept: a wave packs them together first, as most are not
        float* mine = (float*)coarse + wave * 512;
        float next[8];
        auto fetch_part = [&](int i0, int end) {         // (past the end NaN, which is neither)
            const float* from = row + i0;
            if (i0 + 512 <= end) {
#pragma unroll
                for (int n = 0; n < 8; ++n) next[n] = from[64 * n + lane];
            } else {
#pragma unroll
                for (int n = 0; n < 8; ++n) next[n] = i0 + 64 * n + lane < end ? from[64 * n + lane] : __builtin_nanf("");
            }
        };
        if (wave < chunks) fetch_part(wave * chunk, min(v, (wave + 1) * chunk));
        for (int c = wave; c < chunks; c += kDraw / 64) {
            u64 sum = 0;
            const int end = min(v, (c + 1) * chunk), after = c + kDraw / 64;
            for (int i0 = c * chunk; i0 < end; i0 += 512) {
                float x[8];
#pragma unroll
                for (int n = 0; n < 8; ++n) x[n] = next[n];
                if (i0 + 512 < end) fetch_part(i0 + 512, end);
                else if (after < chunks) fetch_part(after * chunk, min(v, (after + 1) * chunk));
                u64 ends[8];
                int kept = 0, ending = 0;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const u64 m = __ballot(x[n] >= from_kept);
                    if (x[n] >= from_kept) mine[lanes_before(m, kept)] = x[n];
                    kept += __popcll(m);
                    ends[n] = __ballot(x[n] >= from_ending) & ~m;
                    ending += __popcll(ends[n]);
                }
                __builtin_amdgcn_wave_barrier();
                for (int j = lane; j < kept; j += 64) {
                    sum += weigh.whole_from(mine[j], min_p);
                }
                __builtin_amdgcn_wave_barrier();
                if (!ending) continue;
                int to = 0;
                if (lane == 0) to = atomicAdd(&listed, ending);
                to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    const int k = lanes_before(ends[n], to);
                    if (ends[n] >> lane & 1 && k < kList) list[k] = rank_of(x[n], i0 + 64 * n + lane);
                    to += __popcll(ends[n]);
                }
            }
            sum = wave_sum(sum);
            if (lane == 0) parts[c] = sum;
        }
        __syncthreads();
        const int n = listed;
        __syncthreads();
        if (n <= kList) {
            if (keep_listed(n, n, f.before, [&](u64) { return want; }, f.before == 0)) return;
        } else {
            cut_key = select<false>(row, v, 0, 0, no_key, want, weigh, coarse, lds, &found, before);
            const u64 each = weigh.whole(value_of(cut_key));
            ties = each ? (want - before + each - 1) / each : 1;
            by_key = true;
        }
    } else if (cut_p) {
        // the part p of the weight of the top-k beginning, which may end among its last, equal tokens
        u64 sum = 0, weight;
        for (int i = threadIdx.x; i < v; i += kDraw) {
            const float x = row[i];
            if (key_of(x) > cut_key) sum += weigh.whole(x);
        }
        scan(sum, lds, weight);
        weight += ties * weigh.whole(value_of(cut_key));
        const u64 want = part_of(weight);
        const unsigned end = select<false>(row, v, cut_key, ties, cut_key, want, weigh, coarse, lds, &found, before);
        const u64 each = weigh.whole(value_of(end));
        u64 n = each ? (want - before + each - 1) / each : 1;
        if (end == cut_key && n > ties) n = ties;
        cut_key = end;
        ties = n;
    }

    if (!done)
        for (int c = wave; c < chunks; c += kDraw / 64) {
            u64 sum = 0;
            unsigned tied = 0;
            if (by_key)
                each_of_part(row, c * chunk, min(v, (c + 1) * chunk), [&](float x) {
                    const unsigned key = key_of(x);
                    if (key < cut_key) return;
                    if (key > cut_key) sum += weigh.whole_from(x, min_p);
                    else if (x == x && weigh.real(x) >= min_p) ++tied;
                });
            else
                each_of_part(row, c * chunk, min(v, (c + 1) * chunk), [&](float x) {
                    sum += weigh.whole_from(x, min_p);
                });
            sum = wave_sum(sum);
            if (by_key) tied = wave_sum(tied);
            if (lane == 0) parts[c] = sum, marks[c] = tied;
        }
    __syncthreads();
    // the part and the token in which the draw falls
    const u64 each = by_key ? weigh.whole(value_of(cut_key)) : 0;
    const int c0 = 2 * threadIdx.x;
    unsigned t0 = 0, t1 = 0;
    u64 every, tied_before = 0;
    if (by_key) {
        if (c0 < chunks) t0 = marks[c0];
        if (c0 + 1 < chunks) t1 = marks[c0 + 1];
        tied_before = scan(t0 + t1, lds, every);
    }
    auto kept = [&](u64 from, u64 count) { return from >= ties ? 0 : (ties - from < count ? ties - from : count); };
    const u64 w0 = c0 < chunks ? parts[c0] + each * kept(tied_before, t0) : 0;
    const u64 w1 = c0 + 1 < chunks ? parts[c0 + 1] + each * kept(tied_before + t0, t1) : 0;
    u64 weight;
    const u64 weight_before = scan(w0 + w1, lds, weight);
    const u64 target = target_of(weight);
    if (weight_before <= target && target < weight_before + w0) chunk_at = c0, chunk_before = weight_before, chunk_tied = tied_before;
    if (weight_before + w0 <= target && target < weight_before + w0 + w1) chunk_at = c0 + 1, chunk_before = weight_before + w0, chunk_tied = tied_before + t0;
    __syncthreads();
    if (wave) return;
    u64 sum = chunk_before, tied = chunk_tied;
    int token = -1;
    const int first = chunk_at * chunk, end = min(v, first + chunk);
    for (int i1 = first; i1 < end && token < 0; i1 += 512) {
        float x[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) x[n] = row[min(i1 + 64 * n + lane, end - 1)];
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int i = i1 + 64 * n + lane;
            const unsigned key = key_of(x[n]);
            const double w = weigh.real(x[n]);
            bool in = i < end && (by_key ? key >= cut_key : rank_of(x[n], i) >= cut) && w >= min_p;
            const bool tie = in && by_key && key == cut_key;
            const u64 m = __ballot(tie);
            if (tie) in = tied + __popcll(m & ((1ull << lane) - 1)) < ties;
            tied += __popcll(m);
            const u64 run = wave_scan(in ? weigh.whole(x[n]) : 0);
            const u64 past = __ballot(sum + run > target);
            if (past && token < 0) token = i1 + 64 * n + __builtin_ctzll(past);
            sum += of_lane(run, 63);
        }
    }
    if (lane == 0) p.tokens[b] = token < 0 ? first : token;       // (one is always found: target < weight)
}

}  // namespace

extern "C" uint64_t drhip_k_rotary_work(const drhip_rotary_t* p) {
    if (!p->dweight) return 0;
    return (uint64_t)grad_slots(*p) * p->heads * p->d_pad * (p->is_double ? 8 : 4);
}

extern "C" int64_t drhip_k_rotary_blocks(const drhip_rotary_t* p) { return rotary_blocks(*p); }

extern "C" int drhip_k_rotary(const drhip_rotary_t* p, hipStream_t s) {
    if (p->dweight)
        p->is_double ? launch_rotary_grad<double>(*p, s) : launch_rotary_grad<float>(*p, s);
    else
        p->is_double ? launch_rotary<double>(*p, s) : launch_rotary<float>(*p, s);
    return (int)hipGetLastError();
}

extern "C" int drhip_k_sample(const drhip_sample_t* p, hipStream_t s) {
    sample_kernel<<<p->batch, kDraw, 0, s>>>(*p);
    return (int)hipGetLastError();
}
