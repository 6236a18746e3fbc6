// Attention on gfx950: forward (many and few rows), joining of split key ranges, and the gradient.
// Interface: drhip_attention_t in include/drhip.h.
//
//   x_ij = scale q_i . k_j            z_ij = cap tanh(x_ij / cap) - slope_h |p_i - j|
//   o_i  = sum_j P_ij v_j,  P_ij = exp(z_ij - lse_i),  lse_i = log sum_j exp z_ij
//   dV_j = sum_i P_ij dO_i            D_i = dO_i . o_i
//   dX_ij = P_ij (dO_i . v_j - D_i) (1 - tanh^2(x_ij / cap))
//   dQ_i = scale sum_j dX_ij k_j      dK_j = scale sum_i dX_ij q_i
//
// Sums run over the pairs that count: j below the row's limit (the sequence's length; for causal
// rows max(p_i + 1, prefix) as well) and, with documents, of the row's own document.  A row
// without pairs gives zeros and lse = -inf.  A pair that does not count contributes nothing
// whatever its key holds: tiles are freed of values that are not finite when they are packed or loaded,
// and the rows that held one are added by themselves, where their weight is not zero.
//
// Operands, sums and the statistics of the softmax are float32.  Many rows and the gradient are bound by the matrix
// units and compute each float32 product as six bfloat16 ones (below); few rows are bound by memory and use
// v_mfma_f32_16x16x4f32.
#include "../../include/drhip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef drhip_attention_t Args;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr int kThreads = 256;        // 4 waves
constexpr int kRows = 128;           // query rows (or keys, in the dK/dV kernel) of a block: 32 for each wave
constexpr int kTile = 32;            // keys (query rows) staged at a time

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh to about an ulp: an odd polynomial (own fit on |y| <= 0.55, relative error 4.4e-9) where
// 1 - 2 / (e^2y + 1) would cancel, that form elsewhere
constexpr float kSmall = 0.55f;

__device__ __forceinline__ float tanh_small(float y) {
    const float u = y * y;
    const float p = fmaf(u, fmaf(u, fmaf(u, fmaf(u, -0.0062742396257817745f, 0.021071678027510643f),
                                         -0.05385230854153633f), 0.13332585990428925f), -0.33333316445350647f);
    return fmaf(y * u, p, y);
}

__device__ __forceinline__ float tanh_(float y) {
    const float a = fabsf(y);
    const float large = copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(exp2_(a * (2.0f * kLog2e)) + 1.0f), y);
    return a <= kSmall ? tanh_small(y) : (a == a ? large : y);
}

__device__ __forceinline__ bool finite_(float x) { return fabsf(x) < __builtin_inff(); }

__device__ __forceinline__ int clamp_(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Four neighbouring elements of a row, zeros past its end; `wide`: rows are 16-byte aligned multiples of four
__device__ __forceinline__ f32x4 load4(const float* row, int d, int size, bool ok, bool wide) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (wide) {
        if (ok && d < size) x = *(const f32x4*)(row + d);
    } else if (ok) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (d + c < size) x[c] = row[d + c];
    }
    return x;
}

// What a sequence says about its rows
struct Seq {
    int len, start, prefix;
    const int32_t* docs;
};

__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.len = a.lengths ? clamp_(a.lengths[b], 0, a.lk) : a.lk;
    const int far = 1 << 30;      // positions stay far from the ends of int32
    s.start = a.start ? clamp_(a.start[b], -far, far) : a.start_mode ? clamp_(a.start_value, -far, far) : s.len - a.lq;
    s.prefix = a.prefix ? clamp_(a.prefix[b], 0, a.lk) : a.prefix_value;
    s.docs = a.documents ? a.documents + (int64_t)b * a.documents_stride : nullptr;
    return s;
}

// The keys that the row at position p may see are those below its limit, of its own document
__device__ __forceinline__ int row_limit(const Args& a, const Seq& s, int p) {
    int lim = s.len;
    if (a.causal) {
        const int seen = p + 1 > s.prefix ? p + 1 : s.prefix;
        lim = clamp_(seen, 0, s.len);
    }
    if (s.docs && (p < 0 || p >= s.len)) lim = 0;      // a row without a document
    return lim;
}

// Row of register v in a 32x32 accumulator, for the lanes of half h
__device__ __forceinline__ int acc_row(int v, int h) { return 8 * (v >> 2) + 4 * h + (v & 3); }

// Score of one pair from its product, in units of log 2, and the factor of its derivative
__device__ __forceinline__ float score(const Args& a, float x, float slope2, int p, int j) {
    float z;
    if (a.cap > 0.f)
        z = a.cap * kLog2e * tanh_(x / a.cap);
    else
        z = x * kLog2e;
    if (a.slopes) z -= slope2 * fabsf((float)(p - j));
    return z;
}


// How the rows of a key head's gradient are spread over blocks: `count` parts, (query heads) x `ranges` of `span` rows
struct Parts {
    int count, ranges, span;
};

struct Plan {
    int few;             // the kernel for few rows
    int waves;           // of a block of the other one
    int splits, chunk;   // key ranges, and keys in one
    int wide;            // rows can be read and written 16 bytes at a time
};

// ---- float32 products on bfloat16 matrix instructions ------------------------------------------
// v_mfma_f32_32x32x16_bf16 does sixteen times the work of v_mfma_f32_32x32x2_f32 in half its cycles.  A
// float32 number is the sum of three bfloat16 (8 bits each, rounded to nearest, the differences exact):
// x = h + m + l up to 2^-27 |x|.  Of the nine products of two such sums the six largest are added, small
// ones first; the others are below 2^-26 of the product, a quarter of float32's own rounding.  So the result is
// that of float32 arithmetic at 16 x 2 / 6 = 2.7 times its rate.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct Three {
    bf16x8 p[3];
};

// (numbers past bfloat16's largest would round to infinity)
__device__ __forceinline__ float in_range(float x) { return __builtin_amdgcn_fmed3f(x, -3.3895313892515355e38f, 3.3895313892515355e38f); }

// With FULL x may be any finite number (one past bfloat16's largest is that and the rest); a NaN or an infinity has a NaN
// among its parts
template <bool FULL = false> __device__ __forceinline__ void split2(f32x2 x, int at, Three& out) {
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const bf16x2 y = __builtin_convertvector(FULL && n == 0 ? f32x2{in_range(x[0]), in_range(x[1])} : x, bf16x2);
        out.p[n][at] = y[0], out.p[n][at + 1] = y[1];
        if (n < 2) x = x - __builtin_convertvector(y, f32x2);
    }
}

__device__ __forceinline__ f32x16 mac6(const Three& a, const Three& b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// A 32-row tile in three planes: [plane][element / 8][row][element % 8], 16-byte chunks of eight elements of a
// row, whose bits 2 and 3 are turned by the chunk's number.  A product contracts over elements (row_chunk: a lane
// takes a chunk of its row, consecutive lanes consecutive chunks) or over rows (column_chunk: a lane takes
// eight rows of its element with transposing reads, of which 32 lanes read four rows of four chunks; the turned
// bits put these into different banks).  The eight rows are those that a lane half holds in eight registers
// of an accumulator (acc_row), so that weights go from one product to the next without a move.
template <int NT> struct Planes {
    static constexpr int PLANE = 2 * 32 * 32 * NT;    // bytes
    static constexpr int BYTES = 3 * PLANE;           // of a tile
    __device__ __forceinline__ static int place(int row, int chunk) { return (chunk * 32 + (row ^ 4 * (chunk & 3))) * 16; }
    __device__ __forceinline__ static Three row_chunk(const char* tile, int row, int t, int h) {
        Three x;
        const char* at = tile + place(row, h + 2 * (t & 1)) + 2048 * (t / 2);
#pragma unroll
        for (int n = 0; n < 3; ++n) x.p[n] = *(const bf16x8*)(at + n * PLANE);
        return x;
    }
    // element 32 c + lane % 32, rows acc_row(8u .. 8u + 7, lane / 32)
    __device__ __forceinline__ static Three column_chunk(const char* tile, int u, int c, int lane) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const int l = lane & 15, chunk = 2 * (lane >> 4 & 1) + (l >> 1 & 1);
        const char* at = tile + place(4 * (lane >> 5) + (l >> 2), chunk) + (l & 1) * 8 + 2048 * c + 256 * u;
        const int other = place(8 + 4 * (lane >> 5) + (l >> 2), chunk) - place(4 * (lane >> 5) + (l >> 2), chunk);
        Three x;
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + n * PLANE));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + other + n * PLANE));
            x.p[n] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return x;
    }
};

// Nothing is moved across the end of a step of six matrix instructions, which has the chunks of the next
// one on their way from LDS: 24 registers of chunks at a time.  Left to the compiler's own order the loads of
// a whole tile come first, and what they displace goes to scratch memory, whose waits are also waits for the
// next tile's copies.
__device__ __forceinline__ void step_ends() { __builtin_amdgcn_sched_barrier(0); }

// MIX: the order within a step is reads of LDS, then matrix instructions with vector instructions behind each, which
// run while it does (a matrix instruction that waits for the one before it holds up all that come after).  For
// kernels with one wave on each SIMD; two waves fill each other's gaps, and the order costs registers.
template <int READS> __device__ __forceinline__ void mix_step() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int n = 0; n < 6; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 7, 0);
    }
}

// tanh(x * by); scores are mostly small against their cap, and then a third of the work is enough
__device__ __forceinline__ void tanh_tile(f32x16& x, float by) {
    float most = 0.f;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        x[v] *= by;
        most = fmaxf(most, fabsf(x[v]));
    }
    if (__any(most > kSmall)) {             // (a NaN stays one either way)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            x[v] = tanh_(x[v]);
            if (v & 1) step_ends();
        }
    } else {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            x[v] = tanh_small(x[v]);
            if (v & 1) step_ends();
        }
    }
}

struct Nothing {
    __device__ __forceinline__ void operator()(int) const {}
};

// acc[row][col] = sum_d tile[row][d] own[col][d]: lane l holds elements 16t + 8h .. + 7 of column l % 32.
// between(t) is vector work that step t's matrix instructions hide (here and below).
template <int NT, bool MIX, typename F = Nothing>
__device__ __forceinline__ f32x16 product6(const char* tile, const Three (&own)[2 * NT], int lane, F between = F()) {
    f32x16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.f;
    const int h = lane >> 5, row = lane & 31;
    Three x = Planes<NT>::row_chunk(tile, row, 0, h);
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) {
        Three y = x;
        if (t + 1 < 2 * NT) y = Planes<NT>::row_chunk(tile, row, t + 1, h);
        acc = mac6(x, own[t], acc);
        between(t);
        x = y;
        if (MIX) mix_step<3>();
        step_ends();
    }
    return acc;
}

__device__ __forceinline__ Three split8(const f32x16& w, int from) {
    Three x;
#pragma unroll
    for (int e = 0; e < 8; e += 2) split2(f32x2{w[from + e], w[from + e + 1]}, e, x);
    return x;
}

// acc[c][i][col] += sum_row tile[row][32 c + i] w[row][col]; `lo`: the first eight registers of w, split.
// The others are split between the products of those, then comes between(c).
template <int NT, bool MIX, typename F = Nothing>
__device__ __forceinline__ void spread6(f32x16 (&acc)[NT], const char* tile, const Three& lo, const f32x16& w, int lane, F between = F()) {
    Three x = Planes<NT>::column_chunk(tile, 0, 0, lane), hi;
    step_ends();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            Three y = x;
            if (c + 1 < NT) y = Planes<NT>::column_chunk(tile, u, c + 1, lane);
            else if (u == 0) y = Planes<NT>::column_chunk(tile, 1, 0, lane);
            if (u == 0) {
#pragma unroll
                for (int e = 8 * c / NT; e < 8 * (c + 1) / NT; ++e)
                    if (e % 2 == 0) split2(f32x2{w[8 + e], w[9 + e]}, e, hi);
            } else {
                between(c);
            }
            acc[c] = mac6(x, u == 0 ? lo : hi, acc[c]);
            x = y;
            if (MIX) mix_step<6>();
            step_ends();
        }
}

template <int NT>
__device__ void spread6_bad(f32x16 (&acc)[NT], unsigned bad, const float* base, int64_t stride, int size, const f32x16& w, int lane) {
    while (bad) {
        int h = lane >> 5;
        asm volatile("" : "+v"(h));      // (nothing of this rare path is computed ahead of it and kept in registers)
        const int r = __builtin_ctz(bad);
        bad &= bad - 1;
        const int from = 4 * (r >> 3) + (r & 3);
        float mine = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) mine = v == from ? w[v] : mine;
        const float weight = __shfl(mine, (lane & 31) + 32 * ((r >> 2) & 1));
        const float* row = base + r * stride;
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int d = 32 * c + acc_row(v, h);
                const float x = row[d < size ? d : 0], y = weight * x;
                acc[c][v] += !finite_(x) && d < size && weight != 0.f ? y : 0.f;
                if (v % 2) step_ends();
            }
    }
}

// The same where there are no registers to spare: the elements of a lane's column that become NaN are kept as bits
template <int NT>
__device__ void note_bad(unsigned (*poison)[NT], unsigned bad, const float* base, int64_t stride, int size, const f32x16& w, int lane) {
    while (bad) {
        const int r = __builtin_ctz(bad);
        bad &= bad - 1;
        const int from = 4 * (r >> 3) + (r & 3);
        float mine = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) mine = v == from ? w[v] : mine;
        const float weight = __shfl(mine, (lane & 31) + 32 * ((r >> 2) & 1));
        const float* row = base + r * stride;
        if (weight != 0.f && lane < 32)
            for (int d = 0; d < size; ++d)
                if (!finite_(row[d])) poison[lane][d >> 5] |= 1u << (d & 31);
    }
}

template <int NT>
__device__ __forceinline__ void store_column(float* row, const f32x16 (&acc)[NT], float by, int size, bool wide, int h) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = 32 * c + 8 * u + 4 * h;
            if (wide) {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[c][4 * u + e] * by;
                if (d < size) *(f32x4*)(row + d) = x;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < size) row[d + e] = acc[c][4 * u + e] * by;
            }
        }
}

// One matrix to be packed: keys and values up to their sequence's length, or q and dO, of which a row
// without pairs counts as zeros.  With dO goes D = rowsum(dO o).
struct Pack {
    const float* x;
    int64_t stride[3];
    int heads, tiles, keys;         // tiles of 32 rows of one head
    char* planes;
    unsigned* marks;
    int2* docs;                     // least and largest document of a tile
    float* delta;
};
struct Packs {
    Pack job[4];
};

// Matrices in planes, for every tile that counts; values that are not finite become zeros and their rows
// are marked; with documents, their range in the tile is noted.  Bound by memory: 4 bytes read and 6 written for each
// number, once for all blocks that read the tile (8 heads of 4096 keys and values of 128: 84 MB in 15 us; with
// q and dO of 32 heads of 2048 rows and 8 of keys 243 MB in 41 us, 5.9 TB/s).
template <int NT> __global__ __launch_bounds__(kThreads) void attention_pack(Args a, Packs packs, int wide) {
    __shared__ float lds[kTile][32 * NT + 1];
    __shared__ unsigned bad;
    int id = blockIdx.x, n = 0;
    while (id >= a.batch * packs.job[n].heads * packs.job[n].tiles) {
        id -= a.batch * packs.job[n].heads * packs.job[n].tiles;
        ++n;
    }
    const Pack& job = packs.job[n];
    const int tile = id % job.tiles, head = id / job.tiles;
    const int b = head / job.heads, nh = head % job.heads;
    const int first = tile * kTile;
    const int end = job.keys ? sequence(a, b).len : a.lq;
    if (first >= end) return;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const float* base = job.x + b * job.stride[0] + nh * job.stride[1];
    const float* lse = job.keys ? nullptr : a.lse + (int64_t)head * a.lq;
#pragma unroll
    for (int p = 0; p < NT; ++p) {
        const int at = threadIdx.x + p * kThreads, row = at / (8 * NT), d = at % (8 * NT) * 4, i = first + row;
        const bool in = i < end && !(lse && lse[i] == -__builtin_inff());
        const f32x4 x = load4(base + i * job.stride[2], d, a.d, in, wide);
        bool fine = true;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            fine = fine && finite_(x[c]);
            lds[row][d + c] = finite_(x[c]) ? x[c] : 0.f;
        }
        if (!fine) atomicOr(&bad, 1u << row);
    }
    __syncthreads();
    const int64_t place = (int64_t)head * job.tiles + tile;
    if (threadIdx.x == 0) job.marks[place] = bad;
    if (job.docs && threadIdx.x < 64) {
        const Seq s = sequence(a, b);
        const int i = first + (threadIdx.x & 31), j = job.keys ? i : s.start + i;
        const bool in = i < end && j >= 0 && j < s.len;
        int lo = in ? s.docs[j] : 0x7fffffff, hi = in ? lo : -0x7fffffff - 1;
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
            lo = min(lo, __shfl_xor(lo, m));
            hi = max(hi, __shfl_xor(hi, m));
        }
        if (threadIdx.x == 0) job.docs[place] = make_int2(lo, hi);
    }
    char* to = job.planes + place * Planes<NT>::BYTES;
    for (int at = threadIdx.x; at < 32 * 4 * NT; at += kThreads) {
        Three x;
        const int row = at & 31, chunk = at >> 5;
#pragma unroll
        for (int e = 0; e < 8; e += 2) split2<true>(f32x2{lds[row][8 * chunk + e], lds[row][8 * chunk + e + 1]}, e, x);
#pragma unroll
        for (int k = 0; k < 3; ++k) *(bf16x8*)(to + k * Planes<NT>::PLANE + Planes<NT>::place(row, chunk)) = x.p[k];
    }
    if (job.delta) {                      // eight lanes for each row
        const int row = threadIdx.x >> 3, i = first + row;
        const bool in = i < end && lse[i] != -__builtin_inff();
        const float* orow = a.o + b * a.o_stride[0] + nh * a.o_stride[1] + i * a.o_stride[2];
        float sum = 0.f;
        for (int d = 4 * (threadIdx.x & 7); d < a.d; d += 32) {
            const f32x4 y = load4(orow, d, a.d, in, wide);
#pragma unroll
            for (int c = 0; c < 4; ++c) sum = fmaf(lds[row][d + c], y[c], sum);
        }
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) sum += __shfl_xor(sum, m);
        if ((threadIdx.x & 7) == 0 && i < end) job.delta[(int64_t)head * a.lq + i] = sum;
    }
}

// `bytes` (a multiple of 1024) from memory to LDS without a register between, by the block's waves in turn.
// As instructions that the compiler does not know for writes to LDS: it would wait for them ahead of the next
// read of LDS, though that is one of the other buffer.  They have no result in registers; copies_done() and a
// barrier stand before the first read of what they write.  (m0 is the compiler's own register, which these kernels
// use for nothing else.)
// The address is a base in scalar registers and 16 bytes for each lane, so that a copy costs no vector instructions
// (the wait states are those between a vector instruction that writes a scalar register and a load that reads it).
template <int WAVES, int BYTES> __device__ __forceinline__ void copy_to_lds(char* lds, const char* from) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
    const uint64_t base = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)from >> 32)) << 32 |
                          (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)from);
#pragma unroll
    for (int n = 0; n < (BYTES / 1024 + WAVES - 1) / WAVES; ++n) {
        const int at = (n * WAVES + wave) * 1024;
        if (at < BYTES)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + at), "v"(lane * 16), "s"(base + at) : "memory");
    }
}

__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Whether the tile's documents (one in each of 32 lanes, `range`: least and largest) are the lane's own, as bits in the
// order of the accumulator's registers
__device__ __forceinline__ unsigned same_document(int docs, int2 range, int doc, int h) {
    if (range.x == range.y) return range.x == doc ? ~0u : 0u;
    unsigned m = 0;
    asm volatile("" : "+v"(h));              // (no sixteen addresses computed ahead and kept)
#pragma unroll
    for (int v = 0; v < 16; ++v) m |= (__shfl(docs, acc_row(v, 0) + 4 * h) == doc ? 1u : 0u) << v;
    return m;
}

// What the kernels read of the packed matrices
struct Packed {
    const char *key, *value, *query, *grad;
    const unsigned *key_marks, *value_marks, *query_marks, *grad_marks;
    const int2 *key_docs, *query_docs;
    float* delta;
};

// The next of `count` tiles from t on that may hold a document in [lo, hi], 64 tiles at a look
struct Active {
    const int2* ranges;
    int count, lo, hi, group;
    unsigned long long mask;
    int2 ours;
    __device__ __forceinline__ int next(int t) {
        while (t < count) {
            if (t >> 6 != group) {
                group = t >> 6;
                const int mine = (group << 6) + (threadIdx.x & 63);
                ours = ranges[mine < count ? mine : 0];
                mask = __ballot(mine < count && ours.x <= hi && ours.y >= lo);
            }
            const unsigned long long left = mask >> (t & 63);
            if (left) return t + __builtin_ctzll(left);
            t = (group + 1) << 6;
        }
        return count;
    }
    // least and largest document of a tile that next() gave last
    __device__ __forceinline__ int2 range(int t) const {
        return make_int2(__builtin_amdgcn_readlane(ours.x, t & 63), __builtin_amdgcn_readlane(ours.y, t & 63));
    }
};

// ---- forward, many rows ---------------------------------------------------------------------
// A block owns 32 WAVES rows of the queries that share a key head (query positions one after the other, the
// heads of a position together, so that the rows of a block see nearly the same keys), each wave 32 of them, one
// per column of its accumulators: S^T = K Q^T leaves the scores of a row in one lane pair, so the softmax
// needs one exchange, and P^T in the layout that O^T += V^T P^T reads.
// Keys and values come 32 at a time from the packed planes through LDS, two buffers, copied a tile ahead.
// Bound by the matrix units: 32 heads, 4096 rows of 128, causal: 651 us at best and 690 at the median under the profiler,
// 199 TFLOP/s of float32 products (a large product of f32 matrices reaches 155), 1.2 PFLOP/s of bfloat16 ones, of which a
// loop of nothing else reaches 2.1 to 2.25.  Two waves on a SIMD fill each other's waits; four-wave blocks, two on a
// compute unit, read each tile twice as often from L2 (695 for 639 us).  With a cap a tanh for each pair comes on top (8
// heads, 8192 rows: 695 and 711 us).
template <int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NT < 4 ? 2 : WAVES / 4) void attention_rows(Args a, Plan plan, int tiles, Packed in, float* part, float* part_lse) {
    using P = Planes<NT>;
    __shared__ __attribute__((aligned(16))) char lds[2][2 * P::BYTES];
    __shared__ int ends[WAVES], doc_range[2][WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int heads = a.batch * a.hkv;
    int id = blockIdx.x;
    const int head = id % heads;
    id /= heads;
    // The longest rows first, range by range: blocks go to the shader engines in turn, so that ranges of one tile
    // next to each other would give all first ranges, the long ones, to half of them (1.7 times the time)
    const int tile = tiles - 1 - id % tiles, split = id / tiles;
    const int b = head / a.hkv, kh = head % a.hkv, group = a.hq / a.hkv;
    const Seq s = sequence(a, b);
    const bool wide = plan.wide;

    const int rows = group * a.lq;
    const int r = (tile * WAVES + wave) * 32 + (lane & 31);
    const bool valid = r < rows;
    const int i = valid ? r / group : 0, g = valid ? r - i * group : 0;
    const int qh = kh * group + g, p = s.start + i;
    const int lim = valid ? row_limit(a, s, p) : 0;
    const int doc = s.docs && lim > 0 ? s.docs[p] : 0;
    const float slope2 = a.slopes ? a.slopes[qh] * kLog2e : 0.f;

    // scores come out in units of log 2, or with a cap as they are
    const float scale = a.cap > 0.f ? a.scale : a.scale * kLog2e;
    Three own[2 * NT];
    const float* qrow = a.q + b * a.q_stride[0] + qh * a.q_stride[1] + i * a.q_stride[2];
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4 x = load4(qrow, 16 * t + 8 * h + e, a.d, valid, wide) * scale;
            split2<true>(f32x2{x[0], x[1]}, e, own[t]);
            split2<true>(f32x2{x[2], x[3]}, e + 2, own[t]);
        }
    }

    // range of limits (and documents) in the wave and in the block
    int top = lim, low = valid ? lim : 0x7fffffff, dlo = lim > 0 ? doc : 0x7fffffff, dhi = lim > 0 ? doc : -0x7fffffff - 1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        top = max(top, __shfl_xor(top, m));
        low = min(low, __shfl_xor(low, m));
        dlo = min(dlo, __shfl_xor(dlo, m));
        dhi = max(dhi, __shfl_xor(dhi, m));
    }
    if (lane == 0) ends[wave] = top, doc_range[0][wave] = dlo, doc_range[1][wave] = dhi;
    __syncthreads();
    const int begin = split * plan.chunk;
    int end = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        end = max(end, ends[w]);
        dlo = min(dlo, doc_range[0][w]);
        dhi = max(dhi, doc_range[1][w]);
    }
    end = __builtin_amdgcn_readfirstlane(min(end, begin + plan.chunk));
    top = __builtin_amdgcn_readfirstlane(top);
    low = __builtin_amdgcn_readfirstlane(low);

    int docs_next = 0;
    int2 range_next = {0, 0};
    // the first key of the next tile that any row of the block may see
    const int key_tiles = (a.lk + kTile - 1) / kTile;
    const int64_t place = (int64_t)head * key_tiles;
    Active active{in.key_docs + place, (end + kTile - 1) / kTile, dlo, dhi, -1, 0, {0, 0}};
    auto next = [&](int j0) {
        if (!s.docs) return j0;
        return __builtin_amdgcn_readfirstlane(active.next(j0 / kTile)) * kTile;
    };
    unsigned marks_next[2] = {0, 0};
    auto copy = [&](int to, int j) {                  // (marks are read ahead of the copies: a wait for them would wait for these)
        marks_next[0] = in.key_marks[place + j / kTile];
        marks_next[1] = in.value_marks[place + j / kTile];
        if (s.docs) docs_next = s.docs[min(j + (lane & 31), s.len - 1)], range_next = active.range(j / kTile);
        copy_to_lds<WAVES, P::BYTES>(lds[to], in.key + (place + j / kTile) * P::BYTES);
        copy_to_lds<WAVES, P::BYTES>(lds[to] + P::BYTES, in.value + (place + j / kTile) * P::BYTES);
    };

    f32x16 acc[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[c][v] = 0.f;
    float most = -__builtin_inff(), total = 0.f;      // running maximum of the row, sum over this lane's keys

    int j0 = next(begin), buf = 0;
    if (j0 < end) copy(0, j0);
    while (j0 < end) {
        copies_done();
        __syncthreads();                               // this tile is there, and everyone is done with the other buffer
        const int docs = docs_next;
        const int2 range = range_next;
        const unsigned kbad = __builtin_amdgcn_readfirstlane(marks_next[0]), vbad = __builtin_amdgcn_readfirstlane(marks_next[1]);
        const int j1 = next(j0 + kTile);
        if (j1 < end) copy(buf ^ 1, j1);
        if (j0 < top) {                                // some row of this wave sees the tile
            f32x16 x = product6<NT, false>(lds[buf], own, lane);
            if (a.cap > 0.f) {
                tanh_tile(x, 1.f / a.cap);
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] *= a.cap * kLog2e;
            }
            if (a.slopes) {
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] -= slope2 * fabsf((float)(p - j0 - 4 * h - acc_row(v, 0)));
            }
            if (j0 + kTile > low || s.docs || kbad) {
                const unsigned same = s.docs ? same_document(docs, range, doc, h) : ~0u;
                const unsigned nans = kbad >> 4 * h;
                const int left = lim - j0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const bool ok = acc_row(v, 0) < left && (same >> v & 1);
                    x[v] = nans >> acc_row(v, 0) & 1 ? __builtin_nanf("") : x[v];
                    x[v] = ok ? x[v] : -__builtin_inff();
                }
            }
            float peak = most;
#pragma unroll
            for (int v = 0; v < 16; ++v) peak = fmaxf(peak, x[v]);          // (a NaN shows in the sum)
            peak = fmaxf(peak, __shfl_xor(peak, 32));
            const float ref = peak == -__builtin_inff() ? 0.f : peak;
            const float shrink = exp2_(most - ref);
            if (__any(shrink != 1.f)) {
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[c][v] *= shrink;
                total *= shrink;
            }
            most = peak;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[v] = exp2_(x[v] - ref);
                total += x[v];
            }
            spread6<NT, false>(acc, lds[buf] + P::BYTES, split8(x, 0), x, lane);
            if (vbad)
                spread6_bad<NT>(acc, vbad, a.v + b * a.v_stride[0] + kh * a.v_stride[1] + j0 * a.v_stride[2], a.v_stride[2], a.d, x, lane);
        }
        buf ^= 1;
        j0 = j1;
    }

    total += __shfl_xor(total, 32);
    if (!valid) return;
    const float by = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;      // (a NaN stays one)
    const float lse = total == 0.f ? -__builtin_inff() : (most + __builtin_amdgcn_logf(total)) * kLn2;
    if (split && lim <= plan.chunk) return;              // (the first range has all of the row's keys)
    if (part && lim > plan.chunk) {
        const int64_t row = (((int64_t)split * a.batch + b) * a.hq + qh) * a.lq + i;
        if (total != 0.f) store_column<NT>(part + row * a.d, acc, by, a.d, wide, h);     // (the join reads no others)
        if (h == 0) part_lse[row] = lse;
    } else {
        store_column<NT>(a.o + b * a.o_stride[0] + qh * a.o_stride[1] + i * a.o_stride[2], acc, by, a.d, wide, h);
        if (h == 0 && a.lse) a.lse[((int64_t)b * a.hq + qh) * a.lq + i] = lse;
    }
}

// ---- forward, few rows ----------------------------------------------------------------------
// Single tokens, with all query heads of a key head together, and small calls: 16 rows to a block, against a
// long key range bound by reading keys and values once.  No LDS: a wave takes 16 keys at a time, the blocks'
// waves in turn, and its loads are the operands of v_mfma_f32_16x16x4f32 as they come (K: lane = key,
// 16 bytes of its row; V: 16 neighbouring bytes of four rows each).  Key ranges of one sequence go to
// `splits` blocks, whose results are joined by `attention_join`.  64 sequences of up to 8192 keys, 8 key heads of
// 128: 451 us, 5.8 TB/s.  One sequence of 5000: 17 us, a third of it the blocks' start, a quarter the first
// load's way.
template <int NB, bool WIDE>
__global__ __launch_bounds__(kThreads, 2) void attention_few(Args a, Plan plan, int sets, float* part, float* part_lse) {
    constexpr int KS = 4 * NB;                 // 16-byte steps of a key row for each quarter of the wave
    __shared__ __attribute__((aligned(16))) float merged[4][16][64 * NB + 4];
    __shared__ float stat[4][2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, h = lane >> 4;
    const int heads = a.batch * a.hkv;
    int id = blockIdx.x;
    const int head = id % heads;
    id /= heads;
    const int set = id % sets, split = id / sets;          // (sets of one range together: the others find its keys in L2)
    const int b = head / a.hkv, kh = head % a.hkv, group = a.hq / a.hkv;
    const Seq s = sequence(a, b);
    constexpr bool wide = WIDE;       // (apart, for the size of the code: short calls wait for it)
    const int rows = group * a.lq;

    const int row = 16 * set + col;
    const bool valid = row < rows;
    const int g = valid ? row / a.lq : 0, i = valid ? row - g * a.lq : 0, qh = kh * group + g;
    const int pos = s.start + i, lim = valid ? row_limit(a, s, pos) : 0;
    const int doc = s.docs && lim > 0 ? s.docs[pos] : 0;
    const float slope2 = a.slopes ? a.slopes[qh] * kLog2e : 0.f;
    const float* qrow = a.q + b * a.q_stride[0] + qh * a.q_stride[1] + i * a.q_stride[2];
    f32x4 own[KS];
#pragma unroll
    for (int t = 0; t < KS; ++t) {
        own[t] = load4(qrow, 16 * t + 4 * h, a.d, valid, wide) * a.scale;
#pragma unroll
        for (int c = 0; c < 4; ++c) own[t][c] = finite_(own[t][c]) ? own[t][c] : __builtin_nanf("");      // (an infinity could give -inf, a pair without weight)
    }
    int top = lim, low = valid ? lim : 0x7fffffff;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) {
        top = max(top, __shfl_xor(top, m));
        low = min(low, __shfl_xor(low, m));
    }
    const int begin = split * plan.chunk, end = min(begin + plan.chunk, top);
    const float* kbase = a.k + b * a.k_stride[0] + kh * a.k_stride[1];
    const float* vbase = a.v + b * a.v_stride[0] + kh * a.v_stride[1];

    f32x4 acc[NB][4];
    float most = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int e = 0; e < NB; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[e][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 kx[KS], vx[4][NB];
    // Past the end of the range and of the row the last values are read again: such keys do not count, and such
    // elements meet zeros of q or are not stored.
    auto quad = [&](const float* row, int d) {
        if constexpr (WIDE) return *(const f32x4*)(row + min(d, a.d - 4));
        f32x4 x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = row[min(d + c, a.d - 1)];
        return x;
    };
    auto fetch_keys = [&](int j0) {
        const float* krow = kbase + (int64_t)min(j0 + col, end - 1) * a.k_stride[2];
#pragma unroll
        for (int t = 0; t < KS; ++t) kx[t] = quad(krow, 16 * t + 4 * h);
    };
    auto fetch_values = [&](int j0) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float* vrow = vbase + (int64_t)min(j0 + 4 * h + v, end - 1) * a.v_stride[2];
#pragma unroll
            for (int e = 0; e < NB; ++e) vx[v][e] = quad(vrow, 64 * e + 4 * col);
        }
    };
    int j0 = begin + 16 * wave;
    if (j0 < end) {
        fetch_keys(j0);
        fetch_values(j0);
    }
    while (j0 < end) {
        const int j1 = j0 + 64;
        // keys that are not finite become zeros, and their scores NaN
        bool kbad = false;
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) kbad = kbad || !finite_(kx[t][c]);
        unsigned kmask = 0;
        if (__any(kbad)) {                    // (a key's row is spread over four lanes)
            const unsigned long long m = __ballot(kbad);
            kmask = (unsigned)((m | m >> 16 | m >> 32 | m >> 48) & 0xffff);
#pragma unroll
            for (int t = 0; t < KS; ++t)
#pragma unroll
                for (int c = 0; c < 4; ++c) kx[t][c] = finite_(kx[t][c]) ? kx[t][c] : 0.f;
        }
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) x = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[t][c], own[t][c], x, 0, 0, 0);
        if (j1 < end) fetch_keys(j1);         // (values follow when they are used up: each is a step ahead)
        const bool whole = j0 + 16 <= low && !s.docs && !kmask;
        float peak = most;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int j = j0 + 4 * h + v;
            float z = score(a, x[v], slope2, pos, j);
            if (!whole) {
                if (kmask >> (4 * h + v) & 1) z = __builtin_nanf("");
                bool ok = j < lim && j < end;
                if (s.docs) ok = ok && s.docs[j < s.len ? j : 0] == doc;
                z = ok ? z : -__builtin_inff();
            }
            x[v] = z;
            peak = z > peak || z != z ? z : peak;
        }
#pragma unroll
        for (int m = 16; m < 64; m <<= 1) {
            const float other = __shfl_xor(peak, m);
            peak = other > peak || other != other ? other : peak;
        }
        const float ref = peak == -__builtin_inff() ? 0.f : peak;
        const float shrink = exp2_(most - ref);
        if (__any(shrink != 1.f)) {
            total *= shrink;
#pragma unroll
            for (int e = 0; e < NB; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[e][c] *= shrink;
        }
        most = peak;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            x[v] = exp2_(x[v] - ref);
            total += x[v];
        }
        // values that are not finite become zeros here and are added by themselves below
        unsigned vbad = 0;
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int e = 0; e < NB; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (!finite_(vx[v][e][c])) {
                        vx[v][e][c] = 0.f;
                        vbad |= 1u << (4 * h + v);
                    }
        if (__any(vbad != 0)) {
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) vbad |= __shfl_xor(vbad, m);
        }
#pragma unroll
        for (int e = 0; e < NB; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[e][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[v][e][c], x[v], acc[e][c], 0, 0, 0);
        if (j1 < end) fetch_values(j1);
        for (unsigned m = vbad; m; m &= m - 1) {
            const int key = __builtin_ctz(m);
            if (j0 + key >= end) break;              // (the last key again)
            int hh = h;
            asm volatile("" : "+v"(hh));             // (nothing of this is computed ahead and kept)
            const float* vrow = vbase + (int64_t)(j0 + key) * a.v_stride[2];
            float mine = 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) mine = v == (key & 3) ? x[v] : mine;
            const float weight = __shfl(mine, col + 16 * (key >> 2));
#pragma unroll
            for (int e = 0; e < NB; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const int d = 64 * e + 4 * (4 * hh + v) + c;
                        const float y = vrow[d < a.d ? d : 0], z = weight * y;
                        acc[e][c][v] += !finite_(y) && d < a.d && weight != 0.f ? z : 0.f;
                    }
        }
        j0 = j1;
    }

    // the four waves' results
    float sum = total;
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (h == 0) stat[wave][0][col] = most, stat[wave][1][col] = sum;
#pragma unroll
    for (int e = 0; e < NB; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            f32x4 x;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = acc[e][c][v];
            *(f32x4*)&merged[wave][col][64 * e + 4 * (4 * h + v)] = x;
        }
    __syncthreads();
    const int q = threadIdx.x >> 4, r = 16 * set + q;        // 16 threads for each row
    if (r >= rows) return;
    float peak = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float z = stat[w][0][q];
        peak = z > peak || z != z ? z : peak;
    }
    const float ref = peak == -__builtin_inff() ? 0.f : peak;
    float f[4], sum4 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2_(stat[w][0][q] - ref);
        sum4 += f[w] * stat[w][1][q];
    }
    const float by = sum4 > 0.f ? 1.f / sum4 : sum4 == 0.f ? 0.f : sum4;
    const float lse = sum4 == 0.f ? -__builtin_inff() : (peak + __builtin_amdgcn_logf(sum4)) * kLn2;
    const int og = r / a.lq, oi = r - og * a.lq, oh = kh * group + og, at = threadIdx.x & 15;
    const int64_t prow = (((int64_t)split * a.batch + b) * a.hq + oh) * a.lq + oi;
    float* to = part ? part + prow * a.d : a.o + b * a.o_stride[0] + oh * a.o_stride[1] + oi * a.o_stride[2];
#pragma unroll
    for (int e = 0; e < NB; ++e) {
        const int d = 64 * e + 4 * at;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 y = *(const f32x4*)&merged[w][q][d];
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] += f[w] == 0.f ? 0.f : f[w] * y[c];
        }
        x *= by;
        if (wide) {
            if (d < a.d) *(f32x4*)(to + d) = x;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (d + c < a.d) to[d + c] = x[c];
        }
    }
    if (at == 0) {
        if (part)
            part_lse[prow] = lse;
        else if (a.lse)
            a.lse[((int64_t)b * a.hq + oh) * a.lq + oi] = lse;
    }
}

// Results of key ranges into one (of many rows, those with keys in more than the first), four elements to a lane.  Up to kNear ranges: half a wave for each row, all
// loads at once (65536 causal rows of 128 in two ranges, half of them with keys in both: 15 us; if all are joined
// 21, 4.8 TB/s; a wave for each row, which first finds the largest sum, 42).  More: a block for each row, whose eight halves of waves take the ranges in turn (32 rows in
// 40 ranges 4 us, with one wave 6.4).
constexpr int kNear = 4;

template <bool NEAR> __global__ __launch_bounds__(kThreads) void attention_join(Args a, Plan plan, const float* part, const float* part_lse) {
    constexpr int HALVES = NEAR ? 1 : kThreads / 32, BATCH = NEAR ? kNear : 8;
    __shared__ f32x4 sums[HALVES][32];
    __shared__ float totals[HALVES];
    const int64_t rows = (int64_t)a.batch * a.hq * a.lq;
    const int half = threadIdx.x >> 5, lane = threadIdx.x & 31, d = 4 * lane;
    const int64_t row = NEAR ? (int64_t)blockIdx.x * (kThreads / 32) + half : blockIdx.x;
    if (NEAR && row >= rows) return;
    const int i = (int)(row % a.lq), splits = plan.splits, wide = plan.wide;
    const int64_t bh = row / a.lq;
    if (!plan.few) {
        const Seq s = sequence(a, (int)(bh / a.hq));
        if (row_limit(a, s, s.start + i) <= plan.chunk) return;      // (one range alone, and its result is where it belongs)
    }
    const int first = NEAR ? 0 : half;
    float lse[BATCH], peak = -__builtin_inff(), sum = 0.f;
    f32x4 y[BATCH], x = {0.f, 0.f, 0.f, 0.f};
    auto fetch = [&](int s0) {
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            const int s = s0 + e * HALVES;
            const int64_t at = min(s, splits - 1) * rows + row;
            lse[e] = s < splits ? part_lse[at] : -__builtin_inff();
            y[e] = s < splits ? load4(part + at * a.d, d, a.d, true, wide) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    fetch(first);
    if constexpr (NEAR) {
#pragma unroll
        for (int e = 0; e < BATCH; ++e) peak = lse[e] > peak || lse[e] != lse[e] ? lse[e] : peak;
    } else {
        for (int s = threadIdx.x & 63; s < splits; s += 64) {
            const float z = part_lse[s * rows + row];
            peak = z > peak || z != z ? z : peak;
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const float other = __shfl_xor(peak, m);
            peak = other > peak || other != other ? other : peak;
        }
    }
    const float ref = peak == -__builtin_inff() ? 0.f : peak;
    for (int s0 = first;;) {
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            const float w = exp2_((lse[e] - ref) * kLog2e);
            sum += w;
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] += w == 0.f ? 0.f : w * y[e][c];      // (a range without keys has nothing there)
        }
        s0 += BATCH * HALVES;
        if (s0 >= splits) break;
        fetch(s0);
    }
    if constexpr (!NEAR) {
        sums[half][lane] = x;
        if (lane == 0) totals[half] = sum;
        __syncthreads();
        if (half) return;
#pragma unroll
        for (int n = 1; n < HALVES; ++n) {
            x += sums[n][lane];
            sum += totals[n];
        }
    }
    const float by = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    float* to = a.o + bh / a.hq * a.o_stride[0] + bh % a.hq * a.o_stride[1] + i * a.o_stride[2];
    if (wide) {
        if (d < a.d) *(f32x4*)(to + d) = x * by;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (d + c < a.d) to[d + c] = x[c] * by;
    }
    if (lane == 0 && a.lse) a.lse[row] = sum == 0.f ? -__builtin_inff() : peak + __builtin_amdgcn_logf(sum) * kLn2;
}

// ---- gradient -------------------------------------------------------------------------------
// Two kinds of blocks, each with all sums of one output in one place, so that results do not depend on timing:
// dQ (rows own their sums, keys pass by, as in the forward kernel) and dK, dV (keys own their sums, rows pass
// by).  The scores are computed in both: seven products instead of five.  A wave holds two matrices of 32
// columns in planes and its sums, more than 256 registers, so there is one for each SIMD, and what it does on
// the vector unit stands between its matrix instructions.  Bound by the matrix units, which are busy for 54%
// of the time: 2 sequences of 2048 rows, 16 heads of 128, causal: 640 us at best and 669 at the median under the
// profiler, 180 TFLOP/s of float32 products.
template <int NT> struct GradLds {
    __attribute__((aligned(16))) char tile[2][2 * Planes<NT>::BYTES];
    __attribute__((aligned(16))) float stat[2][2][kTile];
    int ends[4], doc_range[2][4];
    unsigned poison[2][kRows][NT];
};

template <int NT, bool CAP>
__device__ __forceinline__ void grad_dq(const Args& a, const Plan& plan, int tiles, const Packed& in, int block, GradLds<NT>& shared) {
    using P = Planes<NT>;
    auto& lds = shared.tile;
    auto& ends = shared.ends;
    auto& doc_range = shared.doc_range;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int heads = a.batch * a.hkv;
    const int head = block % heads, tile = tiles - 1 - block / heads;
    const int b = head / a.hkv, kh = head % a.hkv, group = a.hq / a.hkv;
    const Seq s = sequence(a, b);
    const bool wide = plan.wide;
    const int rows = group * a.lq;
    const int r = (tile * 4 + wave) * 32 + (lane & 31);
    const bool valid = r < rows;
    const int i = valid ? r / group : 0, g = valid ? r - i * group : 0;
    const int qh = kh * group + g, p = s.start + i;
    const int64_t at = ((int64_t)b * a.hq + qh) * a.lq + i;
    const float lse = valid ? a.lse[at] : -__builtin_inff();
    const int lim = valid && lse != -__builtin_inff() ? row_limit(a, s, p) : 0;
    const int doc = s.docs && lim > 0 ? s.docs[p] : 0;
    const float slope2 = a.slopes ? a.slopes[qh] * kLog2e : 0.f;
    const float lse2 = lse == -__builtin_inff() ? __builtin_inff() : lse * kLog2e;       // (weights of exp2(-inf) = 0)
    const float dot = lim > 0 ? in.delta[at] : 0.f;

    const float scale = CAP ? a.scale : a.scale * kLog2e;
    Three own[2 * NT], dout[2 * NT];
    const float* qrow = a.q + b * a.q_stride[0] + qh * a.q_stride[1] + i * a.q_stride[2];
    const float* grow = a.dout + b * a.dout_stride[0] + qh * a.dout_stride[1] + i * a.dout_stride[2];
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4 x = load4(qrow, 16 * t + 8 * h + e, a.d, lim > 0, wide) * scale;
            split2<true>(f32x2{x[0], x[1]}, e, own[t]);
            split2<true>(f32x2{x[2], x[3]}, e + 2, own[t]);
            const f32x4 y = load4(grow, 16 * t + 8 * h + e, a.d, lim > 0, wide);
            split2<true>(f32x2{y[0], y[1]}, e, dout[t]);
            split2<true>(f32x2{y[2], y[3]}, e + 2, dout[t]);
        }
    }

    int top = lim, low = valid ? lim : 0x7fffffff, dlo = lim > 0 ? doc : 0x7fffffff, dhi = lim > 0 ? doc : -0x7fffffff - 1;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        top = max(top, __shfl_xor(top, m));
        low = min(low, __shfl_xor(low, m));
        dlo = min(dlo, __shfl_xor(dlo, m));
        dhi = max(dhi, __shfl_xor(dhi, m));
    }
    if (lane == 0) ends[wave] = top, doc_range[0][wave] = dlo, doc_range[1][wave] = dhi;
    __syncthreads();
    int end = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        end = max(end, ends[w]);
        dlo = min(dlo, doc_range[0][w]);
        dhi = max(dhi, doc_range[1][w]);
    }
    end = __builtin_amdgcn_readfirstlane(end);
    top = __builtin_amdgcn_readfirstlane(top);
    low = __builtin_amdgcn_readfirstlane(low);

    int docs_next = 0;
    int2 range_next = {0, 0};
    const int key_tiles = (a.lk + kTile - 1) / kTile;
    const int64_t place = (int64_t)head * key_tiles;
    Active active{in.key_docs + place, (end + kTile - 1) / kTile, dlo, dhi, -1, 0, {0, 0}};
    auto next = [&](int j0) {
        if (!s.docs) return j0;
        return __builtin_amdgcn_readfirstlane(active.next(j0 / kTile)) * kTile;
    };
    unsigned marks_next[2] = {0, 0};
    auto copy = [&](int to, int j) {                  // (marks are read ahead of the copies: a wait for them would wait for these)
        marks_next[0] = in.key_marks[place + j / kTile];
        marks_next[1] = in.value_marks[place + j / kTile];
        if (s.docs) docs_next = s.docs[min(j + (lane & 31), s.len - 1)], range_next = active.range(j / kTile);
        copy_to_lds<4, P::BYTES>(lds[to], in.key + (place + j / kTile) * P::BYTES);
        copy_to_lds<4, P::BYTES>(lds[to] + P::BYTES, in.value + (place + j / kTile) * P::BYTES);
    };

    f32x16 acc[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[c][v] = 0.f;
    int j0 = next(0), buf = 0;
    if (j0 < end) copy(0, j0);
    while (j0 < end) {
        copies_done();
        __syncthreads();
        const int docs = docs_next;
        const int2 range = range_next;
        const unsigned kbad = __builtin_amdgcn_readfirstlane(marks_next[0]), vbad = __builtin_amdgcn_readfirstlane(marks_next[1]);
        const int j1 = next(j0 + kTile);
        if (j1 < end) copy(buf ^ 1, j1);
        if (j0 < top) {
            f32x16 x = product6<NT, true>(lds[buf], own, lane);
            f32x16 slope;                              // of the capped scores
            if constexpr (CAP) {
                tanh_tile(x, 1.f / a.cap);
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    slope[v] = fmaf(-x[v], x[v], 1.f);
                    x[v] *= a.cap * kLog2e;
                }
            }
            if (a.slopes) {
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] -= slope2 * fabsf((float)(p - j0 - 4 * h - acc_row(v, 0)));
            }
            const bool whole = j0 + kTile <= low && !s.docs && !(kbad | vbad);
            if (!whole) {
                const unsigned same = s.docs ? same_document(docs, range, doc, h) : ~0u;
                const unsigned nans = kbad >> 4 * h;
                const int left = lim - j0 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const bool ok = acc_row(v, 0) < left && (same >> v & 1);
                    x[v] = nans >> acc_row(v, 0) & 1 ? __builtin_nanf("") : x[v];
                    x[v] = ok ? x[v] : -__builtin_inff();
                }
            }
            f32x16 y = product6<NT, true>(lds[buf] + P::BYTES, dout, lane, [&](int t) {
#pragma unroll
                for (int v = 16 * t / (2 * NT); v < 16 * (t + 1) / (2 * NT); ++v) x[v] = exp2_(x[v] - lse2);
            });
            if (vbad) {
#pragma unroll
                for (int v = 0; v < 16; ++v) y[v] = vbad >> 4 * h >> acc_row(v, 0) & 1 ? __builtin_nanf("") : y[v];
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = x[v] == 0.f ? 0.f : x[v] * (y[v] - dot) * (CAP ? slope[v] : 1.f);
            spread6<NT, true>(acc, lds[buf], split8(x, 0), x, lane);
            if (kbad)
                spread6_bad<NT>(acc, kbad, a.k + b * a.k_stride[0] + kh * a.k_stride[1] + j0 * a.k_stride[2], a.k_stride[2], a.d, x, lane);
        }
        buf ^= 1;
        j0 = j1;
    }
    if (valid) store_column<NT>(a.dq + b * a.dq_stride[0] + qh * a.dq_stride[1] + i * a.dq_stride[2], acc, a.scale, a.d, wide, h);
}

// More than one part: the query heads of a key head, and ranges of `span` rows of them, go to different blocks,
// whose sums are added by `attention_add`.
template <int NT, bool CAP>
__device__ __forceinline__ void grad_dkv(const Args& a, const Plan& plan, const Parts& parts, const Packed& in, float* part, int block, GradLds<NT>& shared) {
    using P = Planes<NT>;
    auto& lds = shared.tile;
    auto& stat = shared.stat;
    auto& doc_range = shared.doc_range;
    auto& poison = shared.poison;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int heads = a.batch * a.hkv, group = a.hq / a.hkv;
    int id = block;
    const int head = id % heads;
    id /= heads;
    const int slice = id % parts.count, tile = id / parts.count;       // (causal: the first keys are seen by the most rows)
    const int b = head / a.hkv, kh = head % a.hkv;
    const Seq s = sequence(a, b);
    const bool wide = plan.wide;
    const int key0 = tile * kRows, j = key0 + wave * 32 + (lane & 31);
    const bool valid = j < a.lk, counts = j < s.len;
    const int doc = s.docs && counts ? s.docs[j] : 0;
    // the first row that may see the key, and how many: with documents rows inside the sequence alone.  (The rest of the
    // last tile is no row: a key that is not finite would make its pairs NaN.)
    const int need = max(max(a.causal && j >= s.prefix ? j - s.start : 0, s.docs ? -s.start : 0), 0);
    const unsigned sees = counts ? max((s.docs ? min(a.lq, s.len - s.start) : a.lq) - need, 0) : 0;

    const float scale = CAP ? a.scale : a.scale * kLog2e;
    Three key[2 * NT], val[2 * NT];
    const float* krow = a.k + b * a.k_stride[0] + kh * a.k_stride[1] + (int64_t)j * a.k_stride[2];
    const float* vrow = a.v + b * a.v_stride[0] + kh * a.v_stride[1] + (int64_t)j * a.v_stride[2];
#pragma unroll
    for (int t = 0; t < 2 * NT; ++t) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4 x = load4(krow, 16 * t + 8 * h + e, a.d, counts, wide) * scale;
            split2<true>(f32x2{x[0], x[1]}, e, key[t]);
            split2<true>(f32x2{x[2], x[3]}, e + 2, key[t]);
            const f32x4 y = load4(vrow, 16 * t + 8 * h + e, a.d, counts, wide);
            split2<true>(f32x2{y[0], y[1]}, e, val[t]);
            split2<true>(f32x2{y[2], y[3]}, e + 2, val[t]);
        }
    }
    f32x16 dk[NT], dv[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int v = 0; v < 16; ++v) dk[c][v] = 0.f, dv[c][v] = 0.f;

    int dlo = counts ? doc : 0x7fffffff, dhi = counts ? doc : -0x7fffffff - 1, all = counts ? need : 0x7fffffff;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        dlo = min(dlo, __shfl_xor(dlo, m));
        dhi = max(dhi, __shfl_xor(dhi, m));
        all = max(all, __shfl_xor(all, m));
    }
    all = __builtin_amdgcn_readfirstlane(all);             // from this row on every key of the wave is seen
    if (lane == 0) doc_range[0][wave] = dlo, doc_range[1][wave] = dhi;
    for (int n = threadIdx.x; n < 2 * kRows * NT; n += kThreads) (&poison[0][0][0])[n] = 0;
    __syncthreads();
    dlo = min(min(doc_range[0][0], doc_range[0][1]), min(doc_range[0][2], doc_range[0][3]));
    dhi = max(max(doc_range[1][0], doc_range[1][1]), max(doc_range[1][2], doc_range[1][3]));

    // rows before `first` see none of the block's keys
    int first = 0;
    if (a.causal && key0 >= s.prefix) first = clamp_(key0 - s.start, 0, a.lq) & ~(kTile - 1);
    if (key0 >= s.len) first = a.lq;
    const int g0 = parts.count > 1 ? slice / parts.ranges : 0, g1 = parts.count > 1 ? g0 + 1 : group;
    const int rows_end = min(a.lq, (slice % parts.ranges + 1) * parts.span);
    first = max(first, slice % parts.ranges * parts.span);
    int docs_next = 0;
    int2 range_next = {0, 0};
    const int row_tiles = (a.lq + kTile - 1) / kTile;
    Active active{in.query_docs + (int64_t)b * a.hq * row_tiles, (rows_end + kTile - 1) / kTile, dlo, dhi, -1, 0, {0, 0}};      // (the same for every head)
    auto next = [&](int& g, int& i0) {     // to a tile of rows that may see a key of the block
        for (; g < g1; ++g, i0 = first) {
            if (s.docs) i0 = __builtin_amdgcn_readfirstlane(active.next(i0 / kTile)) * kTile;
            if (i0 < rows_end) return;
        }
    };
    auto place = [&](int g, int i0) { return ((int64_t)b * a.hq + kh * group + g) * row_tiles + i0 / kTile; };
    unsigned marks_next[2] = {0, 0};
    float lse_next = 0.f, delta_next = 0.f;
    auto copy = [&](int to, int g, int i0) {
        const int64_t n = place(g, i0);
        marks_next[0] = in.query_marks[n];
        marks_next[1] = in.grad_marks[n];
        if (s.docs) {
            const int i = i0 + (lane & 31), p = s.start + i;
            docs_next = i < a.lq && p >= 0 && p < s.len ? s.docs[p] : 0;
            range_next = active.range(i0 / kTile);
        }
        if (threadIdx.x < kTile) {
            const int i = i0 + threadIdx.x;
            const int64_t at = ((int64_t)b * a.hq + kh * group + g) * a.lq + i;
            lse_next = i < a.lq ? a.lse[at] : -__builtin_inff();       // (used when it has come: a wait now would be for all copies)
            delta_next = i < a.lq ? in.delta[at] : 0.f;
        }
        copy_to_lds<4, P::BYTES>(lds[to], in.query + n * P::BYTES);
        copy_to_lds<4, P::BYTES>(lds[to] + P::BYTES, in.grad + n * P::BYTES);
    };
    auto stage_stat = [&](int to) {           // weights of rows without pairs: exp2(x - inf) = 0
        if (threadIdx.x < kTile) {
            stat[to][0][threadIdx.x] = lse_next == -__builtin_inff() ? __builtin_inff() : lse_next * kLog2e;
            stat[to][1][threadIdx.x] = delta_next;
        }
    };
    unsigned any_bad = 0;
    int g = g0, i0 = first, buf = 0;
    next(g, i0);
    if (g < g1) copy(0, g, i0);
    while (g < g1) {
        copies_done();
        stage_stat(buf);
        __syncthreads();                      // this tile is there, and everyone is done with the other buffer
        const int docs = docs_next;
        const int2 range = range_next;
        const unsigned qbad = __builtin_amdgcn_readfirstlane(marks_next[0]), gbad = __builtin_amdgcn_readfirstlane(marks_next[1]);
        int ng = g, ni = i0 + kTile;
        next(ng, ni);
        const bool more = ng < g1;
        const float slope2 = a.slopes ? a.slopes[kh * group + __builtin_amdgcn_readfirstlane(g)] * kLog2e : 0.f;
        if (more) copy(buf ^ 1, ng, ni);

        const int qh = kh * group + g;
        f32x16 x = product6<NT, true>(lds[buf], key, lane), slope;
        if constexpr (CAP) {
            tanh_tile(x, 1.f / a.cap);
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                slope[v] = fmaf(-x[v], x[v], 1.f);
                x[v] *= a.cap * kLog2e;
            }
        }
        if (a.slopes) {
            const int apart = s.start + i0 + 4 * h - j;
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] -= slope2 * fabsf((float)(apart + acc_row(v, 0)));
        }
        if (i0 < all || s.docs || qbad) {
            const unsigned same = s.docs ? same_document(docs, range, doc, h) : ~0u;
            const unsigned nans = qbad >> 4 * h;
            const int from = need - i0 - 4 * h;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const bool ok = (unsigned)(acc_row(v, 0) - from) < sees && (same >> v & 1);
                x[v] = nans >> acc_row(v, 0) & 1 ? __builtin_nanf("") : x[v];
                x[v] = ok ? x[v] : -__builtin_inff();
            }
        }
        f32x16 row_lse, row_delta;            // (read ahead: inside a choice a read would be a branch)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const f32x4 e = *(const f32x4*)&stat[buf][0][8 * u + 4 * h], f = *(const f32x4*)&stat[buf][1][8 * u + 4 * h];
#pragma unroll
            for (int c = 0; c < 4; ++c) row_lse[4 * u + c] = e[c], row_delta[4 * u + c] = f[c];
        }
        Three lo;                             // weights of the first eight registers, split as they come
        f32x16 y = product6<NT, true>(lds[buf] + P::BYTES, val, lane, [&](int t) {
#pragma unroll
            for (int v = 16 * t / (2 * NT); v < 16 * (t + 1) / (2 * NT); ++v) {
                x[v] = x[v] == -__builtin_inff() ? 0.f : exp2_(x[v] - row_lse[v]);      // (the row's lse may be NaN)
                if (v < 8 && v % 2) split2(f32x2{x[v - 1], x[v]}, v - 1, lo);
            }
        });
        if (gbad) {
#pragma unroll
            for (int v = 0; v < 16; ++v) y[v] = gbad >> 4 * h >> acc_row(v, 0) & 1 ? __builtin_nanf("") : y[v];
        }
        Three dlow;
        spread6<NT, true>(dv, lds[buf] + P::BYTES, lo, x, lane, [&](int c) {
#pragma unroll
            for (int e = 16 * c / NT; e < 16 * (c + 1) / NT; ++e) {
                y[e] = x[e] == 0.f ? 0.f : x[e] * (y[e] - row_delta[e]) * (CAP ? slope[e] : 1.f);
                if (e < 8 && e % 2) split2(f32x2{y[e - 1], y[e]}, e - 1, dlow);
            }
        });
        spread6<NT, true>(dk, lds[buf], dlow, y, lane);
        if (gbad)
            note_bad<NT>(&poison[1][wave * 32], gbad, a.dout + b * a.dout_stride[0] + qh * a.dout_stride[1] + i0 * a.dout_stride[2], a.dout_stride[2], a.d, x, lane);
        if (qbad)
            note_bad<NT>(&poison[0][wave * 32], qbad, a.q + b * a.q_stride[0] + qh * a.q_stride[1] + i0 * a.q_stride[2], a.q_stride[2], a.d, y, lane);
        any_bad |= gbad | qbad;
        buf ^= 1;
        g = ng, i0 = ni;
    }
    if (any_bad) {
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NT; ++c) {
            const unsigned no_dk = poison[0][wave * 32 + (lane & 31)][c], no_dv = poison[1][wave * 32 + (lane & 31)][c];
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                dk[c][v] = no_dk >> acc_row(v, h) & 1 ? __builtin_nanf("") : dk[c][v];
                dv[c][v] = no_dv >> acc_row(v, h) & 1 ? __builtin_nanf("") : dv[c][v];
            }
        }
    }
    if (!valid) return;
    if (part) {
        const int64_t rows = (int64_t)heads * a.lk;
        float* to = part + (((int64_t)slice * 2) * rows + (int64_t)head * a.lk + j) * a.d;
        store_column<NT>(to, dk, a.scale, a.d, wide, h);
        store_column<NT>(to + rows * a.d, dv, 1.f, a.d, wide, h);
    } else {
        store_column<NT>(a.dk + b * a.dk_stride[0] + kh * a.dk_stride[1] + (int64_t)j * a.dk_stride[2], dk, a.scale, a.d, wide, h);
        store_column<NT>(a.dv + b * a.dv_stride[0] + kh * a.dv_stride[1] + (int64_t)j * a.dv_stride[2], dv, 1.f, a.d, wide, h);
    }
}

// Both in one launch, the longer dK, dV blocks first: neither waits for the other's last blocks (3 sequences of
// 517 rows, 6 heads of 64: 40 us, in two launches 25 more; 2 of 2048 rows, 16 heads of 128: 8 more).  The two take their
// arguments from copies: of one the compiler would read all values ahead of the choice and keep them, a hundred
// scalar registers more than there are.  Mixing the two kinds block by block costs 5%: an XCD's L2 then holds
// neither's matrices.
template <int NT, bool CAP>
__global__ __launch_bounds__(kThreads, 1) void attention_grad(Args a, Args same, Plan plan, Parts parts, Packed in, Packed same_in, int row_tiles, int dq_sets, int sets, float* part) {
    __shared__ GradLds<NT> shared;
    const int keys = a.batch * a.hkv * (sets - dq_sets);
    if ((int)blockIdx.x < keys)
        grad_dkv<NT, CAP>(a, plan, parts, in, part, blockIdx.x, shared);
    else
        grad_dq<NT, CAP>(same, plan, row_tiles, same_in, blockIdx.x - keys, shared);
}

// dK and dV from the parts of the query heads, in their order: half a wave for one row of one of them, four
// elements to a lane and four parts on their way.  Bound by memory.
__global__ __launch_bounds__(kThreads) void attention_add(Args a, int parts, int wide, const float* part) {
    const int64_t rows = (int64_t)a.batch * a.hkv * a.lk;
    const int d = 4 * (threadIdx.x & 31);
    int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (row >= 2 * rows) return;
    const float* from = part + row * a.d;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int n0 = 0; n0 < parts; n0 += 4) {
        f32x4 y[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) y[n] = load4(from + min(n0 + n, parts - 1) * 2 * rows * a.d, d, a.d, n0 + n < parts, wide);
#pragma unroll
        for (int n = 0; n < 4; ++n) x += y[n];
    }
    const bool second = row >= rows;
    if (second) row -= rows;
    const int64_t* stride = second ? a.dv_stride : a.dk_stride;
    const int64_t bh = row / a.lk;
    float* to = (second ? a.dv : a.dk) + bh / a.hkv * stride[0] + bh % a.hkv * stride[1] + row % a.lk * stride[2];
    if (wide) {
        if (d < a.d) *(f32x4*)(to + d) = x;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (d + c < a.d) to[d + c] = x[c];
    }
}

// ---- arguments of 64 bits -----------------------------------------------------------------------

__global__ __launch_bounds__(kThreads) void clamp_numbers(drhip_clamp_t a) {
    const int n = blockIdx.x * kThreads + threadIdx.x;
    if (n >= a.n) return;
    const int64_t x = a.x[n * a.x_stride];
    a.y[n] = (int32_t)(x < a.low ? a.low : x > a.high ? a.high : x);
}

// Document numbers are told apart by equality alone, so a number may become the place where it first stands in its
// sequence.  A table of at least twice as many slots as there are numbers holds for each of them that place: the first of each
// run of equal numbers looks for its slot from the number's hash on (multiplicative, upwards), then every number reads
// its place.  What it gives does not depend on timing.  Bound by its three launches (3 sequences of
// 1111: 4, 2.3 and 2.8 us, 6 us more for a call than with numbers of 32 bits).
constexpr int kFree = 0x7fffffff;

__device__ __forceinline__ unsigned slot_of(int64_t x, int log) { return (unsigned)((uint64_t)x * 0x9e3779b97f4a7c15ull >> (64 - log)); }

__global__ __launch_bounds__(kThreads) void renumber_clear(int32_t* table, int64_t count) {
    for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < count; n += (int64_t)gridDim.x * kThreads) table[n] = kFree;
}

__global__ __launch_bounds__(kThreads) void renumber_enter(drhip_renumber_t a, int log, int blocks) {
    const int b = blockIdx.x / blocks, j = blockIdx.x % blocks * kThreads + threadIdx.x;
    if (j >= a.n) return;
    const int64_t* row = a.x + b * a.x_stride;
    const int64_t x = row[j];
    if (j && row[j - 1] == x) return;
    int32_t* table = a.table + ((int64_t)b << log);
    for (unsigned at = slot_of(x, log);; at = (at + 1) & ((1u << log) - 1)) {      // (half of the slots stay free)
        const int i = atomicCAS(&table[at], kFree, j);
        if (i != kFree && row[i] != x) continue;
        if (i != kFree) atomicMin(&table[at], j);
        return;
    }
}

__global__ __launch_bounds__(kThreads) void renumber_read(drhip_renumber_t a, int log, int blocks) {
    const int b = blockIdx.x / blocks, j = blockIdx.x % blocks * kThreads + threadIdx.x;
    if (j >= a.n) return;
    const int64_t* row = a.x + b * a.x_stride;
    const int64_t x = row[j];
    const int32_t* table = a.table + ((int64_t)b << log);
    unsigned at = slot_of(x, log);
    int i = table[at];
    while (i != kFree && row[i] != x) {
        at = (at + 1) & ((1u << log) - 1);
        i = table[at];
    }
    a.y[(int64_t)b * a.n + j] = i;
}

bool aligned(const void* p, const int64_t* stride) {
    return (uintptr_t)p % 16 == 0 && stride[0] % 4 == 0 && stride[1] % 4 == 0 && stride[2] % 4 == 0;
}

// Sets of 16 rows of a key head (one without rows, for the sizes of workspaces)
constexpr int64_t kSmall16 = 25000000;       // (sets of 16 rows) x keys x elements

int few_sets(const Args& a) { return a.lq ? (int)(((int64_t)(a.hq / a.hkv) * a.lq + 15) / 16) : 1; }

int row_tiles(const Args& a) { return (int)(((int64_t)(a.hq / a.hkv) * a.lq + kRows - 1) / kRows); }

// Which forward kernel, and into how many key ranges.  Up to 64 rows of a key head, and few rows times keys in
// all, go to the kernel for few rows, whose blocks are smaller and whose operands are not packed first: 32
// sequences of 4096 keys, 8 key heads of 128, 64 rows: 621 us, in the other kernel 848; 96 rows: 927 and 857; 32 heads of 128
// with 256 rows and keys 24 us and 36, 512 60 and 50; 16 with 64 of 777 and head size 80 35 and 40, 128 54 and
// 43.  With documents only the other one passes over tiles.  Its blocks of eight waves share each tile among 256 rows, of
// four where that leaves compute units without a block.  Ranges: enough for a block on each compute unit (two,
// as causal blocks are of unequal length; not with documents, whose rows see a part of the keys alone: 60 us
// against 85 for three sequences of 1111), none shorter than 256 keys, whose work pays for joining.  For few rows,
// two blocks for each compute unit with ranges of 128 keys or more, and up to eight, since sequences are of
// unequal length, as long as ranges have 512.
Plan plan_forward(const Args& a) {
    Plan p;
    p.wide = a.d % 4 == 0 && aligned(a.q, a.q_stride) && aligned(a.k, a.k_stride) && aligned(a.v, a.v_stride) && aligned(a.o, a.o_stride);
    const int64_t rows = (int64_t)(a.hq / a.hkv) * a.lq, heads = (int64_t)a.batch * a.hkv;
    p.few = rows <= 64 || (!a.documents && heads * few_sets(a) * a.lk * a.d <= kSmall16);
    p.waves = heads * ((rows + 255) / 256) >= 256 ? 8 : 4;
    const int64_t blocks = heads * (p.few ? few_sets(a) : (rows + 32 * p.waves - 1) / (32 * p.waves));
    int64_t splits;
    if (p.few) {
        splits = (512 + blocks - 1) / blocks;
        const int64_t fine = (2048 + blocks - 1) / blocks, most = (a.lk + 127) / 128, long_ranges = a.lk / 512;
        if (splits < fine) splits = fine < long_ranges ? fine : long_ranges > splits ? long_ranges : splits;
        if (splits > most) splits = most;
    } else {
        const int64_t want = a.documents ? 64 : a.causal ? 512 : 256, most = (a.lk + 255) / 256;
        splits = blocks >= want ? 1 : (want + blocks - 1) / blocks;
        if (splits > most) splits = most;
    }
    if (splits < 1) splits = 1;
    p.chunk = (int)(((a.lk + splits - 1) / splits + 63) / 64 * 64);
    if (p.chunk < 64) p.chunk = 64;
    p.splits = a.lk > 0 ? (a.lk + p.chunk - 1) / p.chunk : 1;
    return p;
}

uint64_t up(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

// Workspaces, as offsets; packed matrices first
struct Room {
    Packed packed;              // (offsets from null)
    uint64_t lse, part, all;
};

// One array of `bytes` behind the others
template <typename T> T* next_room(uint64_t& at, uint64_t bytes) {
    T* p = (T*)at;
    at += up(bytes);
    return p;
}

Room room_forward(const Args& a, const Plan& p) {
    const uint64_t rows = (uint64_t)a.batch * a.hq * a.lq, tiles = (uint64_t)a.batch * a.hkv * ((a.lk + kTile - 1) / kTile);
    const uint64_t planes = tiles * 6144 * ((a.d + 31) / 32);
    Room r{};
    uint64_t at = 0;
    if (!p.few) {
        r.packed.key_marks = next_room<unsigned>(at, tiles * 4);
        r.packed.value_marks = next_room<unsigned>(at, tiles * 4);
        r.packed.key_docs = next_room<int2>(at, a.documents ? tiles * 8 : 0);
        r.packed.key = next_room<char>(at, planes);
        r.packed.value = next_room<char>(at, planes);
    }
    r.lse = at;
    if (p.splits > 1) next_room<float>(at, rows * p.splits * 4);
    r.part = at;
    if (p.splits > 1) next_room<float>(at, rows * p.splits * a.d * 4);
    r.all = at;
    return r;
}

Room room_grad(const Args& a, const Parts& parts) {
    const uint64_t rows = (uint64_t)a.batch * a.hq * a.lq, nt = (a.d + 31) / 32;
    const uint64_t keys = (uint64_t)a.batch * a.hkv * ((a.lk + kTile - 1) / kTile), queries = (uint64_t)a.batch * a.hq * ((a.lq + kTile - 1) / kTile);
    Room r{};
    uint64_t at = 0;
    r.packed.delta = next_room<float>(at, rows * 4);
    r.packed.key_marks = next_room<unsigned>(at, keys * 4);
    r.packed.value_marks = next_room<unsigned>(at, keys * 4);
    r.packed.query_marks = next_room<unsigned>(at, queries * 4);
    r.packed.grad_marks = next_room<unsigned>(at, queries * 4);
    r.packed.key_docs = next_room<int2>(at, a.documents ? keys * 8 : 0);
    r.packed.query_docs = next_room<int2>(at, a.documents ? queries * 8 : 0);
    r.packed.key = next_room<char>(at, keys * 6144 * nt);
    r.packed.value = next_room<char>(at, keys * 6144 * nt);
    r.packed.query = next_room<char>(at, queries * 6144 * nt);
    r.packed.grad = next_room<char>(at, queries * 6144 * nt);
    r.part = at;
    if (parts.count > 1) next_room<float>(at, (uint64_t)parts.count * 2 * a.batch * a.hkv * a.lk * a.d * 4);
    r.all = at;
    return r;
}

// The packed matrices of a room whose memory begins at `work`
Packed packed_at(const Room& room, char* work) {
    Packed p = room.packed;
    auto move = [&](auto*& x) { x = (std::remove_reference_t<decltype(x)>)(work + (uint64_t)x); };
    move(p.key), move(p.value), move(p.query), move(p.grad);
    move(p.key_marks), move(p.value_marks), move(p.query_marks), move(p.grad_marks), move(p.key_docs), move(p.query_docs), move(p.delta);
    return p;
}

Pack pack_of(const float* x, const int64_t* stride, int heads, int rows, int keys, const char* planes, const unsigned* marks, const int2* docs = nullptr, float* delta = nullptr) {
    return Pack{x, {stride[0], stride[1], stride[2]}, heads, (rows + kTile - 1) / kTile, keys, (char*)planes, (unsigned*)marks, (int2*)docs, delta};
}

template <int NT> void launch_rows(const Args& a, const Plan& p, const Packed& in, float* part, float* part_lse, hipStream_t s) {
    const int64_t rows = (int64_t)(a.hq / a.hkv) * a.lq, heads = (int64_t)a.batch * a.hkv;
    const int key_tiles = (a.lk + kTile - 1) / kTile, tiles = (int)((rows + 32 * p.waves - 1) / (32 * p.waves));
    Packs packs{};
    packs.job[0] = pack_of(a.k, a.k_stride, a.hkv, a.lk, 1, in.key, in.key_marks, a.documents ? in.key_docs : nullptr);
    packs.job[1] = pack_of(a.v, a.v_stride, a.hkv, a.lk, 1, in.value, in.value_marks);
    if (key_tiles) attention_pack<NT><<<dim3((unsigned)(2 * heads * key_tiles)), kThreads, 0, s>>>(a, packs, p.wide);
    const dim3 grid((unsigned)(heads * tiles * p.splits));
    if (p.waves == 8)
        attention_rows<NT, 8><<<grid, 512, 0, s>>>(a, p, tiles, in, part, part_lse);
    else
        attention_rows<NT, 4><<<grid, 256, 0, s>>>(a, p, tiles, in, part, part_lse);
}

template <bool WIDE> void launch_few(const Args& a, const Plan& p, float* part, float* part_lse, hipStream_t s) {
    const int sets = few_sets(a);
    const dim3 grid((unsigned)(a.batch * a.hkv * sets * p.splits));
    if (a.d <= 64)
        attention_few<1, WIDE><<<grid, kThreads, 0, s>>>(a, p, sets, part, part_lse);
    else
        attention_few<2, WIDE><<<grid, kThreads, 0, s>>>(a, p, sets, part, part_lse);
}

template <int NT> void launch_grad(const Args& a, const Plan& p, const Parts& parts, const Packed& in, float* part, hipStream_t s) {
    const int64_t heads = (int64_t)a.batch * a.hkv;
    const int key_tiles = (a.lk + kTile - 1) / kTile, query_tiles = (a.lq + kTile - 1) / kTile, tiles = row_tiles(a);
    Packs packs{};
    packs.job[0] = pack_of(a.k, a.k_stride, a.hkv, a.lk, 1, in.key, in.key_marks, a.documents ? in.key_docs : nullptr);
    packs.job[1] = pack_of(a.v, a.v_stride, a.hkv, a.lk, 1, in.value, in.value_marks);
    packs.job[2] = pack_of(a.q, a.q_stride, a.hq, a.lq, 0, in.query, in.query_marks, a.documents ? in.query_docs : nullptr);
    packs.job[3] = pack_of(a.dout, a.dout_stride, a.hq, a.lq, 0, in.grad, in.grad_marks, nullptr, in.delta);
    const int64_t blocks = 2 * heads * key_tiles + 2 * (int64_t)a.batch * a.hq * query_tiles;
    attention_pack<NT><<<dim3((unsigned)blocks), kThreads, 0, s>>>(a, packs, p.wide);
    const int dq_sets = a.lq ? tiles : 0, sets = dq_sets + parts.count * ((a.lk + kRows - 1) / kRows);
    const dim3 grid((unsigned)(heads * sets));
    if (a.cap > 0.f)
        attention_grad<NT, true><<<grid, kThreads, 0, s>>>(a, a, p, parts, in, in, tiles, dq_sets, sets, part);
    else
        attention_grad<NT, false><<<grid, kThreads, 0, s>>>(a, a, p, parts, in, in, tiles, dq_sets, sets, part);
    if (a.lk && parts.count > 1) attention_add<<<dim3((unsigned)((2 * heads * a.lk + 7) / 8)), kThreads, 0, s>>>(a, parts.count, p.wide, part);
}

// Query heads of a key head go to blocks of their own where the keys alone give fewer than two blocks to a
// compute unit, and ranges of rows as well where that leaves some without one
Parts plan_parts(const Args& a) {
    const int64_t blocks = (int64_t)a.batch * a.hkv * ((a.lk + kRows - 1) / kRows);
    const int group = a.hq / a.hkv;
    Parts p{1, 1, a.lq > 0 ? (a.lq + kTile - 1) / kTile * kTile : kTile};
    if (blocks >= 512 || blocks == 0) return p;
    int64_t ranges = 256 / (blocks * group);
    if (ranges > a.lq / kRows) ranges = a.lq / kRows;
    if (ranges < 1) ranges = 1;
    p.span = (int)(((a.lq + ranges - 1) / ranges + kTile - 1) / kTile * kTile);
    if (p.span < kTile) p.span = kTile;
    p.ranges = (int)(((int64_t)a.lq + p.span - 1) / p.span);
    if (p.ranges < 1) p.ranges = 1;
    p.count = group * p.ranges;
    return p;
}

}  // namespace

extern "C" uint64_t drhip_k_attention_work(const drhip_attention_t* a, int grad) {
    return grad ? room_grad(*a, plan_parts(*a)).all : room_forward(*a, plan_forward(*a)).all;
}

// Whether the forward call packs its keys and values
extern "C" int drhip_k_attention_packs(const drhip_attention_t* a) { return !plan_forward(*a).few; }

extern "C" int drhip_k_attention(const drhip_attention_t* args, hipStream_t s) {
    const Args& a = *args;
    const Plan p = plan_forward(a);
    const int64_t rows = (int64_t)a.batch * a.hq * a.lq, heads = (int64_t)a.batch * a.hkv;
    const Room room = room_forward(a, p);
    char* work = (char*)a.work;
    float* part = p.splits > 1 ? (float*)(work + room.part) : nullptr;
    float* part_lse = p.splits > 1 ? (float*)(work + room.lse) : nullptr;
    if (p.few) {
        p.wide ? launch_few<true>(a, p, part, part_lse, s) : launch_few<false>(a, p, part, part_lse, s);
    } else {
        const Packed in = packed_at(room, work);
        switch ((a.d + 31) / 32) {
            case 1: launch_rows<1>(a, p, in, part, part_lse, s); break;
            case 2: launch_rows<2>(a, p, in, part, part_lse, s); break;
            case 3: launch_rows<3>(a, p, in, part, part_lse, s); break;
            default: launch_rows<4>(a, p, in, part, part_lse, s); break;
        }
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
    if (p.splits > 1) {
        if (p.splits <= kNear)
            attention_join<true><<<dim3((unsigned)((rows + 7) / 8)), kThreads, 0, s>>>(a, p, part, part_lse);
        else
            attention_join<false><<<dim3((unsigned)rows), kThreads, 0, s>>>(a, p, part, part_lse);
        e = hipGetLastError();
    }
    return (int)e;
}

extern "C" int drhip_k_attention_grad(const drhip_attention_t* args, hipStream_t s) {
    const Args& a = *args;
    const Parts parts = plan_parts(a);
    const Room room = room_grad(a, parts);
    char* work = (char*)a.work;
    const Packed in = packed_at(room, work);
    float* part = parts.count > 1 ? (float*)(work + room.part) : nullptr;
    Plan p{};
    p.wide = a.d % 4 == 0 && aligned(a.q, a.q_stride) && aligned(a.k, a.k_stride) && aligned(a.v, a.v_stride) && aligned(a.o, a.o_stride) &&
             aligned(a.dout, a.dout_stride) && aligned(a.dq, a.dq_stride) && aligned(a.dk, a.dk_stride) && aligned(a.dv, a.dv_stride);
    if (!a.lq && !a.lk) return 0;
    switch ((a.d + 31) / 32) {
        case 1: launch_grad<1>(a, p, parts, in, part, s); break;
        case 2: launch_grad<2>(a, p, parts, in, part, s); break;
        case 3: launch_grad<3>(a, p, parts, in, part, s); break;
        default: launch_grad<4>(a, p, parts, in, part, s); break;
    }
    return (int)hipGetLastError();
}

extern "C" int drhip_k_renumber(const drhip_renumber_t* a, int log, hipStream_t s) {
    const int64_t count = (int64_t)a->batch << log;
    const int blocks = (a->n + kThreads - 1) / kThreads;
    renumber_clear<<<dim3((unsigned)(count < 2048 * kThreads ? (count + kThreads - 1) / kThreads : 2048)), kThreads, 0, s>>>(a->table, count);
    renumber_enter<<<dim3((unsigned)(a->batch * blocks)), kThreads, 0, s>>>(*a, log, blocks);
    renumber_read<<<dim3((unsigned)(a->batch * blocks)), kThreads, 0, s>>>(*a, log, blocks);
    return (int)hipGetLastError();
}

extern "C" int drhip_k_clamp(const drhip_clamp_t* a, hipStream_t s) {
    clamp_numbers<<<dim3((unsigned)((a->n + kThreads - 1) / kThreads)), kThreads, 0, s>>>(*a);
    return (int)hipGetLastError();
}
