// paged.h -- a part of attention.hip: many sequences at once over a paged cache of
// 8-bit blocks.  Rotary positions of rows, appending keys and values (with the
// per-head RMSNorm and the rotation on the way), and attention over the cache.
//
// A block is 16 positions of one KV head, K as [16][HD] and V as [HD][16] e4m3
// codes, each with a power of two as scale.  A power of two costs up to a bit of
// range that e4m3 has to spare, and buys that a value's code is the same digits in
// any scale: a block whose scale grows while tokens are appended keeps its codes
// exactly (but for those that become subnormal), and a scale is an addition to the
// exponent of the block's scores and weights, while the matrix instructions take
// the codes themselves, exact in fp16.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "gncx_device.h"
#include "gncx_launch.h"
#include "gncx_wave64.h"

namespace gncx {
namespace {

using namespace dev;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// ---- rotation ------------------------------------------------------------------
// cos and sin of position * freq, times the magnitude, in 64 bits (32 keep a far position's
// angle only to 2^-24 of it; and the chip multiplies and adds 64 bits as fast).  The angle's
// turns less the nearest quarter leave x in [-pi / 4, pi / 4], whose Taylor sums are off by
// 4 10^-13 at most; the quarter swaps and negates them.
__device__ __forceinline__ void turn_of(int32_t pos, double freq, double magnitude, double& c, double& s) {
    double t = static_cast<double>(pos) * freq * 0.15915494309189535;  // 1 / (2 pi)
    t -= rint(t);
    const double k = rint(4.0 * t), x = (t - 0.25 * k) * 6.283185307179586, z = x * x;
    double a = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0), b = fma(z, 1.0 / 479001600.0, -1.0 / 3628800.0);
    a = fma(z, a, 1.0 / 362880.0);
    b = fma(z, b, 1.0 / 40320.0);
    a = fma(z, a, -1.0 / 5040.0);
    b = fma(z, b, -1.0 / 720.0);
    a = fma(z, a, 1.0 / 120.0);
    b = fma(z, b, 1.0 / 24.0);
    a = fma(z, a, -1.0 / 6.0);
    b = fma(z, b, -0.5);
    a = fma(x * z, a, x);
    b = fma(z, b, 1.0);
    const int q = static_cast<int>(k) & 3;
    c = magnitude * (q & 1 ? a : b) * (q == 1 || q == 2 ? -1.0 : 1.0);
    s = magnitude * (q & 1 ? b : a) * (q >= 2 ? -1.0 : 1.0);
}

// Floats of pair p of a head: the rotated part's pairs, then the rest's, paired alike.
__device__ __forceinline__ void pair_floats(int p, int n_rot, int head_dim, bool inter, int& a, int& b) {
    const int half = n_rot / 2;
    if (inter) {
        a = 2 * p;
        b = a + 1;
    } else if (p < half) {
        a = p;
        b = p + half;
    } else {
        a = n_rot + p - half;
        b = a + (head_dim - n_rot) / 2;
    }
}

// Four pairs from 4 u on as two float4 each, where n_rot and head_dim are multiples of 8.
struct FourPairs {
    int off_a, off_b;  // where the two float4 stand
    bool inter;
    __device__ FourPairs(int u, int n_rot, int head_dim, bool interleaved) : inter(interleaved) {
        if (inter) {
            off_a = 8 * u;
            off_b = off_a + 4;
        } else {
            pair_floats(4 * u, n_rot, head_dim, false, off_a, off_b);
        }
    }
    __device__ void load(const float* head, float (&a)[4], float (&b)[4]) const {
        const f32x4 x = *reinterpret_cast<const f32x4*>(head + off_a), y = *reinterpret_cast<const f32x4*>(head + off_b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = inter ? (j < 2 ? x[2 * j & 3] : y[2 * j & 3]) : x[j];
            b[j] = inter ? (j < 2 ? x[(2 * j + 1) & 3] : y[(2 * j + 1) & 3]) : y[j];
        }
    }
    __device__ void store(float* head, const float (&a)[4], const float (&b)[4]) const {
        f32x4 x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = inter ? (j & 1 ? b[j / 2] : a[j / 2]) : a[j];
            y[j] = inter ? (j & 1 ? b[2 + j / 2] : a[2 + j / 2]) : b[j];
        }
        *reinterpret_cast<f32x4*>(head + off_a) = x;
        *reinterpret_cast<f32x4*>(head + off_b) = y;
    }
};

template <class T>
__device__ __forceinline__ void turn_pairs(T (&a)[4], T (&b)[4], const T (&c)[4], const T (&s)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const T x = a[j] * c[j] - b[j] * s[j];
        b[j] = b[j] * c[j] + a[j] * s[j];
        a[j] = x;
    }
}

// (a, b) -> (a cos - b sin, b cos + a sin) over a row's pairs.  Bound by memory, 8 bytes a
// float (2048 rows of 40 heads of 128, half of each turned: 13 to 14 us, 6 TB/s of 84 MB that
// the caches hold in part), a single row by the launch.  A work-group takes a row and some of
// its heads; its first threads form the row's cosines and sines, one pair each, for all of
// them, so that 64-bit angles cost a head's share of the heads.  Heads of 8 floats and more
// move as float4 where strides and addresses allow, others one float at a time (any even
// size, stride and alignment).
constexpr int kRopeThreads = 256;
constexpr int kMaxRopeDim = 1024;
struct RopeRowsParams {
    const float* rows;
    float* out;
    const int32_t* positions;
    RotationArgs rot;
    int32_t n_heads, head_dim, stride, out_stride, heads_per_group;
};

template <bool VEC>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeRowsParams p) {
    __shared__ __align__(16) float cs[kMaxRopeDim / 2], sn[kMaxRopeDim / 2];
    const int row = blockIdx.x, tid = threadIdx.x, half = p.rot.n_rot / 2, pairs = p.head_dim / 2;
    const int h0 = blockIdx.y * p.heads_per_group, h1 = min(h0 + p.heads_per_group, p.n_heads);
    const int32_t pos = p.positions[row];
    for (int i = tid; i < pairs; i += kRopeThreads) {
        double c = 1.0, s = 0.0;
        if (i < half) turn_of(pos, p.rot.freqs[i], p.rot.magnitude, c, s);
        cs[i] = static_cast<float>(c);
        sn[i] = static_cast<float>(s);
    }
    __syncthreads();
    const float* in = p.rows + static_cast<size_t>(row) * p.stride;
    float* out = p.out + static_cast<size_t>(row) * p.out_stride;
    const bool inter = p.rot.interleaved != 0;
    const int units = VEC ? pairs / 4 : pairs, each = kRopeThreads / units;  // heads at once
    if constexpr (VEC) {
        const int u = tid % units;
        const FourPairs at(u, p.rot.n_rot, p.head_dim, inter);
        float c[4], s[4];
        *reinterpret_cast<f32x4*>(c) = reinterpret_cast<const f32x4*>(cs)[u];
        *reinterpret_cast<f32x4*>(s) = reinterpret_cast<const f32x4*>(sn)[u];
        const bool turns = 4 * u < half;
        if (tid < units * each)
            for (int h = h0 + tid / units; h < h1; h += each) {
                float a[4], b[4];
                at.load(in + h * p.head_dim, a, b);
                if (turns) turn_pairs(a, b, c, s);
                at.store(out + h * p.head_dim, a, b);
            }
    } else {
        for (int i = tid; i < (h1 - h0) * pairs; i += kRopeThreads) {
            const int h = h0 + i / pairs, q = i % pairs;
            int a, b;
            pair_floats(q, p.rot.n_rot, p.head_dim, inter, a, b);
            const float x = in[h * p.head_dim + a], y = in[h * p.head_dim + b];
            out[h * p.head_dim + a] = q < half ? x * cs[q] - y * sn[q] : x;
            out[h * p.head_dim + b] = q < half ? y * cs[q] + x * sn[q] : y;
        }
    }
}

// ---- the sequences of a call ------------------------------------------------------
// The rows of a sequence that have a place: [row0, row0 + count) at positions len ..
struct SeqRows {
    int32_t row0, count, len;
};
__device__ __forceinline__ int clamp_row(const PagedArgs& c, int32_t r) { return min(max(r, 0), c.n_rows); }
__device__ __forceinline__ SeqRows seq_rows(const PagedArgs& c, int s) {
    SeqRows r;
    r.row0 = clamp_row(c, c.row_start[s]);
    r.len = c.lengths[s];
    const int32_t room = c.max_pages << c.page_bits;
    r.count = r.len < 0 || r.len > room ? 0 : min(max(clamp_row(c, c.row_start[s + 1]) - r.row0, 0), room - r.len);
    return r;
}
// The last sequence s with first(s) <= at, by a wave; -1 before the first.  first
// ascends (where row_start does; otherwise any sequence, or none, is found).  Sixty-four
// sequences are looked at at once, then those between two of them (one after the other,
// 1000 sequences of one row cost the append 101 us).
template <class F>
__device__ __forceinline__ int find_seq(int n_seqs, int64_t at, F&& first) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    for (int span = n_seqs;;) {
        const int every = (span + 63) / 64, k = lane * every;
        const int found = __builtin_popcountll(__ballot(k < span && first(lo + min(k, span - 1)) <= at));
        if (found == 0) return -1;
        lo += (found - 1) * every;
        span = min(every, span - (found - 1) * every);
        if (every == 1) return lo;
    }
}
// Where a key's page stands in the table (the last one's place for keys past it, which are
// hidden), and its block in the pool, -1 if the page is not there.
__device__ __forceinline__ int32_t page_at(const PagedArgs& c, const int32_t* table, int32_t key) {
    return table[min(key >> c.page_bits, c.max_pages - 1)];
}
__device__ __forceinline__ int64_t block_in(const PagedArgs& c, int32_t page, int head, int32_t key) {
    const int64_t b = ((static_cast<int64_t>(page) * c.n_kv + head) << (c.page_bits - 4)) +
                      ((key >> 4) & ((1 << (c.page_bits - 4)) - 1));
    return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.n_pages) ? b : -1;
}

// The block of a position below max_pages * page_tokens: its number in the pool's
// [page][head] order, -1 if its page is not there.
__device__ __forceinline__ int64_t block_of(const PagedArgs& c, int s, int head, int32_t pos) {
    return block_in(c, page_at(c, c.pages + static_cast<size_t>(s) * c.max_pages, pos), head, pos);
}

// ---- appending ----------------------------------------------------------------------
// Powers of two of the scales
constexpr int kLeastExp = -100, kMostExp = 120;
// The least e with amax <= 448 2^e (448 = 0.875 2^9, e4m3's largest)
__device__ __forceinline__ int scale_exp(float amax) {
    int k;
    const float f = frexpf(amax, &k);
    const int e = amax == 0.0f ? kLeastExp : f <= 0.875f ? k - 9 : k - 8;
    return min(max(e, kLeastExp), kMostExp);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }
__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;  // (NaN compares false)
}
__device__ __forceinline__ float to_code_range(float x, float inv) {
    return fabsf(x) < __builtin_inff() ? x * inv : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return static_cast<uint32_t>(r);
}
// Codes to a scale 1 / f as large
__device__ __forceinline__ uint32_t moved_codes(uint32_t w, float f) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return four_codes(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}

template <int N>
__device__ __forceinline__ double lanes_sum(double v) {  // (the same steps)
    v = dpp_add_f64<0xb1>(v);
    v = dpp_add_f64<0x4e>(v);
    v = dpp_add_f64<0x141>(v);
    if constexpr (N >= 16) v = dpp_add_f64<0x140>(v);
    return N == 32 ? v + __shfl_xor(v, 16, 64) : v;
}
__device__ __forceinline__ float root_inverse(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double root_inverse(double v) {  // one step of Newton's on 24 bits
    const double y = __builtin_amdgcn_rsq(v), e = fma(-v * y, y, 1.0);
    return e == e ? fma(0.5 * y, e, y) : y;  // (0 and infinity)
}
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (N == 32) {
        v = group_sum<16>(v);
        return v + __shfl_xor(v, 16, 64);
    } else {
        return group_sum<N>(v);
    }
}
// v in 32 bits with the last one set where it is not exact: what is then rounded to fewer
// is rounded as v would be.
__device__ __forceinline__ float odd_float(double v) {
    const float f = static_cast<float>(v);
    const double back = static_cast<double>(f);
    if (back == v || !(fabsf(f) < __builtin_inff())) return f;
    const uint32_t bits = __builtin_bit_cast(uint32_t, f) - (fabs(back) > fabs(v) ? 1u : 0u);
    return __builtin_bit_cast(float, bits | 1u);
}

struct AppendParams {
    AppendArgs a;
    int64_t kv_groups;    // work-groups of the cache's blocks
    bool by_rows;         // a slot a row
    int32_t head_groups;  // of a row's queries
    uint32_t first;       // work-group of the launch
};

// scale = max(old, 2^e), e the least with amax <= 448 2^e over the new values; codes are
// x / scale rounded to e4m3, old ones times old / scale again.  Blocks and queries in one
// launch: few rows are bound by it and by two dependent reads (one row 4.8 us, 64 rows of 64
// sequences 7.2), many by memory and the 64-bit rotation of K (2462 rows of 32 heads on 8 of
// 128, 106 MB: 28 us, 3.8 TB/s).  A work-group takes the new tokens of one block
// of K or of V: 16 tokens, HD / 8 threads each.  Nobody else touches the block, so
// its old tokens are moved to a larger scale on the way, without atomics.  Sequence
// s has the blocks from slot row_start[s] / 16 + 2 s on, or from row_start[s] on where those are
// fewer in all (decode steps): as many as it can touch.
// The other work-groups take 16 heads of a query row each.
template <int HD>
__global__ __launch_bounds__(2 * HD) void append_kernel(AppendParams p) {
    constexpr int kPer = HD / 8, kThreadsHere = 2 * HD;  // threads of a token or head
    __shared__ float red[kThreadsHere / 64];
    __shared__ __align__(16) uint8_t vt[HD * kKvBlock];
    __shared__ __align__(16) float cs[HD / 2], sn[HD / 2];
    const AppendArgs& a = p.a;
    const PagedArgs& c = a.c;
    const int tid = threadIdx.x, u = tid % kPer, wv = tid >> 6, lane = tid & 63;
    const bool inter = a.rot.interleaved != 0;
    const int half = a.rot.n_rot / 2;
    const FourPairs at(u, a.rot.n_rot, HD, inter);
    auto normed = [&]<class T>(T(&x)[4], T(&y)[4], const float* gamma) {
        T ss = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss += x[j] * x[j] + y[j] * y[j];
        ss = lanes_sum<kPer>(ss);
        const T inv = root_inverse(ss / HD + static_cast<T>(a.eps));
        float gx[4], gy[4];
        if (gamma) at.load(gamma, gx, gy);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = gamma ? x[j] * inv * gx[j] : x[j] * inv;
            y[j] = gamma ? y[j] * inv * gy[j] : y[j] * inv;
        }
    };
    const uint32_t group = p.first + blockIdx.x;
    if (group >= p.kv_groups) {
        const int64_t b = group - p.kv_groups;
        const int row = static_cast<int>(b / p.head_groups), h = static_cast<int>(b % p.head_groups) * 16 + tid / kPer;
        const int s = find_seq(c.n_seqs, row, [&](int i) { return clamp_row(c, c.row_start[i]); });
        if (s < 0) return;
        const SeqRows r = seq_rows(c, s);
        if (row < r.row0 || row - r.row0 >= r.count) return;
        if (tid < half) {
            double cc, ss;
            turn_of(r.len + row - r.row0, a.rot.freqs[tid], a.rot.magnitude, cc, ss);
            cs[tid] = static_cast<float>(cc);
            sn[tid] = static_cast<float>(ss);
        }
        __syncthreads();
        if (h >= a.n_heads) return;
        const size_t head = (static_cast<size_t>(row) * a.n_heads + h) * HD;
        float x[4], y[4];
        at.load(a.q + head, x, y);
        if (a.norm) normed(x, y, a.q_gamma);
        if (4 * u < half) {
            float cc[4], ss[4];
            *reinterpret_cast<f32x4*>(cc) = reinterpret_cast<const f32x4*>(cs)[u];
            *reinterpret_cast<f32x4*>(ss) = reinterpret_cast<const f32x4*>(sn)[u];
            turn_pairs(x, y, cc, ss);
        }
        at.store(a.out_q + head, x, y);
        return;
    }
    const int which = group & 1, hk = (group >> 1) % c.n_kv;
    const int64_t slot = (group >> 1) / c.n_kv;
    auto first_slot = [&](int i) {
        const int32_t r = clamp_row(c, c.row_start[i]);
        return p.by_rows ? static_cast<int64_t>(r) : static_cast<int64_t>(r >> 4) + 2 * i;
    };
    const int s = find_seq(c.n_seqs, slot, first_slot);
    if (s < 0) return;
    const SeqRows r = seq_rows(c, s);
    const int64_t nth = slot - first_slot(s);
    if (r.count == 0 || nth < 0 || nth > (r.len + r.count - 1) / kKvBlock - r.len / kKvBlock) return;
    const int32_t base = (r.len / kKvBlock + static_cast<int32_t>(nth)) * kKvBlock;  // the block's first position
    const int64_t block = block_of(c, s, hk, base);
    if (block < 0) return;
    // the block's tokens [held, end) are new, those before are kept
    const int held = max(r.len - base, 0), end = min(r.len + r.count - base, kKvBlock), tok = tid / kPer;
    const bool is_new = tok >= held && tok < end;
    float* scale_at = c.scales + 2 * block + which;
    const float was = held ? *scale_at : 0.0f;
    const int row = r.row0 + base - r.len + tok;
    const size_t head = (static_cast<size_t>(row) * c.n_kv + hk) * HD;
    uint8_t* codes = (which ? c.v_pages : c.k_pages) + static_cast<size_t>(block) * (kKvBlock * HD);
    // old codes of V: eight tokens of a float (those of K are read where they move)
    uint2 old = make_uint2(0, 0);
    if (which) old = reinterpret_cast<const uint2*>(codes)[tid];
    float x[4] = {}, y[4] = {};
    if (is_new) {
        if (which) {
            *reinterpret_cast<f32x4*>(x) = reinterpret_cast<const f32x4*>(a.v + head)[2 * u];
            *reinterpret_cast<f32x4*>(y) = reinterpret_cast<const f32x4*>(a.v + head)[2 * u + 1];
        } else {
            at.load(a.k + head, x, y);
        }
    }
    if (!which) {
        // K in 64 bits up to its codes, so that they are the formula's (in 32 one in a million
        // is rounded to the other side; 2462 rows, 32 heads on 8 of 128: 27.5 us for 26.2)
        double dx[4], dy[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            dx[j] = x[j];
            dy[j] = y[j];
        }
        if (a.norm) normed(dx, dy, a.k_gamma);
        if (is_new && 4 * u < half) {
            double cc[4], ss[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) turn_of(base + tok, a.rot.freqs[4 * u + j], a.rot.magnitude, cc[j], ss[j]);
            turn_pairs(dx, dy, cc, ss);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = odd_float(dx[j]);
            y[j] = odd_float(dy[j]);
        }
    }
    float amax = 0.0f;
    if (is_new)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(finite_size(x[j]), finite_size(y[j])));
    amax = wave_max(amax);
    if (lane == 0) red[wv] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreadsHere / 64; ++i) amax = fmaxf(amax, red[i]);
    int e = scale_exp(amax);
    const int e_was = min(max(static_cast<int>(__builtin_bit_cast(uint32_t, was) >> 23 & 0xff) - 127, kLeastExp), kMostExp);
    if (held) e = max(e, e_was);
    const float inv = pow2(-e);
    // (a factor below 2^-126 leaves nothing of any code)
    const bool moves = held && e > e_was;
    const float f = moves ? (e - e_was < 126 ? pow2(e_was - e) : 0.0f) : 1.0f;
    if (tid == 0) *scale_at = pow2(e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[j] = to_code_range(x[j], inv);
        y[j] = to_code_range(y[j], inv);
    }
    if (!which) {
        uint32_t w0, w1;
        if (is_new) {
            // in the order of the thread's two float4
            w0 = inter ? four_codes(x[0], y[0], x[1], y[1]) : four_codes(x[0], x[1], x[2], x[3]);
            w1 = inter ? four_codes(x[2], y[2], x[3], y[3]) : four_codes(y[0], y[1], y[2], y[3]);
        } else {
            if (!moves || tok >= held) return;
            w0 = moved_codes(*reinterpret_cast<const uint32_t*>(codes + tok * HD + at.off_a), f);
            w1 = moved_codes(*reinterpret_cast<const uint32_t*>(codes + tok * HD + at.off_b), f);
        }
        *reinterpret_cast<uint32_t*>(codes + tok * HD + at.off_a) = w0;
        *reinterpret_cast<uint32_t*>(codes + tok * HD + at.off_b) = w1;
        return;
    }
    if (is_new) {
        const uint32_t w0 = four_codes(x[0], x[1], x[2], x[3]), w1 = four_codes(y[0], y[1], y[2], y[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vt[(8 * u + j) * kKvBlock + tok] = static_cast<uint8_t>(byte_of(w0, j));
            vt[(8 * u + 4 + j) * kKvBlock + tok] = static_cast<uint8_t>(byte_of(w1, j));
        }
    }
    __syncthreads();
    const uint2 fresh = reinterpret_cast<const uint2*>(vt)[tid];
    // of bytes t0 .. t0 + 3: those below `held` moved, those in [held, end) new, the others as they are
    auto mixed = [&](uint32_t was_w, uint32_t now, int t0) {
        auto below = [&](int n) {  // bytes of tokens below n
            const int k = min(max(n - t0, 0), 4);
            return k == 4 ? 0xffffffffu : (1u << 8 * k) - 1u;
        };
        const uint32_t kept = below(held), all = below(end);
        const uint32_t m = moves ? moved_codes(was_w, f) : was_w;
        return (m & kept) | (now & all & ~kept) | (was_w & ~all);
    };
    const int t0 = tid % 2 * 8;
    if (t0 < end && (moves || t0 + 8 > held))
        reinterpret_cast<uint2*>(codes)[tid] = make_uint2(mixed(old.x, fresh.x, t0), mixed(old.y, fresh.y, t0 + 4));
}

// ---- attention ----------------------------------------------------------------------
// S^T = K Q^T and O^T = V^T P^T on the matrix instructions, 64 keys a step: a query row
// stays in a lane column (lane % 16) from its scores to its output.  A step is four
// blocks; a 16-key product takes four tokens of each, so that the lanes of group
// lane / 16 hold the scores of all 16 tokens of one block, and read those tokens of
// V as 16 bytes of one float's row.
// Precision: codes are exact in fp16.  Queries go in as pairs of fp16 (22 bits, behind a
// power of two that takes the row's largest to 2^14), and so do weights, each times its
// block's value scale over the largest scale so far, `unit` (powers of two).  Scores, sums
// and outputs are held in 32 bits, maxima rounded up to whole numbers, so that rescaling is
// exact.  (A pair's last bit is 2^-24: a weight is kept to 2^-38 of the row's largest, or to
// 2^-22 where its block's scale is 2^16 below the unit.)  Where the scales are farther apart,
// and where sizes leave no bits, hard_steps goes on.
constexpr int kAttnThreads = 256, kAttnWaves = 4;
__device__ __forceinline__ u32x4 four(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return u32x4{a, b, c, d}; }
constexpr float kInf = __builtin_inff();

// Over the four lanes of a column: lanes 16 apart, then 32 apart.  The swap of two copies
// leaves one of each pair in the first, the other in the second.
template <class F>
__device__ __forceinline__ float over_column(float v, F&& f) {
    const auto a = __builtin_amdgcn_permlane16_swap(as_bits(v), as_bits(v), false, false);
    v = f(as_float(a[0]), as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(as_bits(v), as_bits(v), false, false);
    return f(as_float(b[0]), as_float(b[1]));
}
__device__ __forceinline__ float xor_max(float v) {
    return over_column(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float xor_sum(float v) {
    return over_column(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ f16x8 codes_f16(uint32_t w0, uint32_t w1) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// 0x80 in every byte of w that is a NaN
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ u32x4 without_nan(u32x4 x) {
    auto zeros = [](uint32_t w) { return w & ~((nan_bytes(w) >> 7) * 0xffu); };
    return four(zeros(x.x), zeros(x.y), zeros(x.z), zeros(x.w));
}

struct PagedParams {
    PagedArgs c;
    const float* q;
    float* out;
    float2* part_ml;  // [part][row] maximum, sum
    float* part_o;    // [part][row][HD], divided by the sum
    int32_t n_heads, group, sw;
    int32_t target;   // work-groups that a split aims at
    bool split;       // whether keys are split
    int32_t units;    // that there is place for
    uint32_t first;   // work-group of the launch
    float scale;      // |attn_scale| log2(e), 1 for 0
    float sign;       // attn_scale's, 0 for 0
};
constexpr int kMostParts = 128;  // of a row
constexpr int kLeastSteps = 4;   // of a part

// The work of a call.  Rows of a sequence and KV head are numbered token by token,
// `group` heads each, and cut into tiles of R; a tile's steps of 64 keys are cut into
// equal parts of at most `per`, so many that the whole call's are about p.target work-groups'
// (whatever the lengths are: they are read here).  Units, a tile's part each, are numbered
// sequence by sequence.
struct Unit {
    int seq, tile, part, n_parts, per;
    int64_t first;  // number of the tile's first unit
    SeqRows r;
    // where part k of a tile of `steps` (2^24 at most) begins; parts behind those of `per` are empty
    __device__ __forceinline__ int begin(int k, int steps) const {
        const uint32_t n = static_cast<uint32_t>((steps - 1) / per) + 1;  // (128 at most)
        return static_cast<int>(min(static_cast<uint32_t>(k), n) * static_cast<uint32_t>(steps) / n);
    }
};
// The first key that a row at pos sees
__device__ __forceinline__ int32_t low_of(const PagedParams& p, int32_t pos) {
    return p.sw > 0 ? max(pos - p.sw + 1, 0) : 0;
}
// A sequence's tiles, and the steps of 64 keys that a tile may meet: up to the sequence's
// last key, and with a window no more than its tokens' windows can lie in.
struct SeqWork {
    int tiles, steps;
    SeqRows r;
};
template <int R>
__device__ __forceinline__ SeqWork seq_work(const PagedParams& p, int s) {
    SeqWork w{0, 0, {0, 0, 0}};
    if (s >= p.c.n_seqs) return w;
    w.r = seq_rows(p.c, s);
    w.tiles = (w.r.count * p.group + R - 1) / R;
    if (w.tiles == 0) return w;
    w.steps = (w.r.len + w.r.count + 63) / 64 - low_of(p, w.r.len) / 64;
    if (p.sw > 0) w.steps = min(w.steps, (min(p.sw, 1 << 30) + R / p.group + 63) / 64 + 1);
    return w;
}
// Sum over the lanes up to this one: row_shr by 1, 2, 4 and 8 within rows of 16, then the
// rows' totals carried up, as in wave_sum_lane63.  Sums stop at INT_MAX (a row_start that
// does not ascend may count any number).
__device__ __forceinline__ int add_up(int a, int b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int dpp_add_int(int v) {
    return add_up(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xf, false));
}
__device__ __forceinline__ int wave_prefix(int v) {
    v = dpp_add_int<0x111>(v);
    v = dpp_add_int<0x112>(v);
    v = dpp_add_int<0x114>(v);
    v = dpp_add_int<0x118>(v);
    v = dpp_add_int<0x142, 0xa>(v);
    return dpp_add_int<0x143, 0xc>(v);
}
// Unit `index` of the call (or, by_tile, the first unit of tile `index`), by a wave; false
// if there is none.
template <int R, bool BY_TILE>
__device__ __forceinline__ bool find_unit(const PagedParams& p, int index, Unit& u) {
    const int lane = threadIdx.x & 63;
    constexpr int kAll = 1 << 26;  // (more steps than there can be)
    if (!BY_TILE && !p.split && p.c.n_seqs > 64) {
        // tiles have places from row_start[s] group / R + s on: as many as there can be
        auto first = [&](int s) { return static_cast<int64_t>(clamp_row(p.c, p.c.row_start[s])) * p.group / R + s; };
        const int s = find_seq(p.c.n_seqs, index, first);
        if (s < 0) return false;
        const SeqWork w = seq_work<R>(p, s);
        const int64_t tile = index - first(s);
        if (tile < 0 || tile >= w.tiles) return false;
        u.seq = s;
        u.tile = static_cast<int>(tile);
        u.part = 0;
        u.n_parts = 1;
        u.per = kAll;
        u.first = index;
        u.r = w.r;
        return true;
    }
    SeqWork w = seq_work<R>(p, lane);
    int per = kAll;
    if (p.split) {
        float total = 0.0f;  // (of 24 bits: it only sets the split)
        int most = 0;
        for (int s0 = 0;;) {
            total += static_cast<float>(w.tiles) * static_cast<float>(w.steps);
            most = max(most, w.steps);
            s0 += 64;
            if (s0 >= p.c.n_seqs) break;
            w = seq_work<R>(p, s0 + lane);
        }
        total = wave_sum(total);
        most = static_cast<int>(wave_max(static_cast<float>(most)));  // (2^24 at most)
        per = max(max(kLeastSteps, (most + kMostParts - 1) / kMostParts),
                  static_cast<int>(ceilf(fminf(total * static_cast<float>(p.c.n_kv) / static_cast<float>(p.target), 1 << 26))));
        if (p.c.n_seqs > 64) w = seq_work<R>(p, lane);
    }
    int seq = lane;
    // Few long parts end unevenly: those of many rows are in falling order (four prompts as
    // above 272 -> 241 us, 16 of 64 to 200 tokens behind up to 6000 250 -> 222).
    if (R >= 64 && p.split && p.c.n_seqs > 1 && p.c.n_seqs <= 64) {
        const int parts = w.steps ? (w.steps - 1) / per + 1 : 1, each = w.steps ? (w.steps - 1) / parts + 1 : 0;
        int rank = 0;
        for (int l = 0; l < p.c.n_seqs; ++l) {
            const int o = __builtin_amdgcn_readlane(each, l);
            rank += o > each || (o == each && l < lane);
        }
        seq = __builtin_amdgcn_ds_permute(4 * (lane < p.c.n_seqs ? rank : lane), lane);
        auto moved = [&](int v) { return __shfl(v, seq, 64); };
        w = SeqWork{moved(w.tiles), moved(w.steps), {moved(w.r.row0), moved(w.r.count), moved(w.r.len)}};
    }
    int units = 0, tiles = 0;  // of the sequences before
    for (int s0 = 0; s0 < p.c.n_seqs; s0 += 64) {
        if (s0) {
            seq = s0 + lane;
            w = seq_work<R>(p, seq);
        }
        const int parts = w.steps ? (w.steps - 1) / per + 1 : 0;
        const int64_t own = static_cast<int64_t>(w.tiles) * parts;
        const int to_unit = add_up(units, wave_prefix(static_cast<int>(min(own, int64_t{0x7fffffff}))));
        const int to_tile = BY_TILE ? add_up(tiles, wave_prefix(w.tiles)) : 0;
        const uint64_t past = __ballot((BY_TILE ? to_tile : to_unit) > index);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            auto before = [&](int v, int none) { return l ? __builtin_amdgcn_readlane(v, l - 1) : none; };
            u.seq = of(seq);
            u.n_parts = of(parts);
            u.per = (of(w.steps) - 1) / u.n_parts + 1;
            u.r = SeqRows{of(w.r.row0), of(w.r.count), of(w.r.len)};
            const int first = before(to_unit, units);
            if constexpr (BY_TILE) {
                u.tile = index - before(to_tile, tiles);
                u.part = 0;
            } else {
                u.tile = (index - first) / u.n_parts;
                u.part = index - first - u.tile * u.n_parts;
            }
            u.first = first + static_cast<int64_t>(u.tile) * u.n_parts;
            if (R >= 64) u.tile = of(w.tiles) - 1 - u.tile;  // (the last tiles see the most keys)
            return true;
        }
        units = __builtin_amdgcn_readlane(to_unit, 63);
        if constexpr (BY_TILE) tiles = __builtin_amdgcn_readlane(to_tile, 63);
    }
    return false;
}

// Rows of queries as the products take them: lane (n, g) has floats 64 i + 16 g + 0 .. 15
// of row n, as the keys' lanes do, in units of 2^exp.  The scale's sign goes into them, so
// that the factor of their products is positive and keeps the scores' order.
template <int HD>
__device__ __forceinline__ void split_queries(const float* q, int g, float sign, f16x8 (&qh)[HD / 32],
                                              f16x8 (&ql)[HD / 32], int& exp) {
    f32x4 v[HD / 64][4];
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[i][j] = *reinterpret_cast<const f32x4*>(q + 64 * i + 16 * g + 4 * j);
#pragma unroll
            for (int k = 0; k < 4; ++k) most = fmaxf(most, fabsf(v[i][j][k]));
        }
    most = xor_max(most);
    int e = 0;
    (void)frexpf(most, &e);
    e = most > 0.0f && most < kInf ? e - 14 : 0;
    exp = e;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = ldexpf(sign * v[i][j / 4][j % 4], -e);
            const _Float16 h = static_cast<_Float16>(x);
            qh[2 * i + j / 8][j % 8] = h;
            ql[2 * i + j / 8][j % 8] = static_cast<_Float16>(x - static_cast<float>(h));
        }
}

// Maxima up to which a weight is 2^(f s - (use - up)) in one fma: use - up is exact, and f s,
// not rounded there, at most 1/4 above use, which is.  (From 2^24 on use - up would be rounded
// by 1 and more, and equal scores of two blocks weigh differently; from 2^25 on f s may lie so
// far above use that a weight is infinite in fp16, and later so far below that all are 0.)
constexpr float kMostOneFma = 0x1p22f;

// A row's running maximum, sum (of this lane's keys) and output, in units of 2^(unit - 14).
template <int HD>
struct PagedRow {
    float m = -kInf, l = 0.0f;
    f32x4 o[HD / 16];
    __device__ PagedRow() {
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // A step's scores, f s for the `seen` of this lane's 16 keys: the others to -inf, the
    // maximum raised, sum and output rescaled to it (and the output by `units`).  Returns
    // the maximum to weigh by, and in `large` whether one was raised past kMostOneFma.
    __device__ __forceinline__ float raise(f32x4 (&s)[4], float f, uint32_t seen, bool full, float units, bool& large) {
        float most = -kInf;
        if (!full)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j / 4][j % 4] = seen >> j & 1u ? s[j / 4][j % 4] : -kInf;
#pragma unroll
        for (int j = 0; j < 16; ++j) most = fmaxf(most, s[j / 4][j % 4]);
        const float mx = fmaxf(m, ceilf(xor_max(most * f))), use = mx == -kInf ? 0.0f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - use), by = alpha * units;
        m = mx;
        l *= alpha;
        // (most steps leave every row's maximum as it is)
        if (__any(by != 1.0f)) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[d] *= by;
            large = large || __any(fabsf(use) > kMostOneFma);
        }
        return use;
    }
};
// o += the values a and b (of tokens 0 to 7 and 8 to 15 of the lane's block) by their weights
__device__ __forceinline__ void add_values(f32x4& o, f16x8 a, f16x8 b, const f16x8 (&hi)[2], const f16x8 (&lo)[2]) {
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, lo[0], o, 0, 0, 0);
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, lo[1], o, 0, 0, 0);
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi[0], o, 0, 0, 0);
    o = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, hi[1], o, 0, 0, 0);
}
// Weights w(product) of this lane's 16 keys as fp16 pairs; returns their sum.  Two a
// conversion, and the rest as one mixed fma that reads its half in place (written out, as
// the compiler converts every half back, alone).
template <class Weight>
__device__ __forceinline__ float weigh(const f32x4 (&s)[4], f16x8 (&hi)[2], f16x8 (&lo)[2], Weight&& w) {
    float sum = 0.0f;
    uint32_t h[8], r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = w(s[j / 2][2 * j % 4]), y = w(s[j / 2][2 * j % 4 + 1]);
        sum += x + y;
        h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2));
        float a, b;
        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(a) : "v"(x), "v"(h[j]));
        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(b) : "v"(y), "v"(h[j]));
        r[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        hi[k] = __builtin_bit_cast(f16x8, four(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]));
        lo[k] = __builtin_bit_cast(f16x8, four(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]));
    }
    return sum;
}
// The largest of the four lane groups' values
__device__ __forceinline__ int most_of_groups(int v) {
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
constexpr int kNoUnit = -1000;

// Keys at .. at + 15 that the row at pos sees, one bit each
__device__ __forceinline__ uint32_t below_bits(int32_t at, int32_t n) {  // those below n
    return (1u << min(max(n - at, 0), 16)) - 1u;
}
__device__ __forceinline__ uint32_t seen_bits(int32_t at, int32_t pos, int32_t sw) {
    const uint32_t in = below_bits(at, pos + 1);
    return sw > 0 ? in & ~below_bits(at, max(pos - sw + 1, 0)) : in;
}
// What a wave's rows are, and where they look.
template <int HD, int RT>
struct WaveRows {
    f16x8 qh[RT][HD / 32], ql[RT][HD / 32];
    int exp[RT];  // of its queries' units
    int32_t pos[RT];
    int32_t pos_first, pos_last, low_first, low_last;  // of its rows; the first keys that they see
    __device__ __forceinline__ void look(const PagedParams& p, const SeqRows& r, int row_lo, int row_hi) {
        pos_first = r.len + row_lo / p.group;
        pos_last = r.len + (row_hi - 1) / p.group;
        low_first = low_of(p, pos_first);
        low_last = low_of(p, pos_last);
    }
    // the last key of a step, and its first, are seen by every row
    __device__ __forceinline__ bool whole(int32_t k0) const { return k0 + 63 <= pos_first && k0 >= low_last; }
    // keys at .. at + 15 may be seen by some row
    __device__ __forceinline__ bool meets(int32_t at) const { return at <= pos_last && at + 16 > low_first; }
    // s += the keys' floats 64 i + 16 g .. by the queries'
    __device__ __forceinline__ void score(f32x4& s, u32x4 x, int i, int rt) const {
        const f16x8 a = codes_f16(x.x, x.y), b = codes_f16(x.z, x.w);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[rt][2 * i], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, ql[rt][2 * i + 1], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[rt][2 * i], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qh[rt][2 * i + 1], s, 0, 0, 0);
    }
};
// 0xff for the bytes of tokens that are in `seen`
__device__ __forceinline__ uint32_t bytes_of(uint32_t seen, int t0) {
    return ((seen >> t0 & 1u) * 0xffu) | ((seen >> (t0 + 1) & 1u) * 0xff00u) |
           ((seen >> (t0 + 2) & 1u) * 0xff0000u) | ((seen >> (t0 + 3) & 1u) * 0xff000000u);
}
__device__ __forceinline__ u32x4 only_seen(u32x4 x, uint32_t seen) {
    return four(x.x & bytes_of(seen, 0), x.y & bytes_of(seen, 4), x.z & bytes_of(seen, 8), x.w & bytes_of(seen, 12));
}
__device__ __forceinline__ int scale_exponent(float scale) { return static_cast<int>(as_bits(scale) >> 23 & 0xffu) - 127; }
// What a product of a row in units of 2^row_exp and a block of keys counts as a score.  From
// the exponents' sum, as either's float alone may be subnormal where both make an ordinary
// number; and never 0, by which a hidden key's -inf would be NaN, or infinite, by which a
// product of 0 would.
__device__ __forceinline__ float score_factor(float scale, int row_exp, bool there, float key_scale) {
    const float f = ldexpf(scale, row_exp + (there ? scale_exponent(key_scale) : 0));
    return fminf(fmaxf(f, 0x1p-126f), 0x1.fffffep127f);
}

// Whether the blocks' value scales allow one unit for all: a scale of more than 16 below
// the unit would leave bits of its weights behind in fp16, and one of more than 16 above it
// those of weights that are small by now (but above the least scale, of blocks of zeros: 100,
// by which outputs can be multiplied without loss).  Raises the unit; `units` is what outputs
// are to be multiplied by.
__device__ __forceinline__ bool one_unit(bool there, float scale, int& unit, float& units) {
    const int own = scale_exponent(scale);
    const int top = max(unit, most_of_groups(there ? own : kNoUnit)), rise = unit == kLeastExp ? 100 : 16;
    if (-most_of_groups(there ? -own : kNoUnit) < top - 16 || (unit != kNoUnit && top > unit + rise)) return false;
    units = ldexpf(1.0f, max(unit - top, -200));
    unit = top;
    return true;
}
// A step of RT row tiles, from their products with the keys on: sc are the scales of this
// lane's block, if it is there, and values(d) the codes of its float 16 d + n.  False if a
// maximum is larger than that: then nothing but maxima, sums and outputs in their units is
// changed, so that the step can be taken again.
template <int HD, int RT, class Values>
__device__ __forceinline__ bool take_step(PagedRow<HD> (&st)[RT], f32x4 (&s)[RT][4], float scale, const int (&exp)[RT],
                                          float2 sc, bool there, bool full, const uint32_t (&seen)[RT], int unit,
                                          float units, Values&& values) {
    f16x8 hi[RT][2], lo[RT][2];
    const int up = there ? scale_exponent(sc.y) - unit + 14 : 0;
    float sum[RT];
    bool large = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float f = score_factor(scale, exp[rt], there, sc.x), use = st[rt].raise(s[rt], f, seen[rt], full, units, large);
        __builtin_amdgcn_sched_barrier(0);
        const float base = use - static_cast<float>(up);
        sum[rt] = weigh(s[rt], hi[rt], lo[rt], [&](float x) { return __builtin_amdgcn_exp2f(fmaf(x, f, -base)); });
        __builtin_amdgcn_sched_barrier(0);
    }
    if (large) return false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) st[rt].l += ldexpf(sum[rt], -up);
    if (RT > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
        if (RT > 1 && d % 2 == 0) __builtin_amdgcn_sched_barrier(0);
        const u32x4 x = values(d);
        const f16x8 a = codes_f16(x.x, x.y), b = codes_f16(x.z, x.w);
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                st[rt].o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h & 1 ? b : a, h < 2 ? lo[rt][h] : hi[rt][h - 2],
                                                                     st[rt].o[d], 0, 0, 0);
    }
    return true;
}
// The distance of a score of any size to its row's maximum: f s is rounded before that is
// taken off, so that the largest's is 0 and equal scores' are equal
__device__ __forceinline__ float below_most(float s, float f, float use) {
#pragma clang fp contract(off)
    const float score = s * f;
    return score - use;
}
// The same of one row tile for every step, from `step` on, one after the other: for those with
// large scores, those not seen whole with NaN codes among the values, and those whose values'
// scales are far apart.  Rows that do not see a NaN code must not meet it (0 NaN is NaN), so
// these are taken out and met by a product of their own.  From the first step with scales far
// apart on, outputs are in one unit that holds a sum of the largest values as of the smallest,
// and blocks are taken by their scales, 2^16 at a time, with weights by the row's maximum
// among them: what a block adds has its own 22 bits, whatever others hold and weigh.
// (64 sequences of 100 to 8000 tokens, 32 heads on 8 of 128, the four prompts below: 112 and
// 235 us, with large scores from the start 196 and 498, with a block 2^30 above the others 160
// and 496, with every block's scale far from the next one's 300 and 786.  Inside the loops of
// the others this would cost them 60 registers, and here two row tiles at once spilled: the
// prompts 248.)
template <int HD>
__device__ __forceinline__ void hard_steps(const PagedParams& p, const int32_t* table, int hk, const WaveRows<HD, 1>& w,
                                           PagedRow<HD>& st, int& unit, int step, int every, int end) {
    const PagedArgs& c = p.c;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    // 448 2^120 of every key, by 2^(far - 14), is below 2^127
    const int far = 48 - __builtin_clz(w.pos_last + 1);
    bool wide = false;
    for (; step < end; step += every) {
        const int32_t k0 = 64 * step, at_k = k0 + 16 * (n >> 2), at_v = k0 + 16 * g;
        const int64_t bk = block_in(c, page_at(c, table, at_k), hk, at_k);
        const int64_t bv = block_in(c, page_at(c, table, at_v), hk, at_v);
        const uint8_t* kp = c.k_pages + max(bk, int64_t{0}) * (kKvBlock * HD) + (n & 3) * HD + 16 * g;
        const uint8_t* vp = c.v_pages + max(bv, int64_t{0}) * (kKvBlock * HD) + 16 * n;
        const float2 sc = *reinterpret_cast<const float2*>(c.scales + 2 * max(bv, int64_t{0}));
        const bool there = bv >= 0 && w.meets(at_v);
        const bool full = w.whole(k0) && __ballot(there) == ~uint64_t{0};
        const int own = scale_exponent(sc.y);
        float units = 1.0f;
        if (!wide && !one_unit(there, sc.y, unit, units)) {
            wide = true;
            if (unit != kNoUnit) units = ldexpf(1.0f, unit - far);
            unit = far;
        }
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < HD / 64; ++i)
                w.score(s[j], *reinterpret_cast<const u32x4*>(kp + 4 * j * HD + 64 * i), i, 0);
        }
        const uint32_t seen = there ? seen_bits(at_v, w.pos[0], p.sw) : 0u;
        bool large = false;
        const float f = score_factor(p.scale, w.exp[0], there, sc.x), use = st.raise(s, f, seen, full, units, large);
        f16x8 hi[2], lo[2];
        auto values = [&](int d, auto&& add) {
            u32x4 x = *reinterpret_cast<const u32x4*>(vp + 256 * d);
            if (!full) x = without_nan(x);
            add(codes_f16(x.x, x.y), codes_f16(x.z, x.w));
            __builtin_amdgcn_sched_barrier(0);
        };
        if (!wide) {
            const int up = there ? own - unit + 14 : 0;
            const float off = static_cast<float>(up), base = use - off;
            const float sum = __any(fabsf(use) > kMostOneFma)
                                  ? weigh(s, hi, lo, [&](float x) { return __builtin_amdgcn_exp2f(below_most(x, f, use) + off); })
                                  : weigh(s, hi, lo, [&](float x) { return __builtin_amdgcn_exp2f(fmaf(x, f, -base)); });
            st.l += ldexpf(sum, -up);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                values(d, [&](f16x8 a, f16x8 b) { add_values(st.o[d], a, b, hi, lo); });
        }
        for (bool left = wide && there; __any(left);) {
            const int t = most_of_groups(left ? own : kNoUnit);
            const bool now = left && own >= t - 16;
            left = left && !now;
            float most = -kInf;
#pragma unroll
            for (int j = 0; j < 16; ++j) most = fmaxf(most, s[j / 4][j % 4]);
            most = ceilf(xor_max(now ? most * f : -kInf));
            // (a row that sees none of these blocks: nothing is added)
            const float base = most == -kInf ? 0.0f : most, off = now ? static_cast<float>(own - t + 14) : -kInf;
            const int down = static_cast<int>(fmaxf(most - use, -1000.0f));
            const float sum = weigh(s, hi, lo, [&](float x) { return __builtin_amdgcn_exp2f(below_most(x, f, base) + off); });
            st.l += ldexpf(sum, down + (now ? t - own - 14 : 0));
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                values(d, [&](f16x8 a, f16x8 b) {
                    f32x4 part = {0.0f, 0.0f, 0.0f, 0.0f};
                    add_values(part, a, b, hi, lo);
#pragma unroll
                    for (int r = 0; r < 4; ++r) st.o[d][r] += ldexpf(part[r], down + t - far);
                });
        }
        if (full) continue;
        auto ones = [&](int j) {
            return ((seen >> j & 1u) ? 0x3c00u : 0u) | ((seen >> (j + 1) & 1u) ? 0x3c000000u : 0u);
        };
        const f16x8 first = __builtin_bit_cast(f16x8, four(ones(0), ones(2), ones(4), ones(6)));
        const f16x8 second = __builtin_bit_cast(f16x8, four(ones(8), ones(10), ones(12), ones(14)));
        auto marks = [](uint32_t v) { return (nan_bytes(v) >> 7) * 0x38u; };  // (0x38: one)
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(vp + 256 * d);
            f32x4 count = {0.0f, 0.0f, 0.0f, 0.0f};
            count = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16(marks(x.x), marks(x.y)), first, count, 0, 0, 0);
            count = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16(marks(x.z), marks(x.w)), second, count, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (count[r] > 0.0f) st.o[d][r] = __builtin_nanf("");
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}
// A lane's part of a row: its sum over all keys, and the factor of its output
__device__ __forceinline__ float2 sum_and_share(float l, int unit) {
    l = xor_sum(l);
    return make_float2(l, l != 0.0f ? ldexpf(1.0f / l, unit == kNoUnit ? 0 : unit - 14) : 0.0f);
}
__device__ __forceinline__ float* row_of(float* base, const PagedParams& p, const SeqRows& r, int hk, int row, int hd) {
    return base + ((static_cast<size_t>(r.row0) + row / p.group) * p.n_heads + hk * p.group + row % p.group) * hd;
}

// Few rows a sequence (a decode step): a work-group has 16 rows, and its four waves take
// every fourth step each, from memory straight into registers, as no wave needs another's
// keys.  Bound by reading the cache: 64 sequences of 100 to 8000 tokens, 8 KV heads of 128,
// 538 MB in 106 us (5.1 TB/s; the same loads alone take as long); one of 60001 tokens, 4 KV
// heads, 62 MB in 16 us, of which 3 are the start and the last wave's end; one of 1000 tokens
// 7.5 us of latencies: sequence, page, codes, products, parts.
// With ALONE, where they are many and short (nothing is split), each wave has 16 rows of its
// own, all steps of them: no wave is without keys.
template <int HD, bool ALONE>
__global__ __launch_bounds__(kAttnThreads, HD == 256 ? 1 : 2) void paged_keys_kernel(PagedParams p) {
    constexpr int R = 16, kSlices = HD / 64, kDims = HD / 16, kEvery = ALONE ? 1 : kAttnWaves;
    // the waves' parts of a row (a row of HD + 4 floats: no two rows on the same banks)
    __shared__ __align__(16) float os[ALONE ? 1 : kAttnWaves][R][HD + 4];
    __shared__ float2 mls[ALONE ? 1 : kAttnWaves][R];
    const PagedArgs& c = p.c;
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t group = p.first + blockIdx.x, place = ALONE ? kAttnWaves * group + wv : group;
    const int hk = place % c.n_kv, unit = place / c.n_kv;
    Unit u;
    if (!find_unit<R, false>(p, unit, u)) return;
    const int rows = u.r.count * p.group, row_lo = u.tile * R, row_hi = min(row_lo + R, rows);
    WaveRows<HD, 1> w;
    w.look(p, u.r, row_lo, row_hi);
    const int first = w.low_first / 64, steps = w.pos_last / 64 + 1 - first;
    const int step0 = first + u.begin(u.part, steps), step1 = first + u.begin(u.part + 1, steps);
    const int32_t* table = c.pages + static_cast<size_t>(u.seq) * c.max_pages;
    int step = ALONE ? step0 : step0 + wv;
    // keys of a step that this lane's blocks begin at: of K, whose rows it loads, and of V
    const int at_k = 16 * (n >> 2), at_v = 16 * g;
    int32_t page_k = page_at(c, table, 64 * step + at_k), page_v = page_at(c, table, 64 * step + at_v);
    const int row = min(row_lo + n, rows - 1);
    w.pos[0] = u.r.len + row / p.group;
    split_queries<HD>(row_of(const_cast<float*>(p.q), p, u.r, hk, row, HD), g, p.sign, w.qh[0], w.ql[0], w.exp[0]);
    PagedRow<HD> st[1];
    int unit_exp = kNoUnit;
    // (a block that is not there: the first one is read, and hidden)
    u32x4 kw[4][kSlices], vw[kDims];
    auto load_k = [&](int64_t b) {
        const uint8_t* from = c.k_pages + max(b, int64_t{0}) * (kKvBlock * HD) + (n & 3) * HD + 16 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < kSlices; ++i) kw[j][i] = *reinterpret_cast<const u32x4*>(from + 4 * j * HD + 64 * i);
    };
    float2 scale;
    auto in_order = [] { asm volatile("" ::: "memory"); };
    auto load_v = [&](int64_t b) {
        scale = *reinterpret_cast<const float2*>(c.scales + 2 * max(b, int64_t{0}));
        in_order();
        const uint8_t* from = c.v_pages + max(b, int64_t{0}) * (kKvBlock * HD) + 16 * n;
#pragma unroll
        for (int d = 0; d < kDims; ++d) vw[d] = *reinterpret_cast<const u32x4*>(from + 256 * d);
    };
    // Loads return in the order of their issue, so that what is waited for first goes out
    // first: the pages of the step after next, the next step's keys while this one's scores
    // are weighed, its values when this one's are used up.  Behind the last step the
    // first block is read, from the caches.
    int64_t bv = block_in(c, page_v, hk, 64 * step + at_v);
    load_k(block_in(c, page_k, hk, 64 * step + at_k));
    page_k = page_at(c, table, 64 * (step + kEvery) + at_k);
    page_v = page_at(c, table, 64 * (step + kEvery) + at_v);
    in_order();
    load_v(bv);
    for (; step < step1; step += kEvery) {
        const int32_t k0 = 64 * step, next = step + kEvery;
        f32x4 s[1][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[0][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kSlices; ++i) w.score(s[0][j], kw[j][i], i, 0);
        }
        const bool there = bv >= 0 && w.meets(k0 + at_v);
        const bool full = w.whole(k0) && __ballot(there) == ~uint64_t{0};
        const uint32_t seen[1] = {there ? seen_bits(k0 + at_v, w.pos[0], p.sw) : 0u};
        const bool more = next < step1;
        const int64_t next_k = more ? block_in(c, page_k, hk, 64 * next + at_k) : 0;
        bv = more ? block_in(c, page_v, hk, 64 * next + at_v) : 0;
        page_k = page_at(c, table, 64 * (next + kEvery) + at_k);
        page_v = page_at(c, table, 64 * (next + kEvery) + at_v);
        load_k(next_k);
        // values that no row sees may hold anything
        u32x4 seen_bytes = four(~0u, ~0u, ~0u, ~0u);
        if (!full) {
            const uint32_t some = there ? seen_bits(k0 + at_v, w.pos_last, 0) & ~below_bits(k0 + at_v, w.low_first) : 0u;
            seen_bytes = only_seen(seen_bytes, some);
            uint32_t bad = 0;
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                const u32x4 x = vw[d] & seen_bytes;
                bad |= nan_bytes(x.x) | nan_bytes(x.y) | nan_bytes(x.z) | nan_bytes(x.w);
            }
            if (__any(bad != 0)) break;
        }
        float units;  // (raised last: the outputs follow in this step, or not at all)
        if (!one_unit(there, scale.y, unit_exp, units)) break;
        if (!take_step<HD, 1>(st, s, p.scale, w.exp, scale, there, full, seen, unit_exp, units,
                              [&](int d) { return vw[d] & seen_bytes; }))
            break;
        load_v(bv);
        // (otherwise the compiler joins these loads with those before the loop, at its top)
        asm volatile("; the next step's values are on their way" ::: "memory");
    }
    if (step < step1) hard_steps<HD>(p, table, hk, w, st[0], unit_exp, step, kEvery, step1);
    // divided by the sum here, before the parts' weights meet the values
    const float2 ls = sum_and_share(st[0].l, unit_exp);
    if constexpr (ALONE) {
        if (row_lo + n >= row_hi) return;
        float* to = row_of(p.out, p, u.r, hk, row_lo + n, HD);
#pragma unroll
        for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(to + 16 * d + 4 * g) = st[0].o[d] * ls.y;
        return;
    }
    if (g == 0) mls[wv][n] = make_float2(st[0].m, ls.x);
#pragma unroll
    for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(&os[wv][n][16 * d + 4 * g]) = st[0].o[d] * ls.y;
    __syncthreads();
    // (a unit's parts: [unit][KV head][row])
    const size_t part_row = (static_cast<size_t>(unit) * c.n_kv + hk) * R;
    for (int i = tid; i < (row_hi - row_lo) * (HD / 4); i += kAttnThreads) {
        const int r = i / (HD / 4), d = i % (HD / 4);
        float M = -kInf, L = 0.0f, wt[kAttnWaves];
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k) M = fmaxf(M, mls[k][r].x);
        const float use = M == -kInf ? 0.0f : M;
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k) {
            wt[k] = mls[k][r].y * __builtin_amdgcn_exp2f(mls[k][r].x - use);
            L += wt[k];
        }
        const float share = L != 0.0f ? 1.0f / L : 0.0f;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k)
            if (wt[k] != 0.0f) x += (wt[k] * share) * *reinterpret_cast<const f32x4*>(&os[k][r][4 * d]);
        float* to = row_of(p.out, p, u.r, hk, row_lo + r, HD);
        if (u.n_parts > 1) {
            if (d == 0) p.part_ml[part_row + r] = make_float2(M, L);
            to = p.part_o + (part_row + r) * HD;
        }
        *reinterpret_cast<f32x4*>(to + 4 * d) = x;
    }
}

// Many rows (prompts): a wave has 16 RT rows of its own, a work-group four times as many.
// Bound by the issue of vector and matrix instructions, which share it (586 of them and 128
// products of two slots each a wave and step): four prompts of 300 to 700 tokens behind 1152
// to 3799, 32 heads on 8 of 128, 2 x 101 GFLOP in 245 us; in the loop 1050 TFLOP/s, of the
// 1315 that a large library product reaches; the rest are the parts' starts and ends.
// (32x32x16 products, half as many instructions: heads of 128 6% slower, of 256 34%, of 64
// 9% faster.)
// The codes of a step are staged in LDS for all of them, two steps in turn: the next one's
// are on their way from memory during a step, and laid down at its end, so that a step
// takes one barrier.
template <int HD, int RT>
__global__ __launch_bounds__(kAttnThreads, HD == 256 ? 1 : 2) void paged_rows_kernel(PagedParams p) {
    constexpr int R = 16 * RT * kAttnWaves, kSlices = HD / 64, kDims = HD / 16;
    constexpr int kChunks = HD / 16;  // 16-byte chunks of a key; of a step there are 64 times as many
    __shared__ __align__(16) u32x4 ks[2][64 * kChunks], vs[2][64 * kChunks];
    __shared__ __align__(16) f16x8 qlow[RT * 2 * kSlices][kAttnThreads];  // the queries' low halves: they would take the registers that a step needs
    const PagedArgs& c = p.c;
    const int tid = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    const uint32_t place = p.first + blockIdx.x;
    const int hk = place % c.n_kv, unit = place / c.n_kv;
    Unit u;
    if (!find_unit<R, false>(p, unit, u)) return;
    const int rows = u.r.count * p.group, tile_lo = u.tile * R, tile_hi = min(tile_lo + R, rows);
    const int32_t* table = c.pages + static_cast<size_t>(u.seq) * c.max_pages;
    const int32_t tile_low = low_of(p, u.r.len + tile_lo / p.group);
    const int first = tile_low / 64, steps = (u.r.len + (tile_hi - 1) / p.group) / 64 + 1 - first;
    const int step0 = first + u.begin(u.part, steps), step1 = first + u.begin(u.part + 1, steps);
    // this wave's rows (the last one again where there are fewer) and what they see
    const int row_lo = min(tile_lo + 16 * RT * wv, rows - 1), row_hi = min(row_lo + 16 * RT, rows);
    WaveRows<HD, RT> w;
    w.look(p, u.r, row_lo, row_hi);
    // K's chunk x of key t stands at chunk x ^ turn(t), so that the eight lanes that read at
    // once, keys 0 to 3 of two blocks, meet eight different columns of banks
    auto turn = [](int t) { return HD == 64 ? t & 3 : (t & 3) | (t >> 4 & 1) << 2; };
    // Thread tid stages chunks tid + 256 k of K and of V, which lie in one block for a wave
    u32x4 kw[kSlices], vw[kSlices];
    auto load_step = [&](int32_t page, int step) {
#pragma unroll
        for (int k = 0; k < kSlices; ++k) {
            const int at = tid + kAttnThreads * k, t = at / kChunks;
            const int b = __builtin_amdgcn_readfirstlane(t / kKvBlock);
            const int64_t blk = block_in(c, __builtin_amdgcn_readlane(page, 16 * b), hk, 64 * step + 16 * b);
            const size_t from = static_cast<size_t>(max(blk, int64_t{0})) * (kKvBlock * HD);
            kw[k] = *reinterpret_cast<const u32x4*>(c.k_pages + from + t % kKvBlock * HD + 16 * (at % kChunks ^ turn(t)));
            vw[k] = *reinterpret_cast<const u32x4*>(c.v_pages + from + 16 * (at % (16 * kChunks)));
        }
    };
    const int32_t tile_end = u.r.len + (tile_hi - 1) / p.group + 1;
    auto store_step = [&](int buf, int step) {
        // values that no row of the work-group sees may hold anything: zeros
        const bool inside = 64 * step >= tile_low && 64 * step + 64 <= tile_end;
#pragma unroll
        for (int k = 0; k < kSlices; ++k) {
            if (!inside) {
                const int at = 64 * step + 16 * __builtin_amdgcn_readfirstlane((tid + kAttnThreads * k) / (16 * kChunks));
                vw[k] = only_seen(vw[k], below_bits(at, tile_end) & ~below_bits(at, tile_low));
            }
            ks[buf][tid + kAttnThreads * k] = kw[k];
            vs[buf][tid + kAttnThreads * k] = vw[k];
        }
    };
    auto scale_of = [&](int64_t b) { return *reinterpret_cast<const float2*>(c.scales + 2 * max(b, int64_t{0})); };
    auto in_order = [] { asm volatile("" ::: "memory"); };
    if (step0 >= step1) {
        // (a part behind its tile's last key)
        for (int i = tid; i < tile_hi - tile_lo; i += kAttnThreads)
            p.part_ml[(static_cast<size_t>(unit) * c.n_kv + hk) * R + i] = make_float2(-kInf, 0.0f);
        return;
    }
    int32_t page = page_at(c, table, 64 * step0 + 16 * g);
    load_step(page, step0);
    int64_t bv = block_in(c, page, hk, 64 * step0 + 16 * g);
    float2 scale = scale_of(bv);
    page = page_at(c, table, 64 * (step0 + 1) + 16 * g);
    PagedRow<HD> st[RT];
    int unit_exp = kNoUnit, hard = -1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = min(row_lo + 16 * rt + n, rows - 1);
        w.pos[rt] = u.r.len + row / p.group;
        split_queries<HD>(row_of(const_cast<float*>(p.q), p, u.r, hk, row, HD), g, p.sign, w.qh[rt], w.ql[rt], w.exp[rt]);
#pragma unroll
        for (int k = 0; k < 2 * kSlices; ++k) qlow[2 * kSlices * rt + k][tid] = w.ql[rt][k];
    }
    store_step(0, step0);
    for (int step = step0; step < step1; ++step) {
        const int cur = (step - step0) & 1;
        const int32_t k0 = 64 * step, at_v = k0 + 16 * g;
        __syncthreads();
        // (behind the last step the first block is read, from the caches)
        const bool more = step + 1 < step1;
        const int64_t bv_now = bv;
        const float2 sc = scale;
        const int32_t page_next = more ? page : -1;
        load_step(page_next, step + 1);
        bv = block_in(c, page_next, hk, 64 * (step + 1) + 16 * g);
        scale = scale_of(bv);
        page = page_at(c, table, 64 * (step + 2) + 16 * g);
        in_order();
        if (k0 <= w.pos_last && k0 + 63 >= w.low_first && hard < 0) {
            const bool there = bv_now >= 0 && w.meets(at_v);
            const bool full = w.whole(k0) && __ballot(there) == ~uint64_t{0};
            const u32x4* values = vs[cur] + g * HD + n;  // float 16 d + n of the lane's block
            uint32_t bad = 0;
            if (!full)
#pragma unroll
                for (int d = 0; d < kDims; ++d) {
                    const u32x4 x = values[16 * d];
                    bad |= nan_bytes(x.x) | nan_bytes(x.y) | nan_bytes(x.z) | nan_bytes(x.w);
                }
            float units;
            if (__any(bad != 0) || !one_unit(there, sc.y, unit_exp, units)) {
                hard = step;
            } else {
                __builtin_amdgcn_s_setprio(1);  // (a wave with products to issue goes first: 260 -> 255 us)
                f32x4 s[RT][4];
#pragma unroll
                for (int i = 0; i < kSlices; ++i) {
                    f16x8 low[RT][2];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) low[rt][h] = qlow[2 * (kSlices * rt + i) + h][tid];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int t = 16 * (n >> 2) + 4 * j + (n & 3);
                        const u32x4 x = ks[cur][t * kChunks + ((4 * i + g) ^ turn(t))];
                        const f16x8 k[2] = {codes_f16(x.x, x.y), codes_f16(x.z, x.w)};
                        // (the row tiles in turn: a product waits for the one before it on its sums)
#pragma unroll
                        for (int h = 0; h < 4; ++h)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                s[rt][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                    k[h & 1], h < 2 ? low[rt][h] : w.qh[rt][2 * i + h - 2],
                                    i == 0 && h == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : s[rt][j], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
                uint32_t seen[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) seen[rt] = there ? seen_bits(at_v, w.pos[rt], p.sw) : 0u;
                if (!take_step<HD, RT>(st, s, p.scale, w.exp, sc, there, full, seen, unit_exp, units,
                                       [&](int d) { return values[16 * d]; }))
                    hard = step;
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (more) store_step(cur ^ 1, step + 1);
    }
    int unit_of[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) unit_of[rt] = unit_exp;
    if (hard >= 0)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            WaveRows<HD, 1> one;
#pragma unroll
            for (int k = 0; k < 2 * kSlices; ++k) {
                one.qh[0][k] = w.qh[rt][k];
                one.ql[0][k] = qlow[2 * kSlices * rt + k][tid];
            }
            one.exp[0] = w.exp[rt];
            one.pos[0] = w.pos[rt];
            one.look(p, u.r, row_lo, row_hi);
            hard_steps<HD>(p, table, hk, one, st[rt], unit_of[rt], hard, 1, min(step1, w.pos_last / 64 + 1));
        }
    const int own = tile_lo + 16 * RT * wv;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float2 ls = sum_and_share(st[rt].l, unit_of[rt]);
        const int row = own + 16 * rt + n;
        if (row >= rows) continue;
        float* to = row_of(p.out, p, u.r, hk, row, HD);
        if (u.n_parts > 1) {
            const size_t i = (static_cast<size_t>(unit) * c.n_kv + hk) * R + row - tile_lo;
            if (g == 0) p.part_ml[i] = make_float2(st[rt].m, ls.x);
            to = p.part_o + i * HD;
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(to + 16 * d + 4 * g) = st[rt].o[d] * ls.y;
    }
}

// out = sum_c w_c o_c / sum_c w_c with w_c = l_c 2^(m_c - M) over the parts c.  Bound by
// latency (a launch, the sequences, the parts: 2.9 to 5.4 us for decode steps) or by reading
// the parts (the four prompts 22 us).  In the attention's own launch, by the last work-group
// of a tile with device-scope accesses, it took 2 to 30 us longer.  HD / 4
// threads have a row's floats; up to kAtOnce parts they have the row to themselves, more
// parts are shared by the work-group, whose sums then meet in LDS.
template <int HD, int R>
__global__ __launch_bounds__(kAttnThreads) void paged_merge_kernel(PagedParams p) {
    constexpr int kCols = HD / 4, kWide = kAttnThreads / kCols, kAtOnce = 8;
    __shared__ __align__(16) f32x4 sums[kWide][kCols];
    __shared__ float2 mls[kWide];
    const PagedArgs& c = p.c;
    const int hk = blockIdx.x % c.n_kv, tile = blockIdx.x / c.n_kv;
    Unit u;
    if (!find_unit<R, true>(p, tile, u) || u.n_parts == 1 || u.first + u.n_parts > p.units) return;
    const int col = threadIdx.x % kCols, k0 = threadIdx.x / kCols;
    const int rows = min(u.r.count * p.group - u.tile * R, R);
    const size_t stride = static_cast<size_t>(c.n_kv) * R;
    // a row's parts first, first + every, ..: M, L and x, their mean
    struct Mean {
        float M = -kInf, L = 0.0f;
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    };
    auto parts_of = [&](int r, int first, int every) {
        const size_t base = (static_cast<size_t>(u.first) * c.n_kv + hk) * R + r;
        Mean s;
        for (int k1 = first; k1 < u.n_parts; k1 += every * kAtOnce) {
            float2 ml[kAtOnce];
            f32x4 v[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const size_t at = base + static_cast<size_t>(min(k1 + i * every, u.n_parts - 1)) * stride;
                ml[i] = p.part_ml[at];
                v[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * HD + 4 * col);
            }
            float mx = s.M;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) mx = fmaxf(mx, ml[i].x);
            const float use = mx == -kInf ? 0.0f : mx, old = s.L * __builtin_amdgcn_exp2f(s.M - use);
            float w[kAtOnce], sum = old;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                w[i] = k1 + i * every < u.n_parts ? ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - use) : 0.0f;
                sum += w[i];
            }
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            s.x *= old * inv;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (w[i] != 0.0f) s.x += (w[i] * inv) * v[i];
            s.L = sum;
            s.M = mx;
        }
        return s;
    };
    auto store = [&](int r, const f32x4& x) {
        *reinterpret_cast<f32x4*>(row_of(p.out, p, u.r, hk, u.tile * R + r, HD) + 4 * col) = x;
    };
    if (u.n_parts <= kAtOnce) {
        for (int r = blockIdx.y * kWide + k0; r < rows; r += gridDim.y * kWide) store(r, parts_of(r, 0, 1).x);
        return;
    }
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        const Mean s = parts_of(r, k0, kWide);
        sums[k0][col] = s.x;
        if (col == 0) mls[k0] = make_float2(s.M, s.L);
        __syncthreads();
        if (k0 == 0) {
            float M = -kInf, w[kWide], sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kWide; ++k) M = fmaxf(M, mls[k].x);
            const float use = M == -kInf ? 0.0f : M;
#pragma unroll
            for (int k = 0; k < kWide; ++k) {
                w[k] = mls[k].y * __builtin_amdgcn_exp2f(mls[k].x - use);
                sum += w[k];
            }
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kWide; ++k)
                if (w[k] != 0.0f) x += (w[k] * inv) * sums[k][col];
            store(r, x);
        }
        __syncthreads();
    }
}

// The split of a call, from what the host knows of it: few rows a sequence share
// their keys over the waves, many have waves of their own.  (Equal shares of steps for as many
// work-groups as the chip holds, whatever tiles they end in, were slower: 64 sequences of 100
// to 8000 113 us for 112, one of 60001 26.5 for 21.1, the four prompts below 283 for 255.)
struct PagedPlan {
    bool keys, split, alone;
    int32_t rows, target;
    int64_t tiles, units;  // at most
};
PagedPlan paged_plan(const PagedAttnArgs& a) {
    PagedPlan pl;
    const int64_t group = a.n_heads / a.c.n_kv, rows = group * a.c.n_rows;
    pl.keys = rows <= 32 * static_cast<int64_t>(a.c.n_seqs);
    pl.rows = pl.keys ? 16 : a.c.head_dim == 256 ? 64 : 128;
    pl.tiles = rows / pl.rows + a.c.n_seqs;
    // work-groups without a split, and the steps that one may then have
    const int64_t whole = pl.tiles * a.c.n_kv;
    int64_t steps = ((static_cast<int64_t>(a.c.max_pages) << a.c.page_bits) + 63) / 64;
    if (a.sliding_window > 0) steps = std::min(steps, (a.sliding_window + pl.rows / group + 63) / 64 + 1);
    if (pl.keys) {
        // A work-group of its own has 0.36 us for a step; parts and their merge take 10.6 for
        // one sequence.  So few steps are left whole, and more where others read meanwhile (8 KV
        // heads of 128; split, whole; 1 sequence of 400 10.9, 8.4 us, of 640 10.6, 9.9, of 800
        // 10.6, 11.3; 64 of 1000 38, 29, of 100 to 8000 112, 124; 16 of 100 to 8000 39, 61; 200
        // of 100 to 2000 115, 96).  All by the table's width, as the lengths are the device's:
        // with a table for 8192 tokens one sequence of 400 takes 10.8 and 64 of 1000 38.
        // Targets of 512 and 1024: 16 of 100 to 8000 38.9, 40.8, 8 of 4000 19.4, 24.5, 64 of 100
        // to 8000 120, 112.
        pl.split = steps > 10 + whole / 16 && whole < 2048;
        pl.target = whole < 512 ? 512 : 1024;
    } else {
        // Prompts, 32 heads on 8 KV heads, targets of 512, 768, 1024 and 2048: four of 306 to
        // 674 tokens behind 1152 to 3799 246, 241, 244, 263 us; one of 600 behind 30000 725,
        // 594, 665, 642; 40 of 100 behind 500 to 3000 314, 313, 342, 381.
        pl.split = steps > kLeastSteps && whole < 2048;
        pl.target = 768;
    }
    // (8 KV heads of 128, by four waves and alone: 1000 sequences of 20 to 100 tokens 126, 55 us,
    // 300 of 500 73, 74, of 2000 226, 265; in tables of more than 512 tokens always the former)
    pl.alone = pl.keys && whole >= 2048 && steps <= 8;
    // units = sum over tiles of ceil(steps / per) <= target / n_kv + tiles (and one for the
    // device's rounding of per, which takes less than a part in 10^6 of it)
    pl.units = pl.tiles + (pl.split ? pl.target / a.c.n_kv + 2 : 0);
    return pl;
}

template <int HD>
hipError_t paged_attention(PagedParams& p, const PagedPlan& pl, hipStream_t stream) {
    if (pl.units * p.c.n_kv > 0x7fffffff) return hipErrorInvalidValue;
    constexpr int kOwn = HD == 256 ? 1 : 2;
    const int64_t groups = pl.units * p.c.n_kv;
    const hipError_t e = by_groups(pl.alone ? (groups + kAttnWaves - 1) / kAttnWaves : groups, [&](uint32_t first, dim3 grid) {
        p.first = first;
        if (pl.alone) hipLaunchKernelGGL((paged_keys_kernel<HD, true>), grid, dim3(kAttnThreads), 0, stream, p);
        else if (pl.keys) hipLaunchKernelGGL((paged_keys_kernel<HD, false>), grid, dim3(kAttnThreads), 0, stream, p);
        else hipLaunchKernelGGL((paged_rows_kernel<HD, kOwn>), grid, dim3(kAttnThreads), 0, stream, p);
    });
    if (e != hipSuccess || !pl.split) return e;
    // a tile's rows in as many work-groups as make 2048 of them
    const int64_t rows = std::min<int64_t>(pl.rows, static_cast<int64_t>(p.c.n_rows) * p.group), tiles = pl.tiles * p.c.n_kv;
    const dim3 merge(static_cast<uint32_t>(tiles),
                     static_cast<uint32_t>(std::max<int64_t>(1, std::min<int64_t>(rows, 2048 / tiles))));
    if (pl.keys) hipLaunchKernelGGL((paged_merge_kernel<HD, 16>), merge, dim3(kAttnThreads), 0, stream, p);
    else hipLaunchKernelGGL((paged_merge_kernel<HD, 64 * kOwn>), merge, dim3(kAttnThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope_rows(const float* rows, int32_t n_rows, int32_t row_stride, int32_t n_heads, int32_t head_dim,
                            const int32_t* positions, const RotationArgs& rot, int32_t out_stride, float* out,
                            hipStream_t stream) {
    if (n_rows < 1 || n_heads < 1 || head_dim < 2 || head_dim % 2 || head_dim > kMaxRopeDim || rot.n_rot < 0 ||
        rot.n_rot % 2 || rot.n_rot > head_dim)
        return hipErrorInvalidValue;
    RopeRowsParams p{rows, out, positions, rot, n_heads, head_dim, row_stride, out_stride, n_heads};
    const auto aligned = [](const float* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
    const bool vec = head_dim % 8 == 0 && rot.n_rot % 8 == 0 && row_stride % 4 == 0 && out_stride % 4 == 0 &&
                     aligned(rows) && aligned(out);
    // a row's heads in as many work-groups as make 1024 of them, at least as many
    // heads each as it takes at once
    const int32_t at_once = std::max(1, kRopeThreads / (vec ? head_dim / 8 : head_dim / 2));
    const int32_t most = (n_heads + at_once - 1) / at_once;
    const int32_t groups = std::min(most, std::max(1, (1024 + n_rows - 1) / n_rows));
    p.heads_per_group = (n_heads + groups - 1) / groups;
    const uint32_t per_row = (n_heads + p.heads_per_group - 1) / p.heads_per_group;
    if (per_row > 65535) return hipErrorInvalidValue;
    return by_groups(n_rows, [&](uint32_t first, dim3 grid) {
        grid.y = per_row;
        p.rows = rows + static_cast<size_t>(first) * row_stride;
        p.out = out + static_cast<size_t>(first) * out_stride;
        p.positions = positions + first;
        if (vec) hipLaunchKernelGGL(rope_rows_kernel<true>, grid, dim3(kRopeThreads), 0, stream, p);
        else hipLaunchKernelGGL(rope_rows_kernel<false>, grid, dim3(kRopeThreads), 0, stream, p);
    });
}

hipError_t launch_kv_append_paged(const AppendArgs& a, hipStream_t stream) {
    AppendParams p{a, 0, false, (a.n_heads + 15) / 16, 0};
    const int64_t by_blocks = static_cast<int64_t>(a.c.n_rows / kKvBlock) + 2 * a.c.n_seqs;
    p.by_rows = a.c.n_rows < by_blocks;
    p.kv_groups = std::min<int64_t>(a.c.n_rows, by_blocks) * a.c.n_kv * 2;
    const int64_t groups = p.kv_groups + (a.q ? static_cast<int64_t>(a.c.n_rows) * p.head_groups : 0);
    if (groups > 0x7fffffff) return hipErrorInvalidValue;
    if (a.c.head_dim != 64 && a.c.head_dim != 128 && a.c.head_dim != 256) return hipErrorInvalidValue;
    return by_groups(groups, [&](uint32_t first, dim3 grid) {
        p.first = first;
        if (a.c.head_dim == 64) hipLaunchKernelGGL(append_kernel<64>, grid, dim3(128), 0, stream, p);
        else if (a.c.head_dim == 128) hipLaunchKernelGGL(append_kernel<128>, grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL(append_kernel<256>, grid, dim3(512), 0, stream, p);
    });
}

size_t attention_paged_workspace_bytes(const PagedAttnArgs& a) {
    const PagedPlan pl = paged_plan(a);
    if (!pl.split) return 0;
    return static_cast<size_t>(pl.units) * a.c.n_kv * pl.rows * (sizeof(float2) + sizeof(float) * a.c.head_dim);
}

hipError_t launch_attention_paged(const PagedAttnArgs& a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (workspace_bytes < attention_paged_workspace_bytes(a)) return hipErrorInvalidValue;
    const PagedPlan pl = paged_plan(a);
    PagedParams p{};
    p.c = a.c;
    p.q = a.q;
    p.out = a.out;
    p.n_heads = a.n_heads;
    p.group = a.n_heads / a.c.n_kv;
    p.sw = a.sliding_window;
    p.target = pl.target;
    p.split = pl.split;
    p.units = static_cast<int32_t>(std::min<int64_t>(pl.units, INT32_MAX));
    p.scale = a.scale == 0.0f ? 1.0f : std::fabs(a.scale) * 1.44269504088896341f;
    p.sign = a.scale < 0.0f ? -1.0f : a.scale == 0.0f ? 0.0f : 1.0f;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(pl.units) * a.c.n_kv * pl.rows * a.c.head_dim);
    if (a.c.head_dim == 64) return paged_attention<64>(p, pl, stream);
    if (a.c.head_dim == 128) return paged_attention<128>(p, pl, stream);
    if (a.c.head_dim == 256) return paged_attention<256>(p, pl, stream);
    return hipErrorInvalidValue;
}

}  // namespace gncx
