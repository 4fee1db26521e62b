// Layer operators on device memory: dropout whose mask is computed from a counter and never stored, layer
// normalisation with its backward pass, and both in one pass, y = norm(dropout(x)).
//
//   dropout   d(x) = x * 65536 / (65536 - t) where the unit's 16-bit draw is >= t, else 0; its gradient is d(dy)
//   norm      h = x or d(x);  m = mean h;  r = 1 / sqrt(mean (h - m)^2 + eps);  u = (h - m) r;  y = u w + b
//   backward  g = dy w;  dh = r (g - mean g - u mean(g u));  dx = dh or d(dh);  dw = sum dy u;  db = sum dy
//
// Sums, means and the values between load and store are floats for float, bfloat16 and half, doubles for double; a
// value is rounded to its type once, as it is stored.  All of it is bound by memory: a thread takes chunks of eight
// consecutive columns (one counter of the generator, 16 bytes of a 16-bit type), and the work between is hidden
// behind the loads -- ten rounds of the generator for every chunk of a dropout of 819,200 x 128 bfloat16 leave it at
// the rate of a copy (69.9 us, 6.0 TB/s, with them and 70.4 us without).
#include "epi_layers.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "epi_host.hpp"

#define EPI_API extern "C" __attribute__((visibility("default")))

#pragma clang fp contract(fast)   // products go into sums unrounded

namespace epi {
namespace {

constexpr int kChunk = 8;   // columns a thread takes at once: the eight draws of one counter

template <class T> struct Wide { using type = float; };
template <> struct Wide<double> { using type = double; };
template <class T> using wide_t = typename Wide<T>::type;

// ---- chunks of eight columns ------------------------------------------------------------------
// A chunk on its way is whole 32-bit words: nothing has to wait for it before its first use.  Rows of odd widths
// start at any multiple of the element's size, so accesses are declared with the element's alignment: the hardware
// takes 16 bytes at any address, and rows that do start at 16 bytes lose nothing.  The last chunk of a row that is no
// multiple of eight is put together from a part of four, of two and of one element.
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Part { uint32_t w[N]; };
template <class T> struct Raw {
    static constexpr int kWords = kChunk * sizeof(T) / 4;
    uint32_t w[kWords];
};

// the words of N elements (N even, or elements of 4 bytes and more)
template <class T, int N>
__device__ inline void fetch_part(const T* p, uint32_t* w) {
    constexpr int W = N * sizeof(T) / 4;
    const Part<T, W> v = *reinterpret_cast<const Part<T, W>*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = v.w[i];
}
template <class T, int N>
__device__ inline void put_part(T* p, const uint32_t* w) {
    constexpr int W = N * sizeof(T) / 4;
    Part<T, W> v;
#pragma unroll
    for (int i = 0; i < W; ++i) v.w[i] = w[i];
    *reinterpret_cast<Part<T, W>*>(p) = v;
}

template <class T>
__device__ inline void fetch_chunk(const T* p, int count, Raw<T>& c) {
    constexpr int W = Raw<T>::kWords;
    if (count >= kChunk) {
        fetch_part<T, kChunk>(p, c.w);
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) c.w[i] = 0;
    if (count <= 0) return;
    // from the back: what is there moves up by the part put before it
    if (count & 1) {
        const T* q = p + (count & 6);
        if constexpr (sizeof(T) == 2) c.w[0] = *reinterpret_cast<const uint16_t*>(q);
        else fetch_part<T, 1>(q, c.w);
    }
    if (count & 2) {
        uint32_t v[W / 4];
        fetch_part<T, 2>(p + (count & 4), v);
#pragma unroll
        for (int i = W / 2 - 1; i >= W / 4; --i) c.w[i] = c.w[i - W / 4];
#pragma unroll
        for (int i = 0; i < W / 4; ++i) c.w[i] = v[i];
    }
    if (count & 4) {
        uint32_t v[W / 2];
        fetch_part<T, 4>(p, v);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) { c.w[i + W / 2] = c.w[i]; c.w[i] = v[i]; }
    }
}
template <class T>
__device__ inline void put_chunk(T* p, int count, Raw<T> c) {
    constexpr int W = Raw<T>::kWords;
    if (count >= kChunk) {
        put_part<T, kChunk>(p, c.w);
        return;
    }
    if (count <= 0) return;
    if (count & 4) {
        put_part<T, 4>(p, c.w);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) c.w[i] = c.w[i + W / 2];
        p += 4;
    }
    if (count & 2) {
        put_part<T, 2>(p, c.w);
#pragma unroll
        for (int i = 0; i < W / 4; ++i) c.w[i] = c.w[i + W / 4];
        p += 2;
    }
    if (count & 1) {
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)c.w[0];
        else put_part<T, 1>(p, c.w);
    }
}

template <class T> struct Pair { T lo, hi; };
template <class T>
__device__ inline void widen_chunk(const Raw<T>& c, wide_t<T> (&out)[kChunk]) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
        if constexpr (std::is_same_v<T, __bf16>) {
            out[k] = __builtin_bit_cast(float, (k & 1) ? c.w[k / 2] & 0xffff0000u : c.w[k / 2] << 16);
        } else if constexpr (sizeof(T) == 2) {
            const auto h = __builtin_bit_cast(Pair<T>, c.w[k / 2]);
            out[k] = (float)((k & 1) ? h.hi : h.lo);
        } else if constexpr (sizeof(T) == 4) {
            out[k] = __builtin_bit_cast(T, c.w[k]);
        } else {
            out[k] = __builtin_bit_cast(T, (uint64_t)c.w[2 * k + 1] << 32 | c.w[2 * k]);
        }
    }
}
template <class T>
__device__ inline void narrow_chunk(const wide_t<T> (&in)[kChunk], Raw<T>& c) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
        if constexpr (sizeof(T) == 2) {
            if (k & 1) c.w[k / 2] = __builtin_bit_cast(uint32_t, Pair<T>{(T)in[k - 1], (T)in[k]});
        } else if constexpr (sizeof(T) == 4) {
            c.w[k] = __builtin_bit_cast(uint32_t, in[k]);
        } else {
            const uint64_t b = __builtin_bit_cast(uint64_t, in[k]);
            c.w[2 * k] = (uint32_t)b; c.w[2 * k + 1] = (uint32_t)(b >> 32);
        }
    }
}
template <class T>
__device__ inline void load_chunk(const T* p, int count, wide_t<T> (&out)[kChunk]) {
    Raw<T> c;
    fetch_chunk(p, count, c);
    widen_chunk(c, out);
}
template <class T>
__device__ inline void store_chunk(T* p, int count, const wide_t<T> (&in)[kChunk]) {
    Raw<T> c;
    narrow_chunk<T>(in, c);
    put_chunk(p, count, c);
}
// Keeps the compiler from holding on to what it formed of the words before.
template <class T>
__device__ inline void forget(Raw<T>& c) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kWords; ++i) asm volatile("" : "+v"(c.w[i]));
}
// How many of the eight columns from `col` on exist.
template <class I>
__device__ inline int chunk_count(I cols, I col) {
    const I room = cols - col;
    return room < 0 ? 0 : room < kChunk ? (int)room : kChunk;
}
// Values behind a row's end become zero.
template <class A>
__device__ inline void clear_tail(int count, A (&v)[kChunk]) {
    if (count < kChunk) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k) v[k] = k < count ? v[k] : (A)0;
    }
}

// ---- the generator ------------------------------------------------------------------------------
// The four words of Philox4x32-10 for chunk `chunk` of row `row`.
__device__ inline void draw_words(const DropArgs& d, const uint32_t (&off)[2], uint32_t chunk, uint32_t row, uint32_t (&w)[4]) {
    uint32_t c0 = chunk, c1 = row, c2 = off[0], c3 = off[1], k0 = d.key[0], k1 = d.key[1];
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

__device__ inline void drop_offset(const DropArgs& d, uint32_t (&off)[2]) {
    uint64_t o = ((uint64_t)d.offset[1] << 32) | d.offset[0];
    if (d.offset_dev) o += (uint64_t)*d.offset_dev;
    off[0] = (uint32_t)o; off[1] = (uint32_t)(o >> 32);
}

// Which of the eight units are kept: the draw of 16 bits in the upper half of a word w is at least the threshold t
// exactly where w > t * 2^16 - 1, whatever the lower half holds; the draw in the lower half is shifted there.  For
// t = 2^16 nothing is above the border; t = 0 has none, and is not asked for.
struct Keep {
    uint32_t w[4], border;
    __device__ bool operator()(int k) const { return ((k & 1) ? w[k >> 1] : w[k >> 1] << 16) > border; }
};
__device__ inline Keep keep_of(const DropArgs& d, const uint32_t (&off)[2], uint32_t chunk, uint32_t row) {
    Keep keep;
    draw_words(d, off, chunk, row, keep.w);
    keep.border = (uint32_t)(((uint64_t)d.threshold << 16) - 1);
    return keep;
}
// A dropped value becomes zero whatever it was: infinities and NaN do not pass through the product.
template <class A>
__device__ inline void drop_chunk(const Keep& keep, A scale, A (&v)[kChunk]) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) v[k] = keep(k) ? v[k] * scale : (A)0;
}

// The same as one bit a unit.
__device__ inline uint32_t pack(const Keep& keep) {
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < kChunk; ++k) bits |= keep(k) ? 1u << k : 0u;
    return bits;
}
template <class A>
__device__ inline void drop_bits(uint32_t bits, A scale, A (&v)[kChunk]) {
#pragma unroll
    for (int k = 0; k < kChunk; ++k) v[k] = (bits >> k & 1) ? v[k] * scale : (A)0;
}

// ---- sums over the threads of a row ---------------------------------------------------------------
// One step of a sum over 2 * D lanes whose halves hold a value each: every lane adds the other half's value.  Steps
// within 16 lanes are data-parallel moves of the vector unit, the two beyond swap rows of 16 or 32 lanes; nothing goes
// through LDS.
template <int D>
__device__ inline uint32_t other_half(uint32_t v) {
    if constexpr (D == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);        // lanes 1 0 3 2
    else if constexpr (D == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);   // lanes 2 3 0 1
    else if constexpr (D == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);  // 8 lanes mirrored
    else return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true);                        // 16 lanes mirrored
}
template <int D>
__device__ inline void halves(uint32_t v, uint32_t& lo, uint32_t& hi) {
    if constexpr (D == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        lo = p[0]; hi = p[1];
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        lo = p[0]; hi = p[1];
    }
}
template <int D>
__device__ inline float add_half(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    if constexpr (D < 16) return v + __builtin_bit_cast(float, other_half<D>(b));
    uint32_t lo, hi;
    halves<D < 16 ? 16 : D>(b, lo, hi);
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
template <int D>
__device__ inline double add_half(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    if constexpr (D < 16) {
        const uint64_t o = (uint64_t)other_half<D>((uint32_t)(b >> 32)) << 32 | other_half<D>((uint32_t)b);
        return v + __builtin_bit_cast(double, o);
    }
    uint32_t l0, l1, h0, h1;
    halves<D < 16 ? 16 : D>((uint32_t)b, l0, h0);
    halves<D < 16 ? 16 : D>((uint32_t)(b >> 32), l1, h1);
    return __builtin_bit_cast(double, (uint64_t)l1 << 32 | l0) + __builtin_bit_cast(double, (uint64_t)h1 << 32 | h0);
}
// Sum over N consecutive lanes, N a power of two; every lane gets it.
template <int N, class A>
__device__ inline A lane_sum(A v) {
    if constexpr (N > 1) v = add_half<1>(v);
    if constexpr (N > 2) v = add_half<2>(v);
    if constexpr (N > 4) v = add_half<4>(v);
    if constexpr (N > 8) v = add_half<8>(v);
    if constexpr (N > 16) v = add_half<16>(v);
    if constexpr (N > 32) v = add_half<32>(v);
    return v;
}

// N sums at once over TPR consecutive lanes (TPR <= 64) or over the whole workgroup of TPR threads, in a fixed order;
// every thread gets them.  The workgroup form alternates between two LDS buffers, so one barrier a call is enough: a
// buffer is written again only after the barrier of the call between.
template <int TPR, int N> constexpr int kRowLds = TPR > 64 ? 2 * (TPR / 64) * N : 1;
template <int TPR, int N, class A>
__device__ inline void row_sums(A (&v)[N], A* lds, int& flip) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane_sum<(TPR < 64 ? TPR : 64)>(v[n]);
    if constexpr (TPR > 64) {
        constexpr int kWaves = TPR / 64;
        A* buf = lds + (flip & 1) * kWaves * 2;
        ++flip;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) buf[n * kWaves + (threadIdx.x >> 6)] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = lane_sum<kWaves>(buf[n * kWaves + threadIdx.x % kWaves]);
    }
}

__device__ inline float inverse_root(float v) { return 1.0f / sqrtf(v); }
__device__ inline double inverse_root(double v) { return 1.0 / sqrt(v); }

// Which weights, which dropout counter and which row number a row has.
struct RowPlace {
    int64_t weight;      // element offset of the row's weights
    uint32_t row;        // the row's number in the dropout counter
    uint32_t off[2];
    bool used;
};
template <bool SETS>
__device__ inline RowPlace place_row(const NormArgs& a, int64_t row) {
    RowPlace p;
    p.weight = 0; p.row = (uint32_t)row; p.used = row < a.rows;
    p.off[0] = p.off[1] = 0;
    if constexpr (SETS) {
        if (p.used) {
            const int set = (int)(row / a.sets.set_rows);
            p.row = (uint32_t)(row - (int64_t)set * a.sets.set_rows);
            p.used = (int)p.row < a.sets.set_used[set];
            p.weight = (int64_t)a.sets.set_index[set] * a.sets.weight_stride;
            if (a.sets.set_ctr) { p.off[0] = a.sets.set_ctr[2 * set]; p.off[1] = a.sets.set_ctr[2 * set + 1]; }
        }
    }
    return p;
}

// ---- dropout ----------------------------------------------------------------------------------------
struct DropShape {
    int64_t row0;                // first row of the launch
    uint32_t chunks;             // (row, chunk) pairs of the launch, below 2^31
    uint32_t per_row;            // chunks of a row
    uint32_t magic, shift;       // n / per_row = (n * magic) >> shift for every n below 2^31
    int64_t cols, x_stride, y_stride;
};

template <class T, bool DROP>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, T* y, DropShape s, DropArgs d) {
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= s.chunks) return;
    const uint32_t r = (uint32_t)(((uint64_t)g * s.magic) >> s.shift), c = g - r * s.per_row;
    const int64_t row = s.row0 + r, col = (int64_t)c * kChunk;
    const int count = chunk_count(s.cols, col);
    Raw<T> raw;
    fetch_chunk(x + row * s.x_stride + col, count, raw);
    wide_t<T> v[kChunk];
    widen_chunk(raw, v);
    if constexpr (DROP) {
        uint32_t off[2];
        drop_offset(d, off);
        drop_chunk(keep_of(d, off, c, (uint32_t)row), (wide_t<T>)d.scale, v);
    }
    store_chunk(y + row * s.y_stride + col, count, v);
}

// ---- layer norm, forward: rows that fit the registers of their threads ---------------------------------
// TPR threads hold a row, NV chunks of eight columns each: it is read once, and while it is worked on the next row
// is on its way.  TPR <= 64: 256 / TPR rows side by side in a workgroup, no barrier; else a row per workgroup.  Bound by
// memory: 819,200 x 128 bfloat16 take 77 us (5.4 TB/s, a large copy reaches 5.0 to 5.4), 79 with dropout; 16,384 x
// 4,096 bfloat16 47 us (5.7 TB/s, part of it from the caches); 24,576 x 128 float 6.6 us, of which 2.5 are the launch.
constexpr int norm_threads(int tpr) { return tpr > 64 ? tpr : 256; }

// The chunk of a row of at least eight columns that a thread works on.  Where the row's end cuts it, it is moved back
// to the last eight columns, and its first `skip` columns are another thread's too: both form the same values for
// them from the same inputs and both store them, but only the other counts them in sums.  So no access and no value
// needs a case of its own.  skip = 8: no column of the row is left for this thread, which loads but stores nothing.
struct Spot {
    int col, skip;
};
__device__ inline Spot spot_of(int cols, int chunk) {
    const int col = chunk * kChunk, at = min(col, cols - kChunk);
    return {at, min(col - at, kChunk)};
}
template <class A>
__device__ inline void clear_head(int skip, A (&v)[kChunk]) {
    if (skip > 0) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k) v[k] = k < skip ? (A)0 : v[k];
    }
}
// keep_of for a spot: one that was moved back takes its draws from two counters.
__device__ inline Keep keep_at(const DropArgs& d, const uint32_t (&off)[2], const Spot& p, uint32_t row) {
    const uint32_t chunk = (uint32_t)p.col / kChunk, shift = (uint32_t)p.col % kChunk;
    Keep keep = keep_of(d, off, chunk, row);
    if (shift) {
        uint32_t w[8];
        const Keep next = keep_of(d, off, chunk + 1, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = keep.w[i]; w[i + 4] = next.w[i]; }
        if (shift & 4) {
#pragma unroll
            for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
        }
        if (shift & 2) {
#pragma unroll
            for (int i = 0; i < 7; ++i) w[i] = w[i + 1];
        }
        if (shift & 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = w[i] >> 16 | w[i + 1] << 16;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) keep.w[i] = w[i];
    }
    return keep;
}
template <class T>
__device__ inline void fetch_full(const T* p, Raw<T>& c) { fetch_part<T, kChunk>(p, c.w); }
template <class T>
__device__ inline void load_full(const T* p, wide_t<T> (&out)[kChunk]) {
    Raw<T> c;
    fetch_full(p, c);
    widen_chunk(c, out);
}

template <class T, int TPR, int NV, bool DROP>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_forward_kernel(NormArgs a) {
    using A = wide_t<T>;
    constexpr int kRows = norm_threads(TPR) / TPR;
    constexpr bool kHold = NV == 1 && sizeof(T) < 8;   // registers for the weights
    // registers for the next row, where they are left: 1,024 threads have 128 each (1,021 x 20,000 float with dropout:
    // 43.7 us with the next row's and spills, 38.4 without; without dropout 36.7 with and 36.6 without).  Rows of more than
    // 24,576 doubles spill all the same, 152 bytes a lane, and with dropout 404, from 16,385 on 172: 1,500 x 30,000 take
    // 256 us (2.8 TB/s) and 316, 2,000 x 20,000 179 (3.6) and 226
    constexpr bool kAhead = TPR < 1024 || (DROP ? NV < 4 && NV * sizeof(T) <= 8 : NV * sizeof(T) <= 16);
    __shared__ A lds[kRowLds<TPR, 2>];
    int flip = 0;
    const int t = threadIdx.x % TPR, cols = (int)a.cols;
    int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * kRows;
    const A inv = (A)a.inv_cols, scale = (A)a.drop.scale;
    const T* weight = static_cast<const T*>(a.weight);
    const T* bias = static_cast<const T*>(a.bias);
    uint32_t off[2] = {0, 0};
    if constexpr (DROP) drop_offset(a.drop, off);
    Raw<T> raw[NV];
    auto fetch = [&](int64_t r) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) fetch_full(x + spot_of(cols, t + v * TPR).col, raw[v]);
    };
    auto gains = [&](int col, A (&g)[kChunk], A (&b)[kChunk]) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k) { g[k] = 1; b[k] = 0; }
        if (weight) load_full(weight + col, g);
        if (bias) load_full(bias + col, b);
    };
    if (row < a.rows) fetch(row);
    A hg[kChunk], hb[kChunk];
    if constexpr (kHold) gains(spot_of(cols, t).col, hg, hb);
    while (row < a.rows) {
        A h[NV][kChunk];
#pragma unroll
        for (int v = 0; v < NV; ++v) widen_chunk(raw[v], h[v]);
        const int64_t next = row + step;
        if (kAhead && next < a.rows) fetch(next);
        A s[1] = {0};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Spot p = spot_of(cols, t + v * TPR);
            if constexpr (DROP) drop_chunk(keep_at(a.drop, off, p, (uint32_t)row), scale, h[v]);
            A c[kChunk];
#pragma unroll
            for (int k = 0; k < kChunk; ++k) c[k] = h[v][k];
            clear_head(p.skip, c);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) s[0] += c[k];
        }
        row_sums<TPR>(s, lds, flip);
        const A m = s[0] * inv;
        A q[2] = {0, 0};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            A c[kChunk];
#pragma unroll
            for (int k = 0; k < kChunk; ++k) c[k] = h[v][k] -= m;
            clear_head(spot_of(cols, t + v * TPR).skip, c);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) { q[0] += c[k]; q[1] += c[k] * c[k]; }
        }
        row_sums<TPR>(q, lds, flip);
        const A d = q[0] * inv;
        A var = q[1] * inv - d * d;
        var = var < 0 ? (A)0 : var;   // keeps NaN
        const A r = inverse_root(var + (A)a.eps);
        if (t == 0 && a.mean) { static_cast<A*>(a.mean)[row] = m + d; static_cast<A*>(a.rstd)[row] = r; }
        T* y = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Spot p = spot_of(cols, t + v * TPR);
            if (p.skip == kChunk) continue;
            A g[kChunk], b[kChunk];
            if constexpr (!kHold) gains(p.col, g, b);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) h[v][k] = (h[v][k] - d) * r * (kHold ? hg[k] : g[k]) + (kHold ? hb[k] : b[k]);
            Raw<T> o;
            narrow_chunk<T>(h[v], o);
            put_part<T, kChunk>(y + p.col, o.w);
        }
        row = next;
        if (!kAhead && row < a.rows) fetch(row);
    }
}

// ---- layer norm, forward: any width ------------------------------------------------------------------
// A row is walked three times by TPR threads (mean; spread about it; output); the second and third walk find it in
// the caches.  The spread is taken about the rounded mean m together with the mean d of what is left, so a mean far
// from zero costs no digits: variance = mean (h-m)^2 - d^2 and u = ((h-m) - d) r.  For rows below eight columns, above
// 32,768 (1,000 x 100,000 bfloat16: 116 us with 1,024 threads, 3.4 TB/s over x and y, 147 with 256) and of several
// networks at once.
template <class T, int TPR, bool DROP, bool SETS>
__device__ inline void norm_forward_row(const NormArgs& a, int64_t row, wide_t<T>* lds, int& flip) {
    using A = wide_t<T>;
    const int t = threadIdx.x % TPR;
    RowPlace pl = place_row<SETS>(a, row);
    if (!pl.used) return;   // the same for all threads of the row, and of the workgroup where it has one row
    if (DROP && !(SETS && a.sets.set_ctr)) drop_offset(a.drop, pl.off);
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    T* y = static_cast<T*>(a.y) + row * a.y_stride;
    const A inv = (A)a.inv_cols, scale = (A)a.drop.scale;
    auto load = [&](int64_t col, int& count, A (&h)[kChunk]) {
        count = chunk_count(a.cols, col);
        load_chunk(x + col, count, h);
        if constexpr (DROP) drop_chunk(keep_of(a.drop, pl.off, (uint32_t)(col / kChunk), pl.row), scale, h);
    };
    A s[1] = {0};
    for (int64_t col = (int64_t)t * kChunk; col < a.cols; col += TPR * kChunk) {
        A h[kChunk]; int count;
        load(col, count, h);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) s[0] += h[k];
    }
    row_sums<TPR>(s, lds, flip);
    const A m = s[0] * inv;
    A q[2] = {0, 0};
    for (int64_t col = (int64_t)t * kChunk; col < a.cols; col += TPR * kChunk) {
        A h[kChunk]; int count;
        load(col, count, h);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) h[k] -= m;
        clear_tail(count, h);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) { q[0] += h[k]; q[1] += h[k] * h[k]; }
    }
    row_sums<TPR>(q, lds, flip);
    const A d = q[0] * inv;
    A var = q[1] * inv - d * d;
    var = var < 0 ? (A)0 : var;   // keeps NaN
    const A r = inverse_root(var + (A)a.eps);
    if (t == 0 && a.mean) { static_cast<A*>(a.mean)[row] = m + d; static_cast<A*>(a.rstd)[row] = r; }
    const T* weight = a.weight ? static_cast<const T*>(a.weight) + pl.weight : nullptr;
    const T* bias = a.bias ? static_cast<const T*>(a.bias) + pl.weight : nullptr;
    for (int64_t col = (int64_t)t * kChunk; col < a.cols; col += TPR * kChunk) {
        A h[kChunk], g[kChunk], b[kChunk]; int count;
        load(col, count, h);
        if (weight) load_chunk(weight + col, count, g);
        if (bias) load_chunk(bias + col, count, b);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) {
            const A u = ((h[k] - m) - d) * r;
            h[k] = (weight ? u * g[k] : u) + (bias ? b[k] : (A)0);
        }
        store_chunk(y + col, count, h);
    }
}

// A launch holds at most kMaxBlocks workgroups (a grid has fewer than 2^32 threads): they walk on over the rows or columns.
constexpr int64_t kMaxBlocks = (int64_t)1 << 20;

template <class T, int TPR, bool DROP, bool SETS>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_forward_walk_kernel(NormArgs a) {
    __shared__ wide_t<T> lds[kRowLds<TPR, 2>];
    int flip = 0;
    constexpr int kRows = norm_threads(TPR) / TPR;
    for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * kRows)
        norm_forward_row<T, TPR, DROP, SETS>(a, row, lds, flip);
}

// ---- layer norm, backward: any width -------------------------------------------------------------------
// One launch of two kinds of workgroups that do not wait for each other.  The first row_blocks take rows and write
// dx, TPR threads a row, in two walks (the two means; the result).  The others take columns, 32 of them and
// seg_rows rows each, and form sums of dy u and dy: 4 threads side by side, 64 rows at a time, then the 64 sums of
// every column in a fixed order.  With one segment they are the gradients, else partial sums for
// norm_reduce_kernel.  For what the kernel below does not take: few rows (split_rows), where one launch is what counts
// (512 x 128 double: 8 us, bound by a few loads one after the other), rows below eight columns, and rows beyond the
// registers, whose x and dy are read twice from memory (1,000 x 100,000 bfloat16: 292 us, 2.1 TB/s over x, dy and dx).
constexpr int kTileCols = 32, kTileSlots = 64;

struct SplitShape {
    int64_t row_blocks, col_tiles, segs, seg_rows;
};

template <class T, bool DROP, bool SETS>
__device__ inline void column_sums(const NormArgs& a, const SplitShape& sh, int64_t block, wide_t<T>* lds) {
    using A = wide_t<T>;
    const int64_t tile = block % sh.col_tiles, seg = block / sh.col_tiles;   // SETS: a segment is a set
    const int64_t first = seg * sh.seg_rows;
    int64_t last = first + sh.seg_rows < a.rows ? first + sh.seg_rows : a.rows;
    if constexpr (SETS) last = first + a.sets.set_used[seg] < last ? first + a.sets.set_used[seg] : last;
    const int lane = threadIdx.x % 4, slot = threadIdx.x / 4;
    const int64_t col = tile * kTileCols + lane * kChunk;
    const int count = chunk_count(a.cols, col);
    uint32_t off[2] = {0, 0};
    if constexpr (DROP) drop_offset(a.drop, off);
    if (SETS && a.sets.set_ctr) { off[0] = a.sets.set_ctr[2 * seg]; off[1] = a.sets.set_ctr[2 * seg + 1]; }
    const A scale = (A)a.drop.scale;
    A gw[kChunk], gb[kChunk];
#pragma unroll
    for (int k = 0; k < kChunk; ++k) gw[k] = gb[k] = 0;
    if (count > 0) {
        for (int64_t row = first + slot; row < last; row += kTileSlots) {
            A h[kChunk], dy[kChunk];
            load_chunk(static_cast<const T*>(a.x) + row * a.x_stride + col, count, h);
            load_chunk(static_cast<const T*>(a.dy) + row * a.dy_stride + col, count, dy);
            const A m = static_cast<const A*>(a.mean)[row], r = static_cast<const A*>(a.rstd)[row];
            if constexpr (DROP)
                drop_chunk(keep_of(a.drop, off, (uint32_t)(col / kChunk), (uint32_t)(SETS ? row - first : row)), scale, h);
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                gw[k] += dy[k] * ((h[k] - m) * r);
                gb[k] += dy[k];
            }
        }
    }
    // [2][slot][column]: 64 threads sum the 32 columns of both
#pragma unroll
    for (int k = 0; k < kChunk; ++k) {
        lds[slot * kTileCols + lane * kChunk + k] = gw[k];
        lds[(kTileSlots + slot) * kTileCols + lane * kChunk + k] = gb[k];
    }
    __syncthreads();
    const int which = threadIdx.x / kTileCols, c = threadIdx.x % kTileCols;
    if (which < 2 && tile * kTileCols + c < a.cols) {
        A part[4] = {0, 0, 0, 0};
        for (int k = 0; k < kTileSlots; k += 4) {
#pragma unroll
            for (int u = 0; u < 4; ++u) part[u] += lds[(which * kTileSlots + k + u) * kTileCols + c];
        }
        const A total = (part[0] + part[1]) + (part[2] + part[3]);
        const int64_t at = tile * kTileCols + c;
        if (SETS || sh.segs == 1) {
            T* out = static_cast<T*>(which ? a.dbias : a.dweight);
            if (out) out[seg * a.cols + at] = (T)total;
        } else {
            static_cast<A*>(a.workspace)[(seg * 2 + which) * a.cols + at] = total;
        }
    }
}

template <class T, int TPR, bool DROP, bool SETS>
__device__ inline void norm_backward_row(const NormArgs& a, int64_t row, wide_t<T>* lds, int& flip) {
    using A = wide_t<T>;
    const int t = threadIdx.x % TPR;
    RowPlace pl = place_row<SETS>(a, row);
    if (!pl.used) return;
    if (DROP && !(SETS && a.sets.set_ctr)) drop_offset(a.drop, pl.off);
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
    T* dx = static_cast<T*>(a.dx) + row * a.y_stride;
    const T* weight = a.weight ? static_cast<const T*>(a.weight) + pl.weight : nullptr;
    const A inv = (A)a.inv_cols, scale = (A)a.drop.scale;
    const A m = static_cast<const A*>(a.mean)[row], r = static_cast<const A*>(a.rstd)[row];
    auto load = [&](int64_t col, int& count, A (&u)[kChunk], A (&g)[kChunk], Keep& keep) {
        count = chunk_count(a.cols, col);
        load_chunk(x + col, count, u);
        load_chunk(dy + col, count, g);
        if constexpr (DROP) {
            keep = keep_of(a.drop, pl.off, (uint32_t)(col / kChunk), pl.row);
            drop_chunk(keep, scale, u);
        }
        A gain[kChunk];
        if (weight) load_chunk(weight + col, count, gain);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) {
            u[k] = (u[k] - m) * r;
            if (weight) g[k] *= gain[k];
        }
    };
    A s[2] = {0, 0};
    for (int64_t col = (int64_t)t * kChunk; col < a.cols; col += TPR * kChunk) {
        A u[kChunk], g[kChunk]; Keep keep{}; int count;
        load(col, count, u, g, keep);
        clear_tail(count, u);   // g is zero there, but 0 * u need not be
#pragma unroll
        for (int k = 0; k < kChunk; ++k) { s[0] += g[k]; s[1] += g[k] * u[k]; }
    }
    row_sums<TPR>(s, lds, flip);
    const A c1 = s[0] * inv, c2 = s[1] * inv;
    for (int64_t col = (int64_t)t * kChunk; col < a.cols; col += TPR * kChunk) {
        A u[kChunk], g[kChunk]; Keep keep{}; int count;
        load(col, count, u, g, keep);
#pragma unroll
        for (int k = 0; k < kChunk; ++k) g[k] = ((g[k] - c1) - u[k] * c2) * r;
        if constexpr (DROP) drop_chunk(keep, scale, g);
        store_chunk(dx + col, count, g);
    }
}

template <class T, int TPR, bool DROP, bool SETS>
__global__ __launch_bounds__(256) void norm_backward_split_kernel(NormArgs a, SplitShape sh) {
    using A = wide_t<T>;
    __shared__ A lds[2 * kTileSlots * kTileCols];
    if ((int64_t)blockIdx.x < sh.row_blocks) {
        int flip = 0;
        constexpr int kRows = 256 / TPR;
        for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR; row < a.rows; row += sh.row_blocks * kRows)
            norm_backward_row<T, TPR, DROP, SETS>(a, row, lds, flip);
    } else {
        const int64_t stride = (int64_t)gridDim.x - sh.row_blocks;
        for (int64_t b = (int64_t)blockIdx.x - sh.row_blocks; b < sh.col_tiles * sh.segs; b += stride) {
            column_sums<T, DROP, SETS>(a, sh, b, lds);
            __syncthreads();   // the sums are read before the next tile's are written
        }
    }
}

// ---- layer norm, backward: rows that fit the registers of their threads ---------------------------------
// One pass over x and dy writes dx and keeps sums of dy u and dy for the thread's columns over all rows of its
// workgroup, in registers; at the end the workgroup's rows are summed (lanes, then waves, in a fixed order) and
// one partial row of both gradients is left in the workspace for norm_reduce_kernel.  x and dy stay as they were
// loaded: u and g are formed twice, before and after the row's two means, which is cheaper than the registers of a
// widened copy.  Bound by memory while a wave's registers hold a row: 819,200 x 128 bfloat16 take 122 us with the
// reduction (5.1 TB/s over x, dy and dx), 16,384 x 4,096 bfloat16 91 us (4.4 TB/s: 5 of them are the reduction of 512
// partial rows); beyond 8,192 columns by what a workgroup of 1,024 threads can hold (6,000 x 16,000 bfloat16: 158 us,
// 3.6 TB/s; with dw's sums in registers 171; with dropout, where x and dy are fetched again for the second half, 176 --
// held they take 207 for 16-bit types, but 155 against 164 for float at 4,000 x 12,000).  Doubles with 1,024 threads
// spill 48 bytes a lane (124 with dropout): 3,000 x 8,000 take 190 us with the reduction and 226, 115 at a copy's rate.
// The mean is read as one number of the sums' type, without the remainder that the forward pass takes off as well: u is
// off by up to half a step of |mean| times r, alike over a row.
template <class T, int TPR, int NV, bool DROP>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_backward_kernel(NormArgs a) {
    using A = wide_t<T>;
    constexpr int kRows = norm_threads(TPR) / TPR;
    constexpr bool kWide = TPR == 1024 && NV > 1;    // dw's sums in LDS, the dropped units as bits
    constexpr bool kKeep = NV * sizeof(T) <= 8 && !(kWide && DROP && sizeof(T) == 2);   // registers for x and dy of the row
    constexpr bool kAhead = NV * sizeof(T) <= 4;     // and of the next row
    constexpr bool kHold = NV == 1 && sizeof(T) < 8; // registers for the weights
    constexpr int kCols = TPR * NV * kChunk;
    __shared__ A lds[TPR > 64 ? kRowLds<TPR, 2> : 4 * kCols];
    __shared__ A wide[kWide ? kCols : 1];             // [chunk of a thread][half][thread][4]
    int flip = 0;
    const int t = threadIdx.x % TPR, cols = (int)a.cols;
    int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * kRows;
    const T* weight = static_cast<const T*>(a.weight);
    const A inv = (A)a.inv_cols, scale = (A)a.drop.scale;
    uint32_t off[2] = {0, 0};
    if constexpr (DROP) drop_offset(a.drop, off);
    A gw[kWide ? 1 : NV][kChunk], gb[NV][kChunk], hg[kChunk];
    auto in_lds = [&](int v, int k) -> A& { return wide[((v * 2 + k / 4) * TPR + t) * 4 + k % 4]; };
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int k = 0; k < kChunk; ++k) {
            gb[v][k] = 0;
            if constexpr (kWide) in_lds(v, k) = 0;
            else gw[v][k] = 0;
        }
    auto gains = [&](int v, A (&g)[kChunk]) {
#pragma unroll
        for (int k = 0; k < kChunk; ++k) g[k] = 1;
        if (weight) load_full(weight + spot_of(cols, t + v * TPR).col, g);
    };
    Raw<T> rx[kKeep ? NV : 1], rd[kKeep ? NV : 1], nx[kAhead ? NV : 1], nd[kAhead ? NV : 1];
    A m = 0, r = 0, nm = 0, nr = 0;
    auto fetch_one = [&](int64_t at, int v, Raw<T>& fx, Raw<T>& fd) {
        const int col = spot_of(cols, t + v * TPR).col;
        fetch_full(static_cast<const T*>(a.x) + at * a.x_stride + col, fx);
        fetch_full(static_cast<const T*>(a.dy) + at * a.dy_stride + col, fd);
    };
    auto fetch = [&](int64_t at, Raw<T>* fx, Raw<T>* fd, A& fm, A& fr) {
        fm = static_cast<const A*>(a.mean)[at]; fr = static_cast<const A*>(a.rstd)[at];
        if constexpr (kKeep) {
#pragma unroll
            for (int v = 0; v < NV; ++v) fetch_one(at, v, fx[v], fd[v]);
        }
    };
    if (row < a.rows) fetch(row, rx, rd, m, r);
    if constexpr (kHold) gains(0, hg);
    while (row < a.rows) {
        const int64_t next = row + step;
        if constexpr (kAhead) {
            if (next < a.rows) fetch(next, nx, nd, nm, nr);
        }
        Keep keep[kWide ? 1 : NV];
        uint32_t bits[NV];
        auto drop_again = [&](int v, A (&c)[kChunk]) {
            if constexpr (DROP && kWide) drop_bits(bits[v], scale, c);
            else if constexpr (DROP) drop_chunk(keep[v], scale, c);
        };
        A s[2] = {0, 0};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Spot p = spot_of(cols, t + v * TPR);
            A u[kChunk], g[kChunk], w[kChunk];
            if constexpr (!kKeep) fetch_one(row, v, rx[0], rd[0]);
            widen_chunk(rx[kKeep ? v : 0], u);
            widen_chunk(rd[kKeep ? v : 0], g);
            if constexpr (!kHold) gains(v, w);
            if constexpr (DROP) {
                Keep& kp = keep[kWide ? 0 : v];
                kp = keep_at(a.drop, off, p, (uint32_t)row);
                drop_chunk(kp, scale, u);
                if constexpr (kWide) bits[v] = pack(kp);
            }
            clear_head(p.skip, g);
            if constexpr (kWide) {
#pragma unroll
                for (int k = 0; k < kChunk; ++k) gw[0][k] = in_lds(v, k);
            }
#pragma unroll
            for (int k = 0; k < kChunk; ++k) {
                u[k] = (u[k] - m) * r;
                gw[kWide ? 0 : v][k] += g[k] * u[k];
                if constexpr (kWide) in_lds(v, k) = gw[0][k];
                gb[v][k] += g[k];
                g[k] *= kHold ? hg[k] : w[k];
                s[0] += g[k];
                s[1] += g[k] * u[k];
            }
        }
        row_sums<TPR>(s, lds, flip);
        const A c1 = s[0] * inv, c2 = s[1] * inv;
        if (a.dx) {
            T* dx = static_cast<T*>(a.dx) + row * a.y_stride;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const Spot p = spot_of(cols, t + v * TPR);
                if (p.skip == kChunk) continue;
                A u[kChunk], g[kChunk], w[kChunk];
                if constexpr (!kKeep) fetch_one(row, v, rx[0], rd[0]);
                forget(rx[kKeep ? v : 0]);
                forget(rd[kKeep ? v : 0]);
                widen_chunk(rx[kKeep ? v : 0], u);
                widen_chunk(rd[kKeep ? v : 0], g);
                if constexpr (!kHold) gains(v, w);
                drop_again(v, u);
#pragma unroll
                for (int k = 0; k < kChunk; ++k) {
                    u[k] = (u[k] - m) * r;
                    g[k] *= kHold ? hg[k] : w[k];
                    g[k] = ((g[k] - c1) - u[k] * c2) * r;
                }
                drop_again(v, g);
                Raw<T> o;
                narrow_chunk<T>(g, o);
                put_part<T, kChunk>(dx + p.col, o.w);
            }
        }
        row = next;
        if constexpr (kAhead) {
#pragma unroll
            for (int v = 0; v < NV; ++v) { rx[v] = nx[v]; rd[v] = nd[v]; }
            m = nm; r = nr;
        } else {
            if (row < a.rows) fetch(row, rx, rd, m, r);
        }
    }
    if (!a.workspace) return;
    A* part = static_cast<A*>(a.workspace) + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (TPR > 64) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const Spot p = spot_of(cols, t + v * TPR);
#pragma unroll
            for (int k = 0; k < kChunk; ++k)
                if (k >= p.skip) {
                    if constexpr (kWide) part[p.col + k] = in_lds(v, k);
                    else part[p.col + k] = gw[v][k];
                    part[cols + p.col + k] = gb[v][k];
                }
        }
    } else {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const Spot p = spot_of(cols, t + v * TPR);
#pragma unroll
                for (int k = 0; k < kChunk; ++k) {
                    A z = which ? gb[v][k] : gw[kWide ? 0 : v][k];
#pragma unroll
                    for (int n = TPR; n < 64; n <<= 1) z += __shfl_xor(z, n, 64);
                    if ((threadIdx.x & 63) < TPR && k >= p.skip) lds[(threadIdx.x >> 6) * kCols + p.col + k] = z;
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += 256)
                part[which * cols + c] = (lds[c] + lds[kCols + c]) + (lds[2 * kCols + c] + lds[3 * kCols + c]);
        }
    }
}

// Sums the partial rows of the two gradients: 16 columns and 64 rows at a time, then the 64 sums in a fixed order.  A few
// loads one after the other: 2 to 4 us for 512 rows of 128 or 256 columns, 7 for 4,096 columns (16 MB, in the caches).
template <class T>
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const wide_t<T>* __restrict__ part, int64_t parts, int64_t cols,
                                                           T* dweight, T* dbias) {
    using A = wide_t<T>;
    __shared__ A lds[64][17];
    const int lane = threadIdx.x % 16, slot = threadIdx.x / 16;
    for (int64_t tile = blockIdx.x; tile * 16 < 2 * cols; tile += gridDim.x) {
        const int64_t at = tile * 16 + lane;   // over [2][cols]
        A s = 0;
        if (at < 2 * cols) {
#pragma unroll 8
            for (int64_t p = slot; p < parts; p += 64) s += part[p * 2 * cols + at];
        }
        lds[slot][lane] = s;   // what others read of the tile before lies behind a barrier
        __syncthreads();
        for (int half = 32; half > 0; half >>= 1) {
            if (slot < half) lds[slot][lane] += lds[slot + half][lane];
            __syncthreads();
        }
        if (slot == 0 && at < 2 * cols) {
            T* out = at < cols ? dweight : dbias;
            if (out) out[at < cols ? at : at - cols] = (T)lds[0][lane];
        }
    }
}

// dweight and dbias of no rows at all
template <class T>
__global__ __launch_bounds__(256) void norm_zero_kernel(T* dweight, T* dbias, int64_t cols) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    if (dweight) dweight[c] = (T)0;
    if (dbias) dbias[c] = (T)0;
}

// ---- launching --------------------------------------------------------------------------------------
// Calls f with a value of the element type.
template <class F>
auto with_type(LayerType type, F f) {
    switch (type) {
        case kF64: return f(double{});
        case kF32: return f(float{});
        case kBF16: return f(__bf16{});
        default: return f(_Float16{});
    }
}
template <class F>
auto with_flag(bool on, F f) {
    return on ? f(std::true_type{}) : f(std::false_type{});
}

// Threads of a row and chunks of a thread for rows that are held in registers: calls f(threads, chunks) and returns
// true, or returns false for rows that are too narrow or too wide.  Up to 1,024 columns (forward 1,536) a row stays in
// a wave: no barrier (60,000 x 1,500 bfloat16 with dropout forward: 85 us with 64 x 3, 111 with 256 x 1; backward, where
// the sums take the registers, 180 and 152).  Beyond, the smallest workgroup with one chunk a thread, while there is
// one: at 16,384 x 4,096 bfloat16 the backward pass takes 91 us with 512 x 1, 122 with 256 x 2 and 145 with 128 x 4,
// because the next row's registers then fit beside the sums; the forward pass, which has no sums, does not care (47.2,
// 50.3, 53.0).  Backward rows of more than one chunk a thread keep dw's sums in LDS; where registers still run out, the
// split kernels take them, which read x and dy twice: 4,000 x 24,000 bfloat16 take 186 us with 1,024 x 3 and 262 split,
// but 312 and 264 with dropout; 2,500 x 32,000 300 and 227; 1,500 x 12,000 double 299 and 171.
template <int N> using int_c = std::integral_constant<int, N>;
template <class T, bool FORWARD, bool DROP, class F>
bool with_row_shape(int64_t cols, F f) {
    if (cols < kChunk) return false;
    if (cols <= 32) f(int_c<4>{}, int_c<1>{});
    else if (cols <= 64) f(int_c<8>{}, int_c<1>{});
    else if (cols <= 128) f(int_c<16>{}, int_c<1>{});
    else if (cols <= 256) f(int_c<32>{}, int_c<1>{});
    else if (cols <= 512) f(int_c<64>{}, int_c<1>{});
    else if (cols <= 1024) f(int_c<64>{}, int_c<2>{});
    else if (FORWARD && cols <= 1536) f(int_c<64>{}, int_c<FORWARD ? 3 : 2>{});
    else if (cols <= 2048) f(int_c<256>{}, int_c<1>{});
    else if (cols <= 4096) f(int_c<512>{}, int_c<1>{});
    else if (cols <= 8192) f(int_c<FORWARD ? 512 : 1024>{}, int_c<FORWARD ? 2 : 1>{});
    else if constexpr (!FORWARD && sizeof(T) == 8) return false;
    else if (cols <= 16384) f(int_c<1024>{}, int_c<2>{});
    else if constexpr (!FORWARD && DROP) return false;
    else if (cols <= 24576) f(int_c<1024>{}, int_c<3>{});
    else if constexpr (!FORWARD) return false;
    else if (cols <= 32768) f(int_c<1024>{}, int_c<4>{});
    else return false;
    return true;
}

// Workgroups of the forward pass: several rounds of what the device holds at once, so that a workgroup that falls
// behind is made up for (819,200 x 128 bfloat16: 80.7 us with 4,096, 76.5 with 8,192 or 16,384, 84.6 with one for
// every 16 rows, which spends its time on starting them).
template <int TPR>
int64_t forward_blocks(int64_t rows) {
    constexpr int kRows = norm_threads(TPR) / TPR;
    return std::min((rows + kRows - 1) / kRows, TPR <= 256 ? (int64_t)8192 : (int64_t)2048 * 256 / norm_threads(TPR));
}

// Workgroups of the backward pass.  Each leaves a partial row of both gradients, so here fewer are better until the
// device is no longer full: a row in a wave, 512 (24,576 x 128 float: 12.0 us, 13.0 with 256, 14.0 with 1,024), and 768
// where rows are many (819,200 x 128 bfloat16: 122.8 us, 127.6 with 512, 127.0 with 1,024); a row in a workgroup, what
// fills the device four waves deep, and half of it for a few thousand rows of one workgroup of 256 threads each (3,000 x
// 2,000 bfloat16: 21.3 us, 27.5 with 1,024; 9,001 x 1,500 half: 33.3 with 512, 31.3).
template <int TPR>
int64_t backward_blocks(int64_t rows) {
    constexpr int kRows = norm_threads(TPR) / TPR;
    const int64_t most = TPR <= 64    ? std::min<int64_t>(768, std::max<int64_t>(rows / (kRows * 16), 512))
                         : TPR == 256 ? (rows < 8192 ? 512 : 1024)
                                      : (int64_t)1024 * 256 / norm_threads(TPR);
    return std::min((rows + kRows - 1) / kRows, most);
}
// Up to so many rows the split kernel does it all in one launch: narrow rows until its column workgroups have walked
// longer than a second launch takes (bfloat16 x 128: 768 rows 6.9 us split and 6.8 in two, 1,200 rows 10.1 and 7.0; x
// 1,024: 1,024 rows 8.4 and 9.8), wide ones until reading x and dy twice does (x 4,096: 1,200 rows 17.7 and 26.7, 3,000
// 35 and 32; x 8,192: 1,024 rows 24 and 30, 1,200 32 and 30).
int64_t split_rows(int64_t cols) { return cols <= 512 ? 768 : cols > 1024 && cols <= 4096 ? 1536 : 1024; }

// Threads of a row in the kernels for several networks at once, whose rows have up to 256 columns: one chunk each.
template <class F>
void with_set_shape(int64_t cols, F f) {
    if (cols <= 128) f(int_c<16>{});
    else f(int_c<32>{});
}

// Rows of one column workgroup.  Up to 1,024 rows it takes them all and leaves the gradients themselves; beyond, where a
// second launch sums segments anyway, they are short (1,200 x 2,048 bfloat16: 10.0 us, 13.0 with segments of 1,024).
int64_t seg_rows(int64_t rows) { return rows <= 1024 ? 1024 : 512; }

SplitShape split_shape(const NormArgs& a, int tpr) {
    SplitShape sh{};
    sh.row_blocks = a.dx ? std::min((a.rows + 256 / tpr - 1) / (256 / tpr), kMaxBlocks) : 0;
    sh.col_tiles = (a.cols + kTileCols - 1) / kTileCols;
    if (a.sets.count) {
        sh.segs = a.sets.count; sh.seg_rows = a.sets.set_rows;
    } else {
        sh.seg_rows = seg_rows(a.rows);
        sh.segs = (a.rows + sh.seg_rows - 1) / sh.seg_rows;
    }
    return sh;
}

}  // namespace

DropArgs make_drop(double p, int64_t seed, int64_t offset, const int64_t* offset_dev) {
    DropArgs d{};
    d.threshold = (uint32_t)std::nearbyint(p * 65536.0);
    d.scale = d.threshold < 65536 ? 65536.0 / (65536.0 - d.threshold) : 0.0;
    d.key[0] = (uint32_t)(uint64_t)seed; d.key[1] = (uint32_t)((uint64_t)seed >> 32);
    d.offset[0] = (uint32_t)(uint64_t)offset; d.offset[1] = (uint32_t)((uint64_t)offset >> 32);
    d.offset_dev = offset_dev;
    return d;
}

hipError_t launch_dropout(LayerType type, int64_t rows, int64_t cols, int64_t x_stride, int64_t y_stride, const void* x,
                          void* y, const DropArgs& drop, hipStream_t s) {
    DropShape sh{};
    sh.cols = cols; sh.x_stride = x_stride; sh.y_stride = y_stride;
    sh.per_row = (uint32_t)((cols + kChunk - 1) / kChunk);
    // with l = ceil(log2 per_row) and magic = ceil(2^(31+l) / per_row) the quotient is exact below 2^31, and the
    // magic number stays below 2^32
    int l = 0;
    while (((uint64_t)1 << l) < sh.per_row) ++l;
    sh.shift = 31 + l;
    sh.magic = (uint32_t)((((uint64_t)1 << (31 + l)) + sh.per_row - 1) / sh.per_row);
    const int64_t per_launch = ((int64_t)1 << 31) / sh.per_row - 1;   // rows: at least 7, for fewer than 2^28 chunks a row
    for (int64_t r = 0; r < rows; r += per_launch) {
        const int64_t n = rows - r < per_launch ? rows - r : per_launch;
        sh.row0 = r;
        sh.chunks = (uint32_t)(n * sh.per_row);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_flag(drop.threshold != 0, [&](auto on) {
                hipLaunchKernelGGL((dropout_kernel<T, decltype(on)::value>), dim3((sh.chunks + 255) / 256), dim3(256), 0, s,
                                   static_cast<const T*>(x), static_cast<T*>(y), sh, drop);
            });
        });
    }
    return hipGetLastError();
}

hipError_t launch_norm_forward(LayerType type, const NormArgs& args, hipStream_t s) {
    if (args.rows == 0) return hipSuccess;
    NormArgs a = args;
    a.inv_cols = 1.0 / (double)a.cols;
    if (a.sets.count) {
        with_set_shape(a.cols, [&](auto tpr) { with_flag(a.drop.threshold != 0, [&](auto drop) {
            constexpr int TPR = decltype(tpr)::value, kRows = 256 / TPR;
            hipLaunchKernelGGL((norm_forward_walk_kernel<double, TPR, decltype(drop)::value, true>),
                               dim3((unsigned)std::min((a.rows + kRows - 1) / kRows, kMaxBlocks)), dim3(256), 0, s, a);
        }); });
        return hipGetLastError();
    }
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(a.drop.threshold != 0, [&](auto drop) {
            constexpr bool D = decltype(drop)::value;
            const bool held = with_row_shape<T, true, D>(a.cols, [&](auto tpr, auto nv) {
                constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
                hipLaunchKernelGGL((norm_forward_kernel<T, TPR, NV, D>), dim3((unsigned)forward_blocks<TPR>(a.rows)), dim3(norm_threads(TPR)), 0, s, a);
            });
            if (held) return;
            if (a.cols < kChunk)
                hipLaunchKernelGGL((norm_forward_walk_kernel<T, 1, D, false>), dim3((unsigned)std::min((a.rows + 255) / 256, kMaxBlocks)), dim3(256), 0, s, a);
            else
                hipLaunchKernelGGL((norm_forward_walk_kernel<T, 1024, D, false>), dim3((unsigned)std::min(a.rows, kMaxBlocks)), dim3(1024), 0, s, a);
        });
    });
    return hipGetLastError();
}

size_t norm_backward_workspace(LayerType type, int64_t rows, int64_t cols, bool drop) {
    return with_type(type, [&](auto t) -> size_t {
        using T = decltype(t);
        int64_t parts = 0;
        if (rows > split_rows(cols))
            with_flag(drop, [&](auto on) {
                with_row_shape<T, false, decltype(on)::value>(cols, [&](auto tpr, auto) { parts = backward_blocks<decltype(tpr)::value>(rows); });
            });
        if (!parts) {
            const int64_t segs = (rows + seg_rows(rows) - 1) / seg_rows(rows);
            parts = segs > 1 ? segs : 0;
        }
        return (size_t)parts * 2 * cols * sizeof(wide_t<T>);
    });
}

hipError_t launch_norm_backward(LayerType type, const NormArgs& args, hipStream_t s) {
    NormArgs a = args;
    a.inv_cols = 1.0 / (double)a.cols;
    if (a.sets.count) {
        with_set_shape(a.cols, [&](auto tpr) { with_flag(a.drop.threshold != 0, [&](auto drop) {
            constexpr int TPR = decltype(tpr)::value;
            const SplitShape sh = split_shape(a, TPR);
            hipLaunchKernelGGL((norm_backward_split_kernel<double, TPR, decltype(drop)::value, true>),
                               dim3((unsigned)(sh.row_blocks + std::min(sh.col_tiles * sh.segs, kMaxBlocks))), dim3(256), 0, s, a, sh);
        }); });
        return hipGetLastError();
    }
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool vectors = a.dweight || a.dbias;
        if (a.rows == 0) {
            if (vectors)
                hipLaunchKernelGGL(norm_zero_kernel<T>, dim3((unsigned)((a.cols + 255) / 256)), dim3(256), 0, s,
                                   static_cast<T*>(a.dweight), static_cast<T*>(a.dbias), a.cols);
            return;
        }
        if (!vectors && !a.dx) return;
        int64_t parts = 0;
        with_flag(a.drop.threshold != 0, [&](auto drop) {
            constexpr bool D = decltype(drop)::value;
            if (a.rows > split_rows(a.cols))
                with_row_shape<T, false, D>(a.cols, [&](auto tpr, auto nv) {
                    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
                    NormArgs b = a;
                    if (!vectors) b.workspace = nullptr;
                    parts = backward_blocks<TPR>(a.rows);
                    hipLaunchKernelGGL((norm_backward_kernel<T, TPR, NV, D>), dim3((unsigned)parts), dim3(norm_threads(TPR)), 0, s, b);
                });
            if (parts) return;
            // a thread for rows of one chunk; a workgroup for those of more than four chunks a lane, and for those of
            // more than one where rows are few (bfloat16, 64 x 2,048: 3.7 us, 6.4 with a wave a row; 1,024 x 2,048: 10.0, 8.7)
            const auto split = [&](auto tpr) {
                constexpr int TPR = decltype(tpr)::value;
                const SplitShape sh = split_shape(a, TPR);
                const int64_t col_blocks = vectors ? std::min(sh.col_tiles * sh.segs, kMaxBlocks) : 0;
                hipLaunchKernelGGL((norm_backward_split_kernel<T, TPR, D, false>), dim3((unsigned)(sh.row_blocks + col_blocks)), dim3(256), 0, s, a, sh);
                if (sh.segs > 1) parts = sh.segs;
            };
            if (a.cols <= kChunk) split(int_c<1>{});
            else if (a.cols <= 512 || (a.cols <= 2048 && a.rows > 512)) split(int_c<64>{});
            else split(int_c<256>{});
        });
        if (parts && vectors)
            hipLaunchKernelGGL(norm_reduce_kernel<T>, dim3((unsigned)std::min((2 * a.cols + 15) / 16, kMaxBlocks)), dim3(1024), 0, s,
                               static_cast<const wide_t<T>*>(a.workspace), parts, a.cols, static_cast<T*>(a.dweight),
                               static_cast<T*>(a.dbias));
    });
    return hipGetLastError();
}

// ---- C entry points ------------------------------------------------------------------------------------
namespace {

// Makes the call's device current and puts the caller's back at the end.
struct DeviceScope {
    int before = -1;
    bool changed = false;
    int32_t enter(int device) {
        if (hipGetDevice(&before) != hipSuccess)
            return fail(EPI_ERR_DEVICE, "no HIP device available: the engine has no CPU fallback");
        if (device == before) return EPI_OK;
        if (int32_t rc = use_device(device)) return rc;
        changed = true;
        return EPI_OK;
    }
    ~DeviceScope() { if (changed) (void)hipSetDevice(before); }
};

// [lo, hi) in bytes of `rows` rows of `cols` elements
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    if (!a || !b) return false;
    const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
    return p < q + (uintptr_t)b_bytes && q < p + (uintptr_t)a_bytes;
}

struct Extent {
    int64_t size;   // bytes of an element
    int64_t plane(int64_t rows, int64_t cols, int64_t stride) const { return rows ? ((rows - 1) * stride + cols) * size : 0; }
};

int32_t check_desc(const char* who, const epi_layer_desc* d, Extent* e) {
    if (!d) return fail(EPI_ERR_BAD_ARGUMENT, "%s: null descriptor", who);
    if (d->dtype < EPI_F64 || d->dtype > EPI_F16) return fail(EPI_ERR_BAD_ARGUMENT, "%s: dtype %d outside [0,3]", who, d->dtype);
    e->size = d->dtype == EPI_F64 ? 8 : d->dtype == EPI_F32 ? 4 : 2;
    if (d->rows < 0 || d->cols < 1) return fail(EPI_ERR_BAD_ARGUMENT, "%s: %lld rows of %lld columns", who, (long long)d->rows, (long long)d->cols);
    if (d->rows >= (int64_t)1 << 31 || d->cols >= (int64_t)1 << 31)
        return fail(EPI_ERR_UNSUPPORTED, "%s: %lld rows of %lld columns: both must be below 2^31", who, (long long)d->rows, (long long)d->cols);
    if (!(d->dropout >= 0.0 && d->dropout <= 1.0)) return fail(EPI_ERR_BAD_ARGUMENT, "%s: dropout %g outside [0,1]", who, d->dropout);
    if (reinterpret_cast<uintptr_t>(d->offset_dev) % 8) return fail(EPI_ERR_BAD_ARGUMENT, "%s: offset_dev is not aligned", who);
    return EPI_OK;
}

int32_t check_plane(const char* who, const char* name, const void* p, int64_t rows, int64_t cols, int64_t stride, int64_t size, bool written) {
    if (rows == 0) return EPI_OK;
    if (!p) return fail(EPI_ERR_BAD_ARGUMENT, "%s: %s is null", who, name);
    if (reinterpret_cast<uintptr_t>(p) % size) return fail(EPI_ERR_BAD_ARGUMENT, "%s: %s is not aligned to its elements", who, name);
    int64_t last, bytes;   // the rows end within 2^63 bytes
    if (rows > 1 && (stride < 0 || (written && stride < cols) || stride >= (int64_t)1 << 40 ||
                     __builtin_mul_overflow(rows - 1, stride, &last) || __builtin_add_overflow(last, cols, &last) ||
                     __builtin_mul_overflow(last, size, &bytes)))
        return fail(EPI_ERR_BAD_ARGUMENT, "%s: %s has a row stride of %lld for %lld columns", who, name, (long long)stride, (long long)cols);
    return EPI_OK;
}

int32_t check_vector(const char* who, const char* name, const void* p, int64_t size) {
    if (reinterpret_cast<uintptr_t>(p) % size) return fail(EPI_ERR_BAD_ARGUMENT, "%s: %s is not aligned to its elements", who, name);
    return EPI_OK;
}

}  // namespace
}  // namespace epi

using namespace epi;

EPI_API int32_t epi_dropout(const epi_layer_desc* d, const void* x, void* y, void* stream) {
    const char* who = "dropout";
    Extent e{};
    if (int32_t rc = check_desc(who, d, &e)) return rc;
    if (int32_t rc = check_plane(who, "x", x, d->rows, d->cols, d->x_stride, e.size, false)) return rc;
    if (int32_t rc = check_plane(who, "y", y, d->rows, d->cols, d->y_stride, e.size, true)) return rc;
    const bool in_place = x == y && (d->rows < 2 || d->x_stride == d->y_stride);
    if (!in_place && overlap(x, e.plane(d->rows, d->cols, d->x_stride), y, e.plane(d->rows, d->cols, d->y_stride)))
        return fail(EPI_ERR_BAD_ARGUMENT, "dropout: x and y overlap without being the same rows");
    DeviceScope dev;
    if (int32_t rc = dev.enter(d->device)) return rc;
    if (d->rows == 0) return EPI_OK;
    HIP_TRY(launch_dropout((LayerType)d->dtype, d->rows, d->cols, d->x_stride, d->y_stride, x, y,
                           make_drop(d->dropout, d->seed, d->offset, d->offset_dev), static_cast<hipStream_t>(stream)));
    return EPI_OK;
}

EPI_API int32_t epi_layer_norm_forward(const epi_layer_desc* d, const void* x, const void* weight, const void* bias, void* y,
                                       void* mean, void* rstd, void* stream) {
    const char* who = "layer_norm_forward";
    Extent e{};
    if (int32_t rc = check_desc(who, d, &e)) return rc;
    const int64_t wide = e.size == 8 ? 8 : 4, vec = d->cols * e.size, stat = d->rows * wide;
    if (!(d->eps >= 0.0)) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_forward: eps %g is negative", d->eps);
    if (int32_t rc = check_plane(who, "x", x, d->rows, d->cols, d->x_stride, e.size, false)) return rc;
    if (int32_t rc = check_plane(who, "y", y, d->rows, d->cols, d->y_stride, e.size, true)) return rc;
    if (int32_t rc = check_vector(who, "weight", weight, e.size)) return rc;
    if (int32_t rc = check_vector(who, "bias", bias, e.size)) return rc;
    if (int32_t rc = check_vector(who, "mean", mean, wide)) return rc;
    if (int32_t rc = check_vector(who, "rstd", rstd, wide)) return rc;
    if (!mean != !rstd) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_forward: mean and rstd are asked for together");
    const int64_t ny = e.plane(d->rows, d->cols, d->y_stride), nx = e.plane(d->rows, d->cols, d->x_stride);
    const bool in_place = x == y && (d->rows < 2 || d->x_stride == d->y_stride);
    if ((!in_place && overlap(x, nx, y, ny)) || overlap(y, ny, weight, vec) || overlap(y, ny, bias, vec) ||
        overlap(y, ny, mean, stat) || overlap(y, ny, rstd, stat) || overlap(x, nx, mean, stat) || overlap(x, nx, rstd, stat) ||
        overlap(mean, stat, rstd, stat) || overlap(mean, stat, weight, vec) || overlap(mean, stat, bias, vec) ||
        overlap(rstd, stat, weight, vec) || overlap(rstd, stat, bias, vec))
        return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_forward: an output overlaps another array (y may be x itself)");
    DeviceScope dev;
    if (int32_t rc = dev.enter(d->device)) return rc;
    NormArgs a{};
    a.rows = d->rows; a.cols = d->cols; a.x_stride = d->x_stride; a.y_stride = d->y_stride;
    a.x = x; a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd; a.eps = d->eps;
    a.drop = make_drop(d->dropout, d->seed, d->offset, d->offset_dev);
    HIP_TRY(launch_norm_forward((LayerType)d->dtype, a, static_cast<hipStream_t>(stream)));
    return EPI_OK;
}

EPI_API int32_t epi_layer_norm_backward_workspace(const epi_layer_desc* d, size_t* bytes) {
    Extent e{};
    if (int32_t rc = check_desc("layer_norm_backward_workspace", d, &e)) return rc;
    if (!bytes) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_backward_workspace: null argument");
    *bytes = norm_backward_workspace((LayerType)d->dtype, d->rows, d->cols, make_drop(d->dropout, 0, 0, nullptr).threshold != 0);
    return EPI_OK;
}

EPI_API int32_t epi_layer_norm_backward(const epi_layer_desc* d, const void* x, const void* dy, const void* weight,
                                        const void* mean, const void* rstd, void* dx, void* dweight, void* dbias,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "layer_norm_backward";
    Extent e{};
    if (int32_t rc = check_desc(who, d, &e)) return rc;
    const int64_t wide = e.size == 8 ? 8 : 4, vec = d->cols * e.size, stat = d->rows * wide;
    if (int32_t rc = check_plane(who, "x", x, d->rows, d->cols, d->x_stride, e.size, false)) return rc;
    if (int32_t rc = check_plane(who, "dy", dy, d->rows, d->cols, d->dy_stride, e.size, false)) return rc;
    if (dx) {
        if (int32_t rc = check_plane(who, "dx", dx, d->rows, d->cols, d->y_stride, e.size, true)) return rc;
    }
    if (d->rows && (!mean || !rstd)) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_backward: mean or rstd is null");
    const struct { const char* name; const void* p; int64_t size; } vectors[] = {
        {"weight", weight, e.size}, {"mean", mean, wide}, {"rstd", rstd, wide}, {"dweight", dweight, e.size},
        {"dbias", dbias, e.size}, {"workspace", workspace, wide}};
    for (const auto& v : vectors)
        if (int32_t rc = check_vector(who, v.name, v.p, v.size)) return rc;
    size_t need = 0;
    if (dweight || dbias) need = norm_backward_workspace((LayerType)d->dtype, d->rows, d->cols, make_drop(d->dropout, 0, 0, nullptr).threshold != 0);
    if (need && (!workspace || workspace_bytes < need))
        return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_backward: a workspace of %zu bytes is needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    const struct { const void* p; int64_t n; } in[] = {
        {x, e.plane(d->rows, d->cols, d->x_stride)}, {dy, e.plane(d->rows, d->cols, d->dy_stride)}, {weight, vec}, {mean, stat}, {rstd, stat}};
    const struct { const void* p; int64_t n; } out[] = {
        {dx, e.plane(d->rows, d->cols, d->y_stride)}, {dweight, vec}, {dbias, vec}, {workspace, (int64_t)need}};
    for (int i = 0; i < 4; ++i) {
        for (const auto& j : in)
            if (overlap(out[i].p, out[i].n, j.p, j.n)) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_backward: an output overlaps an input");
        for (int j = 0; j < i; ++j)
            if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return fail(EPI_ERR_BAD_ARGUMENT, "layer_norm_backward: two outputs overlap");
    }
    DeviceScope dev;
    if (int32_t rc = dev.enter(d->device)) return rc;
    NormArgs a{};
    a.rows = d->rows; a.cols = d->cols; a.x_stride = d->x_stride; a.y_stride = d->y_stride; a.dy_stride = d->dy_stride;
    a.x = x; a.dy = dy; a.weight = weight; a.mean = const_cast<void*>(mean); a.rstd = const_cast<void*>(rstd);
    a.dx = dx; a.dweight = dweight; a.dbias = dbias; a.workspace = workspace;
    a.drop = make_drop(d->dropout, d->seed, d->offset, d->offset_dev);
    HIP_TRY(launch_norm_backward((LayerType)d->dtype, a, static_cast<hipStream_t>(stream)));
    return EPI_OK;
}
