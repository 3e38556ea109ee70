// gfx950 kernels of the training step: log probabilities of sampled tokens, the clipped policy loss and its
// gradient, the global gradient norm and clipping, AdamW.  None of them is a contraction (no MFMA): all are passes
// over HBM, and what they are built for is to read and write each element once.
//
// Rates on one MI355X that the figures below are held against: a nontemporal read of 4 GiB 7.1 TB/s, a copy
// 5.63 TB/s (read and written bytes together).  "Rows of 152064" and the like are positions of bf16 logits.
#include "step.h"

#include <crx_math.h>

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace crx {
namespace {

constexpr float kLn2 = 0.69314718055994531f;
// a log2-scaled difference whose power of 2 is 0, as that of everything below it: stands for -inf where it is multiplied
// (and no larger, so that its products with an upstream gradient stay finite: they are multiplied by that 0)
constexpr float kFloor = -256.0f;

__device__ __forceinline__ uint32_t wave_lane() { return threadIdx.x & 63u; }
// (the generic min template of the HIP headers goes through double precision)
__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }

// ------------------------------------------------------------------ elements
struct Bf16 {
    uint16_t u;
};
struct F16 {
    uint16_t u;
};

// Elements of each type, N to a 16-byte access (at any element's alignment).
template <typename T>
struct Lane;
template <>
struct Lane<Bf16> {
    static constexpr uint32_t N = 8;
    template <int WORDS = 4>
    __device__ static __forceinline__ void unpack(const uint32_t *w, float *f) {
        for (int k = 0; k < WORDS; ++k) {
            f[2 * k] = __builtin_bit_cast(float, w[k] << 16);
            f[2 * k + 1] = __builtin_bit_cast(float, w[k] & 0xFFFF0000u);
        }
    }
    template <int WORDS = 4>
    __device__ static __forceinline__ void pack(const float *f, uint32_t *w) {
        for (int k = 0; k < WORDS; ++k) w[k] = pack_bf16(f[2 * k], f[2 * k + 1]);
    }
    __device__ static __forceinline__ float get(const void *p) {
        return __builtin_bit_cast(float, (uint32_t) * static_cast<const uint16_t *>(p) << 16);
    }
    __device__ static __forceinline__ void put(void *p, float f) { *static_cast<uint16_t *>(p) = (uint16_t)pack_bf16(f, 0.0f); }
};
template <>
struct Lane<F16> {
    static constexpr uint32_t N = 8;
    template <int WORDS = 4>
    __device__ static __forceinline__ void unpack(const uint32_t *w, float *f) {
        for (int k = 0; k < WORDS; ++k) {
            f[2 * k] = f16_to_float(w[k] & 0xFFFFu);
            f[2 * k + 1] = f16_to_float(w[k] >> 16);
        }
    }
    template <int WORDS = 4>
    __device__ static __forceinline__ void pack(const float *f, uint32_t *w) {
        for (int k = 0; k < WORDS; ++k) w[k] = pack_f16(f[2 * k], f[2 * k + 1]);
    }
    __device__ static __forceinline__ float get(const void *p) { return f16_to_float(*static_cast<const uint16_t *>(p)); }
    __device__ static __forceinline__ void put(void *p, float f) { *static_cast<uint16_t *>(p) = (uint16_t)pack_f16(f, 0.0f); }
};
template <>
struct Lane<float> {
    static constexpr uint32_t N = 4;
    template <int WORDS = 4>
    __device__ static __forceinline__ void unpack(const uint32_t *w, float *f) { __builtin_memcpy(f, w, 4 * WORDS); }
    template <int WORDS = 4>
    __device__ static __forceinline__ void pack(const float *f, uint32_t *w) { __builtin_memcpy(w, f, 4 * WORDS); }
    __device__ static __forceinline__ float get(const void *p) { return *static_cast<const float *>(p); }
    __device__ static __forceinline__ void put(void *p, float f) { *static_cast<float *>(p) = f; }
};

template <typename T>
__device__ __forceinline__ void load(const uint8_t *p, float *f) {
    uint32_t w[4];
    load16(p, w);
    Lane<T>::unpack(w, f);
}
template <typename T>
__device__ __forceinline__ void store(uint8_t *p, const float *f) {
    uint32_t w[4];
    Lane<T>::pack(f, w);
    store16(p, w);
}
template <typename T>
__device__ __forceinline__ void store_stream(uint8_t *p, const float *f) {
    uint32_t w[4];
    Lane<T>::pack(f, w);
    store16_stream(p, w);
}

// Elements [lo, hi) of a contiguous array as whole 16-byte vectors at 16-byte boundaries and the elements at the edges
// (fewer than N on either side).  Vectors across such boundaries are slow where they are written past the caches:
// 41M bf16 gradients at odd addresses were clipped in 54 us so, 38 through the caches.
template <typename T>
struct Span {
    uint64_t lo, before, first, vectors;  // edges before the first vector's element, vectors
    uint32_t edges;
    __device__ __forceinline__ Span(const uint8_t *p, uint64_t lo_, uint64_t hi) {
        constexpr uint32_t N = Lane<T>::N;
        lo = lo_;
        const uint64_t n = hi - lo, off = (16u - ((uintptr_t)(p + lo * sizeof(T)) & 15u)) % 16u / sizeof(T);
        before = off < n ? off : n;
        first = lo + before;
        vectors = (hi - first) / N;
        edges = (uint32_t)(before + (hi - first - vectors * N));
    }
    __device__ __forceinline__ uint64_t edge(uint32_t k) const {  // element of the k-th edge
        return k < before ? lo + k : first + vectors * Lane<T>::N + (k - before);
    }
};

// ------------------------------------------------------------------ a row's softmax
// Of the elements seen so far: the largest (m), the sum of 2^d and of d 2^d with d = (x - m) c, the log2
// exponent of the softmax.  m starts at the lowest finite value, so x - m is never inf - inf: a row (or a
// part of one) of nothing but -inf ends with s = 0, and one of the type's lowest value with every 2^d = 1.
struct Stat {
    float m, s, t;
};
__device__ __forceinline__ Stat no_elements() { return Stat{-FLT_MAX, 0.0f, 0.0f}; }

template <bool ENT>
__device__ __forceinline__ void add_elements(Stat &a, const float *f, int n, float c) {
    float top = a.m;
    for (int k = 0; k < n; ++k) top = fmaxf(top, f[k]);
    const float d = fmaxf((a.m - top) * c, kFloor), back = exp2_hw(d);
    if (ENT) a.t = back * (a.t + d * a.s);
    a.s *= back;
    a.m = top;
    for (int k = 0; k < n; ++k) {
        const float q = (f[k] - top) * c, e = exp2_hw(q);
        a.s += e;
        if (ENT) a.t += e * fmaxf(q, kFloor);
    }
}

template <bool ENT>
__device__ __forceinline__ Stat join(const Stat &a, const Stat &b, float c) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - r.m) * c, kFloor), db = fmaxf((b.m - r.m) * c, kFloor);
    const float fa = exp2_hw(da), fb = exp2_hw(db);
    r.s = a.s * fa + b.s * fb;
    r.t = ENT ? fa * (a.t + da * a.s) + fb * (b.t + db * b.s) : 0.0f;
    return r;
}

// The first lane's value in every lane.
__device__ __forceinline__ float first_lane(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(uint32_t, v)));
}

// The joined statistics of a wavefront's first `lanes` lanes (a power of two), the same in every lane: what the lanes
// compute may differ in the last place, so the first one's counts.
template <bool ENT>
__device__ __forceinline__ Stat wave_stat(Stat a, int lanes, float c) {
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        Stat b = a;
        b.m = __shfl_xor(a.m, o, 64);
        b.s = __shfl_xor(a.s, o, 64);
        if (ENT) b.t = __shfl_xor(a.t, o, 64);
        a = join<ENT>(a, b, c);
    }
    return Stat{first_lane(a.m), first_lane(a.s), ENT ? first_lane(a.t) : 0.0f};
}

// The statistics of the workgroup's elements, the same in every thread: each wavefront's, then those joined by every
// wavefront alike.
template <int BLOCK, bool ENT>
__device__ __forceinline__ Stat block_stat(Stat a, float c, Stat *lds) {
    a = wave_stat<ENT>(a, 64, c);
    if constexpr (BLOCK == 64) return a;
    if (wave_lane() == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    a = wave_stat<ENT>(lds[wave_lane() & (BLOCK / 64 - 1)], BLOCK / 64, c);
    __syncthreads();
    return a;
}

// Loads a thread has in flight in a row's two passes: with 32 wavefronts on a CU, one load each covers too little
// of the memory's latency.  Loss and gradient of 16384 rows of 152064 bf16 logits: 1962 us with one load each,
// 1911 with four and two.
constexpr uint32_t kStatLoads = 4, kGradLoads = 2;

// Vectors of each thread that the loss's first pass leaves in LDS for its second, the first it reads (the caches have
// lost those soonest): four are 64 KB of a workgroup of 1024, two to a CU; 16384 rows of 152064 bf16 then took 1907 us
// without, 1886 with one, 1844 with two, 1843 with four.  Of rows beyond kAloneBytes a workgroup holds eight, 128 KB, and
// has the CU to itself: half as many rows in work for the last-level cache to keep, and less to read from it.  Loss and
// gradient, us, four and eight held: 4000 rows of 65536 bf16 153 / 203, of 100000 294 / 301, of 130000 411 / 397, of
// 200000 594 / 565; 2000 of 152064 fp32 472 / 449; 16384 rows of 152064 bf16 1801 / 1751 (nine: 1748; eight, and four more
// in registers: 1727; all of the row on chip, in registers and LDS: 1774, for nothing overlaps the next row's read).
constexpr uint32_t kHeld = 4, kHeldAlone = 8;
constexpr uint64_t kAloneBytes = 229376;

// The statistics of a row's elements [lo, hi).  KEEP: the row is read again, so the caches should hold it; and HOLD
// vectors of each thread are left in `hold`.
template <typename T, int BLOCK, bool ENT, bool KEEP, uint32_t HOLD = 0>
__device__ __forceinline__ Stat row_stat(const uint8_t *x, uint32_t lo, uint32_t hi, float c, Stat *lds, uint4 *hold = nullptr) {
    constexpr uint32_t N = Lane<T>::N, STEP = BLOCK * N;
    Stat a = no_elements();
    float f[N];
    uint32_t w[kStatLoads][4];
    const Span<T> sp(x, lo, hi);
    const uint32_t first = (uint32_t)sp.first, body = first + (uint32_t)sp.vectors * N;
    uint32_t i = first + threadIdx.x * N;
    if (HOLD) {
        uint32_t v[HOLD ? HOLD : 1][4];  // all read at once
        for (uint32_t u = 0; u < HOLD; ++u)
            if (i + u * STEP < body) load16_stream(x + (uint64_t)(i + u * STEP) * sizeof(T), v[u]);
        for (uint32_t u = 0; u < HOLD; ++u) {
            if (i + u * STEP >= body) break;
            hold[u * BLOCK + threadIdx.x] = make_uint4(v[u][0], v[u][1], v[u][2], v[u][3]);
            Lane<T>::unpack(v[u], f);
            add_elements<ENT>(a, f, N, c);
        }
        i += HOLD * STEP;
    }
    for (; i + (kStatLoads - 1) * STEP < body; i += kStatLoads * STEP) {
        for (uint32_t u = 0; u < kStatLoads; ++u) {
            const uint8_t *const p = x + (uint64_t)(i + u * STEP) * sizeof(T);
            if (KEEP) load16(p, w[u]);
            else load16_stream(p, w[u]);
        }
        for (uint32_t u = 0; u < kStatLoads; ++u) {
            Lane<T>::unpack(w[u], f);
            add_elements<ENT>(a, f, N, c);
        }
    }
    for (; i < body; i += STEP) {
        load<T>(x + (uint64_t)i * sizeof(T), f);
        add_elements<ENT>(a, f, N, c);
    }
    if (threadIdx.x < sp.edges) {
        f[0] = Lane<T>::get(x + sp.edge(threadIdx.x) * sizeof(T));
        add_elements<ENT>(a, f, 1, c);
    }
    return block_stat<BLOCK, ENT>(a, c, lds);
}

// a (1[j = y] - p_j) - h p_j (ln p_j + H) of a row's elements [lo, hi), rounded once.  The row is read from its end: what
// the pass before read last is nearest in the caches (1993 -> 1962 us at 16384 rows of 152064 bf16).  `hold`: what
// row_stat has left of these vectors.
template <typename T, int BLOCK, bool ENT, uint32_t HOLD = 0>
__device__ __forceinline__ void row_grad(const uint8_t *x, uint8_t *g, uint32_t lo, uint32_t hi, float c, const Stat &st,
                                         uint32_t y, float a, float h, float H, const uint4 *hold = nullptr) {
    constexpr uint32_t N = Lane<T>::N, STEP = BLOCK * N;
    float f[N];
    uint32_t w[kGradLoads][4];
    const float inv = 1.0f / st.s, ls = ENT ? logf(st.s) : 0.0f;
    auto one = [&](float v) {
        const float q = (v - st.m) * c, p = exp2_hw(q) * inv;
        return ENT ? p * (-a - h * (fmaxf(q, kFloor) * kLn2 - ls + H)) : -a * p;
    };
    auto vector = [&](uint32_t i, const uint32_t *v) {
        Lane<T>::unpack(v, f);
        for (uint32_t k = 0; k < N; ++k) f[k] = one(f[k]);
        if (y - i < N)
            for (uint32_t k = 0; k < N; ++k) f[k] += y - i == k ? a : 0.0f;
        store_stream<T>(g + (uint64_t)i * sizeof(T), f);
    };
    const Span<T> sp(g, lo, hi);
    const uint32_t first = (uint32_t)sp.first, vectors = (uint32_t)sp.vectors;
    uint32_t left = vectors > threadIdx.x ? (vectors - threadIdx.x - 1) / BLOCK + 1 : 0;  // this thread's
    // the passes' vectors are the same where logits and gradient are aligned alike
    const uint32_t held = HOLD && (((uintptr_t)x ^ (uintptr_t)g) & 15u) == 0 ? HOLD : 0;
    while (left >= kGradLoads + held) {
        const uint32_t i = first + ((left - 1) * BLOCK + threadIdx.x) * N;
        for (uint32_t u = 0; u < kGradLoads; ++u) load16_stream(x + (uint64_t)(i - u * STEP) * sizeof(T), w[u]);
        for (uint32_t u = 0; u < kGradLoads; ++u) vector(i - u * STEP, w[u]);
        left -= kGradLoads;
    }
    while (left > held) {
        const uint32_t i = first + (--left * BLOCK + threadIdx.x) * N;
        load16_stream(x + (uint64_t)i * sizeof(T), w[0]);
        vector(i, w[0]);
    }
    while (left) {
        const uint4 v = hold[--left * BLOCK + threadIdx.x];
        const uint32_t q[4] = {v.x, v.y, v.z, v.w};
        vector(first + (left * BLOCK + threadIdx.x) * N, q);
    }
    if (threadIdx.x < sp.edges) {
        const uint32_t i = (uint32_t)sp.edge(threadIdx.x);
        float v = one(Lane<T>::get(x + (uint64_t)i * sizeof(T)));
        if (i == y) v += a;
        Lane<T>::put(g + (uint64_t)i * sizeof(T), v);
    }
}

template <typename T, int BLOCK>
__device__ __forceinline__ void row_zero(uint8_t *g, uint32_t lo, uint32_t hi) {
    const uint32_t none[4] = {};
    const Span<T> sp(g, lo, hi);
    uint8_t *const at = g + sp.first * sizeof(T);
    for (uint32_t i = threadIdx.x; i < (uint32_t)sp.vectors; i += BLOCK) store16_stream(at + (uint64_t)i * 16, none);
    if (threadIdx.x < sp.edges) Lane<T>::put(g + sp.edge(threadIdx.x) * sizeof(T), 0.0f);
}

// ------------------------------------------------------------------ a row's place
struct Row {
    uint32_t b, t;
    const uint8_t *x;
    bool on;     // not masked
    uint32_t y;  // its token, or kNoToken where the id is outside the vocabulary
};
constexpr uint32_t kNoToken = 0xFFFFFFFFu;

template <typename T>
__device__ __forceinline__ Row row_at(const RowsIn &in, uint32_t r) {
    Row o;
    o.b = r / in.tokens;
    o.t = r - o.b * in.tokens;
    o.x = static_cast<const uint8_t *>(in.x) + ((int64_t)o.b * in.sb + (int64_t)o.t * in.st) * (int64_t)sizeof(T);
    o.on = !in.mask.p || in.mask.p[(int64_t)o.b * in.mask.sb + (int64_t)o.t * in.mask.st] != 0;
    o.y = kNoToken;
    if (o.on) {
        const int64_t at = (int64_t)o.b * in.ids_sb + (int64_t)o.t * in.ids_st;
        const int64_t id = in.id_bytes == 8 ? static_cast<const int64_t *>(in.ids)[at] : (int64_t) static_cast<const int32_t *>(in.ids)[at];
        if (id >= 0 && id < (int64_t)in.vocab) o.y = (uint32_t)id;
    }
    return o;
}

template <typename T>
__device__ __forceinline__ T value_at(const At<T> &a, const Row &r) {
    return a.p[(int64_t)r.b * a.sb + (int64_t)r.t * a.st];
}

// a + b = hi + lo, but for infinities
struct Two {
    float hi, lo;
};
__device__ __forceinline__ Two two_sum(float a, float b) {
    const float s = a + b, t = s - a;
    return Two{s, (a - (s - t)) + (b - t)};
}

// log softmax at the row's token, (x_y - m) / T - ln s, as a float and what it was rounded by: its difference to another
// policy's (0.1) is what the loss takes, and would be off by the last place of a number of the size of 10.  ln s is k ln 2,
// with ln 2 in two parts, and ln f, s = 2^k f with f near 1.  NaN for an id outside the vocabulary, and for a row without a
// finite logit.
template <typename T>
__device__ __forceinline__ Two row_logp(const RowsIn &in, const Row &r, const Stat &st) {
    if (r.y == kNoToken) return Two{NAN, 0.0f};
    const Two d = two_sum(Lane<T>::get(r.x + (uint64_t)r.y * sizeof(T)), -st.m);
    const float q = rounded(d.hi * in.inv_temp);  // (not fused with the sum that follows)
    const float q_lo = fmaf(d.hi, in.inv_temp, -q) + fmaf(d.hi, in.inv_temp_lo, d.lo * in.inv_temp);
    int k = 0;
    float f = frexpf(st.s, &k);
    if (f < 0.70710678f) {
        f *= 2.0f;
        --k;
    }
    const float ln = (float)k * 1.42860682e-6f + logf(f);
    const Two a = two_sum(q, (float)k * -0.693145752f), b = two_sum(a.hi, -ln);  // (exact products: 0.693145752 has 15 bits)
    const float lo = a.lo + b.lo + q_lo;
    return Two{b.hi, fabsf(lo) < 1.0f ? lo : 0.0f};
}

// ------------------------------------------------------------------ scores
// log p_y = (x_y - m) / T - ln s and H = ln s - (ln 2) t / s, from one pass over the row (Stat).  Bound by its read: 8 x
// 512 rows of 152064, a quarter of them masked (0.93 GB), take 134-142 us, 6.6-6.9 TB/s; with every exponential replaced
// by a multiply 134.  Vectors are read past the caches: through them the read takes a tenth longer.
template <typename T, bool ENT>
__device__ __forceinline__ void write_score(const RowsIn &in, const ScoreOut &o, uint32_t r, const Row &row, const Stat &st) {
    const Two lp = row_logp<T>(in, row, st);
    o.logp[r] = lp.hi + lp.lo;
    if (ENT) o.entropy[r] = logf(st.s) - kLn2 * (st.t / st.s);
    if (o.stats) o.stats[r] = make_float2(st.m, st.s);
}
__device__ __forceinline__ void write_no_score(const ScoreOut &o, uint32_t r) {
    o.logp[r] = 0.0f;
    if (o.entropy) o.entropy[r] = 0.0f;
    if (o.stats) o.stats[r] = make_float2(0.0f, 1.0f);
}

template <typename T, int BLOCK, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_score(RowsIn in, ScoreOut o) {
    __shared__ Stat lds[BLOCK / 64];
    const uint32_t r = in.row0 + blockIdx.x;
    const Row row = row_at<T>(in, r);
    if (!row.on) {
        if (threadIdx.x == 0) write_no_score(o, r);
        return;
    }
    const Stat st = row_stat<T, BLOCK, ENT, false>(row.x, 0, in.vocab, in.c, lds);
    if (threadIdx.x == 0) write_score<T, ENT>(in, o, r, row, st);
}

// ------------------------------------------------------------------ counts of a mask
// Adds the unmasked positions of [begin, end), in the order of their rows, to their sequences' counts (integers: in any
// order).  One wavefront: 64 positions at a time, eight times 64 loaded together, and one addition for all that follow
// each other in a sequence.  Where 64 positions hold the end of one sequence at most, their places follow from the ones
// before; a division for each took 14 us for 16384 positions on 16 wavefronts.
__device__ __forceinline__ void count_run(const At<uint8_t> &mask, uint32_t begin, uint32_t end, uint32_t tokens, uint32_t *counts) {
    constexpr uint32_t LOADS = 8;
    if (begin >= end) return;
    const uint32_t lane = wave_lane();
    uint32_t held = 0, of = 0;                       // positions counted and not yet added, of this sequence
    uint32_t b0 = begin / tokens, t0 = begin - b0 * tokens;  // where the next 64 begin (the same in every lane, as the above)
    for (uint32_t at = begin; at < end;) {
        uint32_t b[LOADS];
        uint8_t on[LOADS];
        for (uint32_t u = 0; u < LOADS; ++u) {
            uint32_t t = t0 + lane;
            b[u] = b0;
            if (tokens < 64) {
                b[u] += t / tokens;
                t %= tokens;
            } else if (t >= tokens) {
                b[u] += 1;
                t -= tokens;
            }
            on[u] = 0;
            if (at + 64 * u + lane < end) on[u] = mask.p[(int64_t)b[u] * mask.sb + (int64_t)t * mask.st];
            t0 += 64;
            if (tokens < 64) {
                b0 += t0 / tokens;
                t0 %= tokens;
            } else if (t0 >= tokens) {
                b0 += 1;
                t0 -= tokens;
            }
        }
        for (uint32_t u = 0; u < LOADS && at < end; ++u, at += 64) {
            const uint64_t set = __ballot(on[u] != 0);
            const uint32_t first = (uint32_t)__builtin_amdgcn_readfirstlane(b[u]);
            const bool one = __ballot(b[u] != first) == 0;
            if (first != of || !one) {
                if (lane == 0 && held) atomicAdd(&counts[of], held);
                held = 0;
                of = first;
            }
            if (one) held += (uint32_t)__popcll(set);
            else if (on[u]) atomicAdd(&counts[b[u]], 1u);
        }
    }
    if (lane == 0 && held) atomicAdd(&counts[of], held);
}

// The counts of k_mask_few, below, by one workgroup; lds: seqs + 2 values.
template <int BLOCK>
__device__ __forceinline__ void count_few(const At<uint8_t> &mask, uint32_t seqs, uint32_t tokens, uint32_t *counts, uint32_t *lds) {
    for (uint32_t b = threadIdx.x; b < seqs + 2; b += BLOCK) lds[b] = 0;
    __syncthreads();
    const uint32_t rows = seqs * tokens, run = (rows + BLOCK - 1) / BLOCK * 64, begin = (threadIdx.x >> 6) * run;
    count_run(mask, begin, min(begin + run, rows), tokens, lds);
    __syncthreads();
    uint32_t n = 0, some = 0;
    for (uint32_t b = threadIdx.x; b < seqs; b += BLOCK) {
        counts[b] = lds[b];
        n += lds[b];
        some += lds[b] != 0;
    }
    if (n) {
        atomicAdd(&lds[seqs], n);
        atomicAdd(&lds[seqs + 1], some);
    }
    __syncthreads();
    if (threadIdx.x < 2) counts[seqs + threadIdx.x] = lds[seqs + threadIdx.x];
}

// ------------------------------------------------------------------ few rows: a row's parts on workgroups of their own
// One row of 152064 on one workgroup occupies one CU of 256; cut into 64 parts it is two launches of 3.6 and 2.2 us, and
// 100 rows of 152064 take what their bytes take.  The gradient's second read of the few rows comes from the L2 caches.
// A loss's mask is counted by one workgroup more of the first launch (14 rows of 20011: 18.0 -> 15.6 us a call).
// the part of the workgroup's row that is its own
struct Part {
    uint32_t r, k, lo, hi;
};
__device__ __forceinline__ Part part_of(const RowsIn &in, const Parts &p, uint32_t i) {
    Part o;
    o.r = i / p.n;
    o.k = i - o.r * p.n;
    o.lo = o.k * p.size;
    o.hi = min(in.vocab, o.lo + p.size);
    return o;
}

template <typename T, bool ENT>
__global__ __launch_bounds__(kPartBlock) void k_part_stat(RowsIn in, Parts p) {
    __shared__ Stat lds[kPartBlock / 64];
    __shared__ uint32_t each[kPartRows + 2];
    if (blockIdx.x == in.rows * p.n) {  // the workgroup more of a loss with a mask
        count_few<kPartBlock>(in.mask, in.seqs, in.tokens, p.counts, each);
        return;
    }
    const Part at = part_of(in, p, blockIdx.x);
    const Row row = row_at<T>(in, at.r);
    if (!row.on) return;
    const Stat st = row_stat<T, kPartBlock, ENT, true>(row.x, at.lo, at.hi, in.c, lds);
    if (threadIdx.x == 0) {
        float *const w = p.stat + 3 * (uint64_t)blockIdx.x;
        w[0] = st.m;
        w[1] = st.s;
        w[2] = st.t;
    }
}

// a row's statistics from its parts', the same in every thread that asks
template <bool ENT>
__device__ __forceinline__ Stat join_parts(const Parts &p, uint32_t r, float c) {
    Stat a = no_elements();
    if (wave_lane() < p.n) {
        const float *const w = p.stat + 3 * ((uint64_t)r * p.n + wave_lane());
        a = Stat{w[0], w[1], w[2]};
    }
    return wave_stat<ENT>(a, 64, c);
}

template <typename T, bool ENT>
__global__ __launch_bounds__(64) void k_score_parts(RowsIn in, Parts p, ScoreOut o) {
    const uint32_t r = blockIdx.x;
    const Row row = row_at<T>(in, r);
    if (!row.on) {
        if (threadIdx.x == 0) write_no_score(o, r);
        return;
    }
    const Stat st = join_parts<ENT>(p, r, in.c);
    if (threadIdx.x == 0) write_score<T, ENT>(in, o, r, row, st);
}

// ------------------------------------------------------------------ gradients from kept statistics
// dL/dx_j of row_grad with p_j from the row's kept largest logit and sum (8 bytes a row): one read and one write of
// the row and nothing to join.  4000 rows of 152064: 425 us, 5.7 TB/s, the rate of a copy.
template <typename T, int BLOCK, bool ENT>
__global__ __launch_bounds__(BLOCK) void k_rows_grad(RowsIn in, Parts p, GradIn g) {
    const float up = g.upstream ? *g.upstream : 1.0f;
    if (g.unless_one && up == 1.0f) return;
    for (uint32_t i = blockIdx.x; i < in.rows * p.n; i += gridDim.x) {
        const Part at = part_of(in, p, i);
        const Row row = row_at<T>(in, at.r);
        uint8_t *const out = static_cast<uint8_t *>(g.grad) + (uint64_t)at.r * in.vocab * sizeof(T);
        if (!row.on) {
            row_zero<T, BLOCK>(out, at.lo, at.hi);
            continue;
        }
        const Stat st{g.stats[at.r].x, g.stats[at.r].y, 0.0f};
        float a = g.slope ? g.slope[at.r] * up : g.up_logp.p ? value_at(g.up_logp, row) * in.inv_temp : 0.0f;
        if (row.y == kNoToken) a = NAN;
        const float h = ENT ? value_at(g.up_entropy, row) * in.inv_temp : 0.0f;
        row_grad<T, BLOCK, ENT>(row.x, out, at.lo, at.hi, in.c, st, row.y, a, h, ENT ? g.entropy[at.r] : 0.0f);
    }
}

// ------------------------------------------------------------------ policy loss
// counts[b]: unmasked positions of sequence b; counts[seqs], counts[seqs + 1]: their sum, and the number of
// sequences with any.  Few enough positions: all by one workgroup, in one launch.
__global__ __launch_bounds__(1024) void k_mask_few(At<uint8_t> mask, uint32_t seqs, uint32_t tokens, uint32_t *counts) {
    __shared__ uint32_t each[kFewSeqs + 2];
    count_few<1024>(mask, seqs, tokens, counts, each);
}

// Otherwise in three launches: counts cleared; a wavefront for each kMaskRun positions; the sum.
constexpr uint32_t kMaskRun = 4096;

__global__ __launch_bounds__(1024) void k_mask_zero(uint32_t *counts, uint32_t seqs) {
    for (uint64_t b = (uint64_t)blockIdx.x * 1024 + threadIdx.x; b < seqs; b += (uint64_t)gridDim.x * 1024) counts[b] = 0;
}

__global__ __launch_bounds__(256) void k_mask_counts(At<uint8_t> mask, uint32_t rows, uint32_t tokens, uint32_t *counts) {
    const uint64_t begin = ((uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kMaskRun;
    count_run(mask, (uint32_t)min64(begin, rows), (uint32_t)min64(begin + kMaskRun, rows), tokens, counts);
}

__global__ __launch_bounds__(1024) void k_mask_total(uint32_t *counts, uint32_t seqs) {
    __shared__ uint32_t lds[32];
    uint32_t n = 0, some = 0;
#pragma unroll 8
    for (uint32_t b = threadIdx.x; b < seqs; b += 1024) {
        const uint32_t v = counts[b];
        n += v;
        some += v != 0;
    }
    for (int o = 32; o > 0; o >>= 1) {
        n += __shfl_xor(n, o, 64);
        some += __shfl_xor(some, o, 64);
    }
    if (wave_lane() == 0) {
        lds[threadIdx.x >> 6] = n;
        lds[16 + (threadIdx.x >> 6)] = some;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        n = 0;
        for (int w = 0; w < 16; ++w) n += lds[16 * threadIdx.x + w];
        counts[seqs + threadIdx.x] = n;
    }
}

// The weight of an unmasked position.
__device__ __forceinline__ float row_weight(const RowsIn &in, const PolicyIn &p, uint32_t b) {
    if (p.reduction == kSum) return 1.0f;
    if (p.reduction == kMeanToken) return 1.0f / (float)(p.counts ? p.counts[in.seqs] : in.rows);
    return 1.0f / ((float)(p.counts ? p.counts[in.seqs + 1] : in.seqs) * (float)(p.counts ? p.counts[b] : in.tokens));
}

struct Token {
    float loss, kl, cut, slope;  // slope: the loss's derivative by the log probability
};

// e^d - 1 - d.  The difference loses leading digits where d is small (five bits at 1/16): below 1, its series, d^2 times the
// sum of d^n / (n + 2)!, of which eleven terms are kept (the twelfth is under 2^-30 of the sum).
__device__ __forceinline__ float kl_term(float d, float expm1_d) {
    if (!(fabsf(d) < 1.0f)) return expm1_d - d;
    constexpr float over[] = {0.5f, 1.0f / 6, 1.0f / 24, 1.0f / 120, 1.0f / 720, 1.0f / 5040, 1.0f / 40320, 1.0f / 362880,
                              1.0f / 3628800, 1.0f / 39916800, 1.0f / 479001600};
    float p = over[10];
#pragma unroll
    for (int k = 9; k >= 0; --k) p = fmaf(d, p, over[k]);
    return d * d * p;
}

// The position's loss.
__device__ __forceinline__ Token token_loss(const PolicyIn &p, const Row &r, Two logp) {
    const float A = value_at(p.adv, r), ratio = expf((logp.hi - value_at(p.old, r)) + logp.lo);
    const float held = fminf(fmaxf(ratio, p.low), p.high);
    const float free = ratio * A, bound = (ratio != ratio ? ratio : held) * A;
    Token o;
    // the smaller of the two; NaN where either is
    o.loss = -(free != free || free < bound ? free : bound);
    const bool cut = (A > 0.0f && ratio > p.high) || (A < 0.0f && ratio < p.low);
    o.cut = cut ? 1.0f : 0.0f;
    o.slope = cut ? 0.0f : -free;
    o.kl = 0.0f;
    if (p.ref.p) {
        const float d = (value_at(p.ref, r) - logp.hi) - logp.lo, g = expm1f(d);
        o.kl = kl_term(d, g);
        o.loss += p.kl * o.kl;
        o.slope -= p.kl * g;
    }
    return o;
}

// What a position leaves behind; returns the factor of its gradient.
template <typename T>
__device__ __forceinline__ float write_policy(const RowsIn &in, const PolicyIn &p, const PolicyOut &o, uint32_t r,
                                              const Row &row, const Stat &st, bool writes) {
    const Two logp = row_logp<T>(in, row, st);
    const float w = row_weight(in, p, row.b);
    const Token k = token_loss(p, row, logp);
    const float a = p.scale * w * in.inv_temp * k.slope;
    if (writes) {
        o.logp[r] = logp.hi + logp.lo;
        if (o.stats) o.stats[r] = make_float2(st.m, st.s);
        if (o.slope) o.slope[r] = a;
        o.terms[r] = w * k.loss;
        o.terms[in.rows + r] = w * k.kl;
        o.terms[2 * (uint64_t)in.rows + r] = w * k.cut;
    }
    return a;
}
__device__ __forceinline__ void write_no_policy(const RowsIn &in, const PolicyOut &o, uint32_t r) {
    o.logp[r] = 0.0f;
    if (o.stats) o.stats[r] = make_float2(0.0f, 1.0f);
    if (o.slope) o.slope[r] = 0.0f;
    for (int k = 0; k < 3; ++k) o.terms[(uint64_t)k * in.rows + r] = 0.0f;
}

// One workgroup per row: its softmax, its loss, and (with a gradient) the row read again, from LDS and the
// caches, and its gradient written.  A row of 152064 is 304 KB: with one workgroup of 1024 on each CU the rows in work
// are 78 MB, of which 128 KB a row are in LDS; the 256 MB last-level cache keeps the rest from the first pass to the
// second, so HBM sees one read and one write (with the first pass read past the caches 16384 rows of 152064 took 2517 us
// instead of 1907).  Bound by the mix of reads and writes: those rows, a tenth of them masked (9.5 GB), take this kernel
// 1750 us, 5.4 TB/s; when it took 1843, 1834 with multiplies for the exponentials and 1739 without the second read at all.
template <typename T, int BLOCK, uint32_t HOLD>
__global__ __launch_bounds__(BLOCK) void k_policy(RowsIn in, PolicyIn p, PolicyOut o) {
    __shared__ Stat lds[BLOCK / 64];
    __shared__ uint4 hold[HOLD * BLOCK];
    const uint32_t r = in.row0 + blockIdx.x;
    const Row row = row_at<T>(in, r);
    uint8_t *const out = o.grad ? static_cast<uint8_t *>(o.grad) + (uint64_t)r * in.vocab * sizeof(T) : nullptr;
    if (!row.on) {
        if (threadIdx.x == 0) write_no_policy(in, o, r);
        if (out) row_zero<T, BLOCK>(out, 0, in.vocab);
        return;
    }
    const Stat st = out ? row_stat<T, BLOCK, false, true, HOLD>(row.x, 0, in.vocab, in.c, lds, hold)
                        : row_stat<T, BLOCK, false, false>(row.x, 0, in.vocab, in.c, lds);
    const float a = write_policy<T>(in, p, o, r, row, st, threadIdx.x == 0);
    if (!out) return;
    if (a == 0.0f) row_zero<T, BLOCK>(out, 0, in.vocab);  // clipped, or without an advantage
    else row_grad<T, BLOCK, false, HOLD>(row.x, out, 0, in.vocab, in.c, st, row.y, a, 0.0f, 0.0f, hold);
}

// The same from parts' statistics: every workgroup of a row joins them and writes its part of the gradient.
template <typename T>
__global__ __launch_bounds__(kPartBlock) void k_policy_parts(RowsIn in, Parts parts, PolicyIn p, PolicyOut o) {
    const Part at = part_of(in, parts, blockIdx.x);
    const Row row = row_at<T>(in, at.r);
    const bool writes = at.k == 0 && threadIdx.x == 0;
    uint8_t *const out = o.grad ? static_cast<uint8_t *>(o.grad) + (uint64_t)at.r * in.vocab * sizeof(T) : nullptr;
    if (!row.on) {
        if (writes) write_no_policy(in, o, at.r);
        if (out) row_zero<T, kPartBlock>(out, at.lo, at.hi);
        return;
    }
    const Stat st = join_parts<false>(parts, at.r, in.c);
    const float a = write_policy<T>(in, p, o, at.r, row, st, writes);
    if (!out) return;
    if (a == 0.0f) row_zero<T, kPartBlock>(out, at.lo, at.hi);
    else row_grad<T, kPartBlock, false>(row.x, out, at.lo, at.hi, in.c, st, row.y, a, 0.0f, 0.0f);
}

// The sums of the rows' terms, in 64 bits and in a fixed order
__global__ __launch_bounds__(1024) void k_policy_sums(const float *terms, uint32_t rows, float scale, float *loss, float *kl, float *clipped) {
    __shared__ double lds[16];
    const float *const t = terms + (uint64_t)blockIdx.x * rows;
    double n = 0.0;
    uint64_t i = threadIdx.x;
    for (; i + 7 * 1024 < rows; i += 8 * 1024) {
        float v[8];
        for (uint32_t k = 0; k < 8; ++k) v[k] = t[i + k * 1024];
        for (uint32_t k = 0; k < 8; ++k) n += (double)v[k];
    }
    for (; i < rows; i += 1024) n += (double)t[i];
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (wave_lane() == 0) lds[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) n += lds[w];
        if (blockIdx.x == 0) *loss = (float)(n * (double)scale);
        else *(blockIdx.x == 1 ? kl : clipped) = (float)n;
    }
}

// ------------------------------------------------------------------ passes over lists of tensors
// The tensor that holds unit u, the last whose first unit is at or before it: each lane of the wavefront asks for some
// of them (a search by halves is a chain of seven dependent loads before a workgroup's first element).
template <uint32_t CAP, typename L>
__device__ __forceinline__ uint32_t tensor_of(const L &l, uint32_t u) {
    uint32_t before = 0;
    for (uint32_t k = 0; k < CAP; k += 64) {
        const uint32_t i = k + wave_lane();
        before += (uint32_t)__popcll(__ballot(i < l.count && l.first[i < CAP ? i : 0] <= u));
    }
    return before - 1;
}

// each(t, lo, hi) for the elements [lo, hi) of tensor t that are share i of n: the list's units are dealt out evenly and
// in order, so a share is one range of one tensor, or one for each of a few.
template <uint32_t CAP, typename L, typename F>
__device__ __forceinline__ void for_share(const L &l, uint32_t i, uint32_t n, F &&each) {
    const uint64_t units = l.first[l.count];
    uint32_t u = (uint32_t)(units * i / n);
    const uint32_t end = (uint32_t)(units * (i + 1) / n);
    if (u >= end) return;
    for (uint32_t t = tensor_of<CAP>(l, u); u < end; ++t) {
        const uint32_t begin = l.first[t], stop = min(end, l.first[t + 1]);
        const uint64_t lo = (uint64_t)(u - begin) * kUnit, hi = (uint64_t)(stop - begin) * kUnit;
        each(t, lo, hi < l.n[t] ? hi : l.n[t]);
        u = stop;
    }
}

// Loads a thread has in flight in the passes over lists.  The norm has one: its 64-bit sums leave few registers, and so eight
// wavefronts fit a SIMD, which hides more (7.6e9 bf16 gradients 2216 us; with two loads 2293, with four 2298).
constexpr uint32_t kClipLoads = 2;

template <typename T, bool KEEP>
__device__ __forceinline__ double squares(const uint8_t *p, uint64_t lo, uint64_t hi) {
    constexpr uint32_t N = Lane<T>::N, STEP = 256 * N;
    double n = 0.0;
    float f[N];
    uint32_t w[4];
    const Span<T> sp(p, lo, hi);
    const uint64_t body = sp.first + sp.vectors * N;
    for (uint64_t i = sp.first + threadIdx.x * N; i < body; i += STEP) {
        if (KEEP) load16(p + i * sizeof(T), w);
        else load16_stream(p + i * sizeof(T), w);
        Lane<T>::unpack(w, f);
        for (uint32_t k = 0; k < N; ++k) n += (double)f[k] * (double)f[k];
    }
    if (threadIdx.x < sp.edges) {
        const double v = (double)Lane<T>::get(p + sp.edge(threadIdx.x) * sizeof(T));
        n += v * v;
    }
    return n;
}

// Squares are summed in 64 bits: no gradient's square over- or underflows, and the pass stays bound by its reads: 7.6e9
// bf16 gradients (15.2 GB) in 2210 us, 6.9 TB/s
// (2.58 ms through the caches, when it was 2.30 past them).  Gradients that fit the last-level cache are read through it (KEEP):
// the pass that follows finds them there.
template <typename T, bool KEEP>
__global__ __launch_bounds__(256) void k_norm_part(NormList l, double *partial, uint32_t used) {
    __shared__ double lds[4];
    double n = 0.0;
    for_share<kNormTensors>(l, blockIdx.x, gridDim.x, [&](uint32_t t, uint64_t lo, uint64_t hi) {
        n += squares<T, KEEP>(static_cast<const uint8_t *>(l.p[t]), lo, hi);
    });
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (wave_lane() == 0) lds[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (blockIdx.x < used ? partial[blockIdx.x] : 0.0) + (lds[0] + lds[1] + lds[2] + lds[3]);
}

__global__ __launch_bounds__(1024) void k_norm_sum(const double *partial, uint32_t count, float *norm) {
    __shared__ double lds[16];
    double n = 0.0;
    for (uint32_t i = threadIdx.x; i < count; i += 1024) n += partial[i];
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    if (wave_lane() == 0) lds[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x < 16) {
        n = lds[threadIdx.x];
        for (int o = 8; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
        if (threadIdx.x == 0) *norm = (float)sqrt(n);
    }
}

// min(1, max_norm / (norm + 1e-6)); NaN of a NaN
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
    const float c = max_norm / (norm + 1e-6f);
    return c > 1.0f ? 1.0f : c;
}

template <typename T, bool KEEP>
__device__ __forceinline__ void scale_range(uint8_t *p, uint64_t lo, uint64_t hi, float c) {
    constexpr uint32_t N = Lane<T>::N, STEP = 256 * N;
    float f[N];
    uint32_t w[kClipLoads][4];
    const Span<T> sp(p, lo, hi);
    const uint64_t body = sp.first + sp.vectors * N;
    uint64_t i = sp.first + threadIdx.x * N;
    auto scale = [&](uint64_t at, const uint32_t *v) {
        Lane<T>::unpack(v, f);
        for (uint32_t k = 0; k < N; ++k) f[k] *= c;
        if (KEEP) store<T>(p + at * sizeof(T), f);
        else store_stream<T>(p + at * sizeof(T), f);
    };
    auto fetch = [&](uint32_t u, uint64_t at) {
        if (KEEP) load16(p + at * sizeof(T), w[u]);
        else load16_stream(p + at * sizeof(T), w[u]);
    };
    for (; i + (kClipLoads - 1) * STEP < body; i += kClipLoads * STEP) {
        for (uint32_t u = 0; u < kClipLoads; ++u) fetch(u, i + u * STEP);
        for (uint32_t u = 0; u < kClipLoads; ++u) scale(i + u * STEP, w[u]);
    }
    for (; i < body; i += STEP) {
        fetch(0, i);
        scale(i, w[0]);
    }
    if (threadIdx.x < sp.edges) {
        uint8_t *const q = p + sp.edge(threadIdx.x) * sizeof(T);
        Lane<T>::put(q, Lane<T>::get(q) * c);
    }
}

// c g, rounded once; a factor of 1 leaves the gradients as they are, and the pass ends before its first read.  7.6e9 bf16
// gradients in 4.87 ms, 6.2 TB/s; 26.6e6 fp32 gradients (213 MB read and written) 33 us, 41e6 bf16 ones at odd addresses
// 27 us.
template <typename T, bool KEEP>
__global__ __launch_bounds__(256) void k_clip(NormList l, const float *norm, float max_norm, uint32_t shares) {
    const float f = clip_factor(*norm, max_norm);
    if (f == 1.0f) return;
    for (uint32_t i = blockIdx.x; i < shares; i += gridDim.x)
        for_share<kNormTensors>(l, i, shares, [&](uint32_t t, uint64_t lo, uint64_t hi) {
            scale_range<T, KEEP>(static_cast<uint8_t *>(l.p[t]), lo, hi, f);
        });
}

// One element's step.  The weight is the new master rounded once more, so the master is rounded first.  The decay's
// factor is held in 64 bits and joins the update before the one rounding: in 32 bits 1 - lr * weight_decay is 1 where the
// product is under 3e-8 (a rate of 1e-6 with a decay of 0.01), and every master would miss its decay alike.  It costs
// nothing next to the memory: 1.5e9 weights with their norm 7770-7790 us, and 7750-7760 with the 32-bit factor on that card.
__device__ __forceinline__ void adam_one(const AdamArgs &a, float g, float &w, float &m, float &v) {
    m = a.beta1 * m + a.one_less_beta1 * g;
    v = a.beta2 * v + a.one_less_beta2 * (g * g);
    w = rounded((float)fma((double)w, a.keep, -(double)(a.rate * m / (sqrtf(v) * a.root + a.eps))));
}

// Four elements of a type in one access, so that a wavefront's accesses to every array are contiguous (with eight
// elements a thread, two accesses to each 32 bytes of the float arrays, a step of 1.5e9 weights took 10.8 ms).
template <typename T>
__device__ __forceinline__ void load4(const void *p, uint64_t i, uint32_t *w) {
    const uint8_t *const q = static_cast<const uint8_t *>(p) + i * sizeof(T);
    if (sizeof(T) == 4) load16_stream(q, w);
    else load8_stream(q, w);
}
template <typename T>
__device__ __forceinline__ void unpack4(const uint32_t *w, float *f) {
    Lane<T>::template unpack<sizeof(T)>(w, f);
}
template <typename T>
__device__ __forceinline__ void store4(void *p, uint64_t i, const float *f) {
    uint8_t *const q = static_cast<uint8_t *>(p) + i * sizeof(T);
    uint32_t w[4];
    Lane<T>::template pack<sizeof(T)>(f, w);
    if (sizeof(T) == 4) store16_stream(q, w);
    else store8_stream(q, w);
}

// elements in flight per thread: so many times four of four arrays (in loops that are unrolled: rolled, with the loaded
// registers copied about, 1.5e9 weights took 8350 us instead of 7770)
constexpr uint32_t kAdamLoads = 2;

template <typename W, typename G>
__device__ __forceinline__ void adam_range(const AdamList &l, const AdamArgs &a, uint32_t t, uint64_t lo, uint64_t hi, float c) {
    float *const master = l.master[t], *const em = l.m[t], *const ev = l.v[t];
    // the vectors begin at the masters' 16-byte boundaries; the other arrays of a flat state share them
    const Span<float> sp(reinterpret_cast<const uint8_t *>(master), lo, hi);
    const uint64_t body = sp.first + sp.vectors * 4;
    uint32_t rg[kAdamLoads][4], rw[kAdamLoads][4], rm[kAdamLoads][4], rv[kAdamLoads][4];
    auto fetch = [&](uint32_t u, uint64_t i) {
        load4<G>(l.g[t], i, rg[u]);
        load4<float>(master, i, rw[u]);
        load4<float>(em, i, rm[u]);
        load4<float>(ev, i, rv[u]);
    };
    auto step = [&](uint32_t u, uint64_t i) {
        float g[4], w[4], m[4], v[4];
        unpack4<G>(rg[u], g);
        unpack4<float>(rw[u], w);
        unpack4<float>(rm[u], m);
        unpack4<float>(rv[u], v);
        for (int k = 0; k < 4; ++k) adam_one(a, c * g[k], w[k], m[k], v[k]);
        store4<float>(master, i, w);
        store4<float>(em, i, m);
        store4<float>(ev, i, v);
        store4<W>(l.w[t], i, w);
    };
    uint64_t i = sp.first + threadIdx.x * 4;
    for (; i + (kAdamLoads - 1) * 1024 < body; i += kAdamLoads * 1024) {
#pragma unroll
        for (uint32_t u = 0; u < kAdamLoads; ++u) fetch(u, i + u * 1024);
#pragma unroll
        for (uint32_t u = 0; u < kAdamLoads; ++u) step(u, i + u * 1024);
    }
    for (; i < body; i += 1024) {
        fetch(0, i);
        step(0, i);
    }
    if (threadIdx.x < sp.edges) {
        const uint64_t e = sp.edge(threadIdx.x);
        float w = master[e], m = em[e], v = ev[e];
        adam_one(a, c * Lane<G>::get(static_cast<const uint8_t *>(l.g[t]) + e * sizeof(G)), w, m, v);
        master[e] = w;
        em[e] = m;
        ev[e] = v;
        Lane<W>::put(static_cast<uint8_t *>(l.w[t]) + e * sizeof(W), w);
    }
}

// Reads 14 bytes an element (bf16 gradients) and writes 14: 1.5e9 weights (43.2 GB) in 24 launches of together 6.84 ms,
// 6.3 TB/s, over the rate of a copy.  Small shares (2048 elements a workgroup, two rounds of its threads) keep every CU
// supplied to the end: with the norm 7.58 ms, 7.69 with shares of 4096, 7.80 of 8192, 8.29 of 32768.
template <typename W, typename G>
__global__ __launch_bounds__(256) void k_adamw(AdamList l, AdamArgs a) {
    const float f = a.norm ? clip_factor(*a.norm, a.max_norm) : 1.0f;
    for_share<kAdamTensors>(l, blockIdx.x, gridDim.x, [&](uint32_t t, uint64_t lo, uint64_t hi) { adam_range<W, G>(l, a, t, lo, hi, f); });
}

}  // namespace

// ================================================================== launchers
#define CRX_STEP_LAUNCH(name, kernel, grid, block, stream, ...)                              \
    do {                                                                                     \
        timing_begin(name, stream);                                                          \
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(block), 0, stream, __VA_ARGS__);         \
        timing_end(name, stream);                                                            \
    } while (0)

// A launch has fewer than 2^32 threads: more rows than that take several.
uint32_t most_blocks(uint32_t block) { return 0xFFFFFFFFu / block; }
#define CRX_ROWS_LAUNCH(name, kernel, block, stream, rows_in, ...)                               \
    do {                                                                                         \
        RowsIn part_ = rows_in;                                                                  \
        for (uint64_t r_ = 0; r_ < part_.rows; r_ += most_blocks(block)) {                       \
            part_.row0 = (uint32_t)r_;                                                           \
            CRX_STEP_LAUNCH(name, kernel, std::min(part_.rows - part_.row0, most_blocks(block)), \
                            block, stream, part_, __VA_ARGS__);                                  \
        }                                                                                        \
    } while (0)

void launch_mask_counts(const RowsIn &x, uint32_t *counts, hipStream_t s) {
    if (x.rows <= kFewPositions && x.seqs <= kFewSeqs) {
        CRX_STEP_LAUNCH("mask_counts", k_mask_few, 1, 1024, s, x.mask, x.seqs, x.tokens, counts);
        return;
    }
    CRX_STEP_LAUNCH("mask_zero", k_mask_zero, std::min((x.seqs + 1023) / 1024, 4096u), 1024, s, counts, x.seqs);
    CRX_STEP_LAUNCH("mask_counts", k_mask_counts, (x.rows + 4 * kMaskRun - 1) / (4 * kMaskRun), 256, s, x.mask, x.rows, x.tokens, counts);
    CRX_STEP_LAUNCH("mask_total", k_mask_total, 1, 1024, s, counts, x.seqs);
}

namespace {
// A workgroup per row: of one wavefront, of 256 threads or of 1024, by the row's bytes.  A short row leaves a large
// workgroup's threads without a vector each; of long rows more workgroups hold more at once than the last-level cache
// keeps for the loss's second pass.  Loss and gradient of 16000 rows of bf16, us with 64 / 256 / 1024 threads: 500 logits
// 23 / 45 / 141, 4096: 56 / 63 / 153, 8192: 110 / 96 / 192, 32768: 459 / 390 / 411, 65536: 1034 / 835 / 749.  Scores: 500:
// 9 / 21 / 78, 8192: 43 / 45 / 104, 65536: 314 / 302 / 308; 4000 rows of 152064: - / 182 / 175.  (At 256 to some 2000 rows,
// where larger workgroups would fill the CUs better, the rule has not been measured.)
constexpr uint64_t kWaveBytes = 8192, kScoreShort = 131072, kPolicyShort = 65536;

template <typename T>
uint64_t row_bytes(const RowsIn &x) {
    return (uint64_t)x.vocab * sizeof(T);
}

template <typename T, bool ENT>
void score(const RowsIn &x, const Parts &p, const ScoreOut &o, hipStream_t s) {
    if (p.n > 1) {
        CRX_STEP_LAUNCH("part_stat", (k_part_stat<T, ENT>), x.rows * p.n, kPartBlock, s, x, p);
        CRX_STEP_LAUNCH("score_parts", (k_score_parts<T, ENT>), x.rows, 64, s, x, p, o);
    } else if (row_bytes<T>(x) <= kWaveBytes) {
        CRX_ROWS_LAUNCH("score", (k_score<T, 64, ENT>), 64, s, x, o);
    } else if (row_bytes<T>(x) <= kScoreShort) {
        CRX_ROWS_LAUNCH("score", (k_score<T, 256, ENT>), 256, s, x, o);
    } else {
        CRX_ROWS_LAUNCH("score", (k_score<T, 1024, ENT>), 1024, s, x, o);
    }
}
// The gradient's rows have no sums to join: they are cut whatever their number, up to the most workgroups of a launch.
Parts grad_parts(uint64_t rows, uint64_t vocab) {
    Parts p{nullptr, 1, (uint32_t)vocab};
    p.n = (uint32_t)((vocab + kGradPart - 1) / kGradPart);
    if (rows * p.n >= (1ULL << 31)) p.n = 1;
    p.size = ((uint32_t)((vocab + p.n - 1) / p.n) + 7) / 8 * 8;
    p.n = (uint32_t)((vocab + p.size - 1) / p.size);
    return p;
}

template <typename T, bool ENT>
void rows_grad(const RowsIn &x, const GradIn &g, hipStream_t s) {
    const Parts p = grad_parts(x.rows, x.vocab);
    // usually nothing is left to do (a loss's own gradient is 1): then the launch's workgroups are what it costs
    const uint32_t blocks = std::min(x.rows * p.n, g.unless_one ? kIdleBlocks : most_blocks(kPartBlock));
    CRX_STEP_LAUNCH("rows_grad", (k_rows_grad<T, kPartBlock, ENT>), blocks, kPartBlock, s, x, p, g);
}
template <typename T>
void policy(const RowsIn &x, const Parts &parts, const PolicyIn &p, const PolicyOut &o, hipStream_t s) {
    if (parts.n > 1) {
        CRX_STEP_LAUNCH("part_stat", (k_part_stat<T, false>), x.rows * parts.n + (parts.counts != nullptr), kPartBlock, s, x, parts);
        CRX_STEP_LAUNCH("policy_parts", (k_policy_parts<T>), x.rows * parts.n, kPartBlock, s, x, parts, p, o);
    } else if (row_bytes<T>(x) <= kWaveBytes) {
        CRX_ROWS_LAUNCH("policy", (k_policy<T, 64, kHeld>), 64, s, x, p, o);
    } else if (row_bytes<T>(x) <= kPolicyShort) {
        CRX_ROWS_LAUNCH("policy", (k_policy<T, 256, kHeld>), 256, s, x, p, o);
    } else if (row_bytes<T>(x) <= kAloneBytes) {
        CRX_ROWS_LAUNCH("policy", (k_policy<T, 1024, kHeld>), 1024, s, x, p, o);
    } else {
        CRX_ROWS_LAUNCH("policy", (k_policy<T, 1024, kHeldAlone>), 1024, s, x, p, o);
    }
}
}  // namespace

Parts parts_of(uint64_t rows, uint64_t vocab) {
    Parts p{nullptr, 1, (uint32_t)vocab};
    if (!rows || rows >= kPartRows) return p;
    const uint64_t most = std::min<uint64_t>(kMostParts, (2 * kPartRows + rows - 1) / rows);
    const uint64_t size = std::max<uint64_t>(kPartLeast, (vocab + most - 1) / most);
    p.size = (uint32_t)((size + 7) / 8 * 8);
    p.n = (uint32_t)((vocab + p.size - 1) / p.size);
    return p;
}

void launch_score(const RowsIn &x, const Parts &p, const ScoreOut &o, int dtype, hipStream_t s) {
    if (dtype == kBf16) o.entropy ? score<Bf16, true>(x, p, o, s) : score<Bf16, false>(x, p, o, s);
    else if (dtype == kF16) o.entropy ? score<F16, true>(x, p, o, s) : score<F16, false>(x, p, o, s);
    else o.entropy ? score<float, true>(x, p, o, s) : score<float, false>(x, p, o, s);
}

void launch_policy(const RowsIn &x, const Parts &parts, const PolicyIn &p, const PolicyOut &o, int dtype, hipStream_t s) {
    if (dtype == kBf16) policy<Bf16>(x, parts, p, o, s);
    else if (dtype == kF16) policy<F16>(x, parts, p, o, s);
    else policy<float>(x, parts, p, o, s);
}

void launch_policy_sums(const float *terms, uint32_t rows, float scale, float *loss, float *kl, float *clipped,
                        hipStream_t s) {
    CRX_STEP_LAUNCH("policy_sums", k_policy_sums, 3, 1024, s, terms, rows, scale, loss, kl, clipped);
}

void launch_rows_grad(const RowsIn &x, const GradIn &g, int dtype, hipStream_t s) {
    const bool ent = g.up_entropy.p != nullptr;
    if (dtype == kBf16) ent ? rows_grad<Bf16, true>(x, g, s) : rows_grad<Bf16, false>(x, g, s);
    else if (dtype == kF16) ent ? rows_grad<F16, true>(x, g, s) : rows_grad<F16, false>(x, g, s);
    else ent ? rows_grad<float, true>(x, g, s) : rows_grad<float, false>(x, g, s);
}

namespace {
template <typename T>
void norm_part(const NormList &l, double *partial, uint32_t used, bool keep, uint32_t blocks, hipStream_t s) {
    if (keep) CRX_STEP_LAUNCH("norm_part", (k_norm_part<T, true>), blocks, 256, s, l, partial, used);
    else CRX_STEP_LAUNCH("norm_part", (k_norm_part<T, false>), blocks, 256, s, l, partial, used);
}
template <typename T>
void clip(const NormList &l, const float *norm, float max_norm, bool keep, uint32_t shares, hipStream_t s) {
    const uint32_t blocks = std::min(shares, kClipBlocks);
    if (keep) CRX_STEP_LAUNCH("clip", (k_clip<T, true>), blocks, 256, s, l, norm, max_norm, shares);
    else CRX_STEP_LAUNCH("clip", (k_clip<T, false>), blocks, 256, s, l, norm, max_norm, shares);
}
template <typename W>
void adamw(const AdamList &l, int gtype, const AdamArgs &a, uint32_t blocks, hipStream_t s) {
    if (gtype == kBf16) CRX_STEP_LAUNCH("adamw", (k_adamw<W, Bf16>), blocks, 256, s, l, a);
    else if (gtype == kF16) CRX_STEP_LAUNCH("adamw", (k_adamw<W, F16>), blocks, 256, s, l, a);
    else CRX_STEP_LAUNCH("adamw", (k_adamw<W, float>), blocks, 256, s, l, a);
}
}  // namespace

void launch_norm_part(const NormList &l, int dtype, double *partial, uint32_t used, bool keep, uint32_t blocks, hipStream_t s) {
    if (dtype == kBf16) norm_part<Bf16>(l, partial, used, keep, blocks, s);
    else if (dtype == kF16) norm_part<F16>(l, partial, used, keep, blocks, s);
    else norm_part<float>(l, partial, used, keep, blocks, s);
}
void launch_norm_sum(const double *partial, uint32_t n, float *norm, hipStream_t s) {
    CRX_STEP_LAUNCH("norm_sum", k_norm_sum, 1, 1024, s, partial, n, norm);
}
void launch_clip(const NormList &l, int dtype, const float *norm, float max_norm, bool keep, uint32_t shares, hipStream_t s) {
    if (dtype == kBf16) clip<Bf16>(l, norm, max_norm, keep, shares, s);
    else if (dtype == kF16) clip<F16>(l, norm, max_norm, keep, shares, s);
    else clip<float>(l, norm, max_norm, keep, shares, s);
}
void launch_adamw(const AdamList &l, int wtype, int gtype, const AdamArgs &a, uint32_t blocks, hipStream_t s) {
    if (wtype == kBf16) adamw<Bf16>(l, gtype, a, blocks, s);
    else if (wtype == kF16) adamw<F16>(l, gtype, a, blocks, s);
    else adamw<float>(l, gtype, a, blocks, s);
}

}  // namespace crx
