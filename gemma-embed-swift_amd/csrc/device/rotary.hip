// Norms and rotary positions of query and key heads, rows to rows or keys and values to their pages (gfx950).
//   y = x / sqrt(mean(x^2) + eps) w over a head (where normed), then for each pair (a, b) of its first 2 `half`
//   elements, at angle t = 2 pi position turns[i]:  (a cos t - b sin t, a sin t + b cos t) magnitude.
//
// One pass: a group of lanes holds a head from its load to its store, in fp32, and rounds once. The angle is
// reduced in fp64 (a position of 2^31 keeps 2^-22 of a turn) and its sine and cosine taken in fp32, each once a row
// for all heads: the wave's lanes take a pair each and share them through LDS.
//
// What bounds it: the bytes of long calls (16384 rows of 32 + 8 heads of 128, 16-bit: 67 us, 5.0 TB/s, what a copy reaches; 8192 tokens
// of 32 + 8 + 8 normed and appended: 47 us, 4.3 TB/s, a third of them to pages), the chain of one load, one reduction and one
// store in short ones (one token of 3 + 1 heads: 4 us).
#include "common.hpp"
#include "half_types.hpp"
#include "rotary.hpp"

namespace ge {
namespace {

struct F32 {
    static __device__ __forceinline__ float value(float x) { return x; }
};

template <typename T>
struct StoredAs {
    typedef uint16_t Type;
};
template <>
struct StoredAs<F32> {
    typedef float Type;
};

// The pieces of a head that a lane holds: N elements of `a` and as many of `b`, the pairs' two sides where
// they turn. UNIT: elements that lie together.
// 8, 4, 2: one unit of each a lane, loaded and stored whole, head_dim / (2 UNIT) lanes a head (a power of two of
// lanes, so that several heads stand side by side in a wave). 1, for whatever does not come in larger ones: four of
// each a lane, head_dim / 8 lanes. 16384 rows of 32 + 8 heads of 128 of which 128, 72, 36 and 34 elements turn: 66, 76, 110
// and 118 us (a whole wave to a head in units of 1: 185).
template <int UNIT>
struct Shape {
    static constexpr int N = UNIT == 1 ? 4 : UNIT, kUnits = N / UNIT;
};

// log2 of the lanes a head takes.
template <int UNIT>
__device__ __forceinline__ int lanes_log(int head_dim) {
    const int lanes = (head_dim / 2 + Shape<UNIT>::N - 1) / Shape<UNIT>::N;
    return lanes <= 1 ? 0 : 32 - __builtin_clz(uint32_t(lanes - 1));
}

// The sum over groups of 2^log lanes: halves of a group hold equal sums, so that a mirrored move is as
// good as the exchange.
__device__ __forceinline__ float group_sum(float v, int log) {
    if (log >= 1) v += dpp_move<0xb1>(v);   // quad_perm 1, 0, 3, 2
    if (log >= 2) v += dpp_move<0x4e>(v);   // quad_perm 2, 3, 0, 1
    if (log >= 3) v += dpp_move<0x141>(v);  // row_half_mirror
    if (log >= 4) v += dpp_move<0x140>(v);  // row_mirror
    if (log >= 5) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (log >= 6) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}

// Where a lane's units lie in a head: their first elements, -1 past the head's end (b likewise), and first pairs, -1
// where they do not turn.
template <int UNIT>
struct Place {
    static constexpr int U = Shape<UNIT>::kUnits;
    int a[U], b[U], pair[U];
    bool any;  // a unit lies in the head

    __device__ __forceinline__ void init(const HeadsArgs& h, int lane_of_head, int lanes) {
        any = false;
#pragma unroll
        for (int j = 0; j < U; j++) {
            const int u = (lane_of_head + lanes * j) * UNIT;  // the unit's first pair
            const bool in = u < h.head_dim / 2, turns = u < h.half;
            any = any || in;
            pair[j] = in && turns ? u : -1;
            a[j] = !in ? -1 : turns && !h.pairs ? u : 2 * u;
            b[j] = !in ? -1 : turns && !h.pairs ? h.half + u : 2 * u + UNIT;
        }
    }
};

// N elements as they lie in memory. (Vectors and single members: arrays that are loaded under a condition went
// through scratch memory.)
template <typename T, int N>
struct Elements {
    typedef uint32_t Words __attribute__((ext_vector_type(N / 2)));
    Words w{};
    __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const Words*>(p); }
    __device__ __forceinline__ void values(float (&x)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = T::value(uint16_t(w[i / 2] >> (16 * (i % 2))));
    }
};
template <typename T>
struct Elements<T, 2> {
    uint32_t w = 0;
    __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const uint32_t*>(p); }
    __device__ __forceinline__ void values(float (&x)[2]) const {
        x[0] = T::value(uint16_t(w));
        x[1] = T::value(uint16_t(w >> 16));
    }
};
template <int N>
struct Elements<F32, N> {
    typedef float Words __attribute__((ext_vector_type(N < 4 ? N : 4)));
    Words w{}, more{};  // more: of 8
    __device__ __forceinline__ void load(const float* p) {
        w = *reinterpret_cast<const Words*>(p);
        if constexpr (N == 8) more = *reinterpret_cast<const Words*>(p + 4);
    }
    __device__ __forceinline__ void values(float (&x)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = i < 4 ? w[i] : more[i - 4];
    }
};
template <>
struct Elements<F32, 2> {
    typedef float Words __attribute__((ext_vector_type(2)));
    Words w{};
    __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const Words*>(p); }
    __device__ __forceinline__ void values(float (&x)[2]) const {
        x[0] = w[0];
        x[1] = w[1];
    }
};

// A lane's elements of one head, loaded ahead.
template <typename T, int UNIT>
struct Raw {
    Elements<T, UNIT> a, b;
    __device__ __forceinline__ void load(const typename StoredAs<T>::Type* p, const Place<UNIT>& at) {
        a.load(p + at.a[0]);
        b.load(p + at.b[0]);
    }
    __device__ __forceinline__ void values(float (&x)[UNIT], float (&y)[UNIT]) const {
        a.values(x);
        b.values(y);
    }
};
template <typename T>
struct Raw<T, 1> {
    float4_t a{}, b{};
    __device__ __forceinline__ void load(const typename StoredAs<T>::Type* p, const Place<1>& at) {
#pragma unroll
        for (int j = 0; j < 4; j++) {  // a unit past the head's end takes the head's first element, and is not used
            a[j] = T::value(p[max(at.a[j], 0)]);
            b[j] = T::value(p[max(at.b[j], 0)]);
            if (at.a[j] < 0) a[j] = b[j] = 0.0f;
        }
    }
    __device__ __forceinline__ void values(float (&x)[4], float (&y)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[j] = a[j];
            y[j] = b[j];
        }
    }
};

// A lane's weights, from the LDS row of its head's kind.
template <int UNIT>
__device__ __forceinline__ void weigh(const float* w, const Place<UNIT>& at, float (&a)[Shape<UNIT>::N], float (&b)[Shape<UNIT>::N]) {
    constexpr int V = UNIT < 4 ? UNIT : 4;
    typedef float Vector __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int j = 0; j < Shape<UNIT>::N; j += V) {
        const int unit = j / UNIT, within = j % UNIT;
        const Vector x = *reinterpret_cast<const Vector*>(w + max(at.a[unit], 0) + within), y = *reinterpret_cast<const Vector*>(w + max(at.b[unit], 0) + within);
#pragma unroll
        for (int i = 0; i < V; i++) {
            a[j + i] *= x[i];
            b[j + i] *= y[i];
        }
    }
}

template <typename O, int UNIT>
__device__ __forceinline__ void store(uint16_t* p, const Place<UNIT>& at, const float (&a)[Shape<UNIT>::N], const float (&b)[Shape<UNIT>::N]) {
    if constexpr (UNIT == 8) {
        *reinterpret_cast<u32x4*>(p + at.a[0]) = u32x4{O::pack(a[0], a[1]), O::pack(a[2], a[3]), O::pack(a[4], a[5]), O::pack(a[6], a[7])};
        *reinterpret_cast<u32x4*>(p + at.b[0]) = u32x4{O::pack(b[0], b[1]), O::pack(b[2], b[3]), O::pack(b[4], b[5]), O::pack(b[6], b[7])};
    } else if constexpr (UNIT == 4) {
        *reinterpret_cast<u32x2*>(p + at.a[0]) = u32x2{O::pack(a[0], a[1]), O::pack(a[2], a[3])};
        *reinterpret_cast<u32x2*>(p + at.b[0]) = u32x2{O::pack(b[0], b[1]), O::pack(b[2], b[3])};
    } else if constexpr (UNIT == 2) {
        *reinterpret_cast<uint32_t*>(p + at.a[0]) = O::pack(a[0], a[1]);
        *reinterpret_cast<uint32_t*>(p + at.b[0]) = O::pack(b[0], b[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (at.a[j] >= 0) {
                p[at.a[j]] = uint16_t(O::pack(a[j], 0.0f));
                p[at.b[j]] = uint16_t(O::pack(b[j], 0.0f));
            }
    }
}

// x / sqrt(mean(x^2) + eps). Squares that leave fp32's range, or get lost below it where eps does not
// outweigh them, are taken of x times a power of two: 2^90 brings the smallest element's square over 512 to 2^-127, which has
// 22 bits, and a sum below 2^-60 to 2^120.
template <int N>
__device__ __forceinline__ void norm(float (&a)[N], float (&b)[N], bool on, int log, float inv_dim, float eps) {
    auto squares = [&] {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) ss = __builtin_fmaf(a[i], a[i], __builtin_fmaf(b[i], b[i], ss));
        return group_sum(ss, log);
    };
    float ss = squares(), e = eps;
    const bool large = on && !(ss <= 1e37f), small = on && ss < 0x1p-60f && eps < 0x1p-100f;
    if (__builtin_amdgcn_ballot_w64(large || small)) {
        const float f = large ? 0x1p-100f : small ? 0x1p90f : 1.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            a[i] *= f;
            b[i] *= f;
        }
        e = eps * f * f;
        ss = squares();
    }
    const float r = on ? 1.0f / sqrtf(__builtin_fmaf(ss, inv_dim, e)) : 1.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        a[i] *= r;
        b[i] *= r;
    }
}

// The pairs (a, b) by their angles; gain: 1 but for magnitudes past 1.
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
    const float x = a;
    a = __builtin_fmaf(x, c, -(b * s));
    b = __builtin_fmaf(x, s, b * c);
}

// I: the input type; O: the results'. A workgroup has up to rows_each rows. A wave takes a row, or, where there are
// fewer rows than waves, a part of its heads, kIts groups of heads at a time, which with four workgroups a CU is what
// the registers hold. 8192 tokens of 32 + 8 + 8 heads of 128 to append, 16-bit: four groups at half the waves 59 us, two 47,
// one 48 (at five workgroups 49, at six, which spill, 103); fp32: two at three workgroups 64 us, one at four 62 (5000
// tokens of 5 heads of 256: 16.6 and 15.3). Smaller units have registers for more, which with few heads stay empty: four
// groups of units of 4 16384 rows of 5 + 1 heads of 72 in 16.0 us, two in 13.6. The norms' weights are in LDS, a row for each kind of head: in
// registers, picked by each lane's kind, they took 10% of that time.
template <typename I, typename O, int UNIT, bool APPEND>
__device__ __forceinline__ void heads_body(const HeadsArgs& h, const AppendItem& it) {
    typedef typename StoredAs<I>::Type Stored;
    constexpr int N = Shape<UNIT>::N, kIts = UNIT * sizeof(Stored) == 32 ? 1 : 2, kMaxDim = 512;
    __shared__ float2 angles[UNIT > 1 ? 4 * kMaxDim / 2 : 1];
    __shared__ __attribute__((aligned(16))) float weights[3][kMaxDim];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int log = lanes_log<UNIT>(h.head_dim), at_once = 64 >> log;
    const int all = h.heads + (APPEND ? 2 : 1) * h.kv_heads;
    const int groups = (all + at_once - 1) / at_once, chunks = (groups + kIts - 1) / kIts;
    Place<UNIT> at;
    at.init(h, lane & ((1 << log) - 1), 1 << log);
    const float inv_dim = 1.0f / float(h.head_dim);
    float2* const mine = angles + (UNIT > 1 ? wave * (kMaxDim / 2) : 0);
    // a head's kind: 0 q, 1 k, 2 v; its number among them
    auto kind_of = [&](int head) { return head < h.heads ? 0 : head < h.heads + h.kv_heads ? 1 : 2; };
    auto number_of = [&](int head, int kind) { return kind == 0 ? head : kind == 1 ? head - h.heads : head - h.heads - h.kv_heads; };
    auto load = [&](Raw<I, UNIT>& raw, int r, int group) {
        const int head = group * at_once + (lane >> log), kind = kind_of(head);
        if (group < groups && head < all && at.any) {
            const void* const base = kind == 0 ? h.q : kind == 1 ? h.k : h.v;
            const int64_t stride = kind == 0 ? h.q_stride : kind == 1 ? h.k_stride : h.v_stride;
            raw.load(static_cast<const Stored*>(base) + (size_t(it.row0) + uint32_t(r)) * size_t(stride) + size_t(number_of(head, kind)) * size_t(h.head_dim), at);
        } else {
            raw = Raw<I, UNIT>{};
        }
    };
    // A wave's steps: chunks [chunk0, chunk1) of its rows r, r + stride, ..., each loaded a step ahead.
    const bool split = int(it.n) < 4;  // parts of a row
    const int chunk0 = split ? wave / int(it.n) : 0, step = split ? (4 + int(it.n) - 1 - wave % int(it.n)) / int(it.n) : 1;
    const int stride = split ? int(it.n) : 4;
    int r = split ? wave % int(it.n) : wave, chunk = chunk0;
    if (chunk >= chunks) r = int(it.n);
    Raw<I, UNIT> raw[kIts];
    if (r < int(it.n)) {
#pragma unroll
        for (int i = 0; i < kIts; i++) load(raw[i], r, chunk * kIts + i);
    }
    if (h.normed) {
        for (int i = threadIdx.x; i < h.head_dim; i += 256) {
            weights[0][i] = h.normed & kNormQ && h.q_norm ? h.q_norm[i] : 1.0f;
            weights[1][i] = h.normed & kNormK && h.k_norm ? h.k_norm[i] : 1.0f;
            weights[2][i] = 1.0f;
        }
        __syncthreads();
    }

    float cs[N], sn[N];
    size_t page_at = 0;  // of the row, in its page's first head
    while (r < int(it.n)) {
        const size_t row = size_t(it.row0) + uint32_t(r);
        if (chunk == chunk0) {
            if constexpr (APPEND) {
                const uint32_t key = it.first + uint32_t(r);
                const int page = __builtin_amdgcn_readfirstlane(h.table[size_t(it.slot) * size_t(h.slot_pages) + (key >> h.page_shift)]);
                page_at = size_t(page) * size_t(h.page_stride) + size_t(key & ((1u << h.page_shift) - 1)) * size_t(h.head_dim);
            }
            if (h.half) {
                const double position = h.positions ? double(h.positions[row]) : double(it.first + uint32_t(r));
                auto turn = [&](int pair, float& c, float& s) {
                    const double t = position * h.turns[pair];
                    sincospif(2.0f * float(t - rint(t)), &s, &c);
                    c *= h.fade;
                    s *= h.fade;
                };
                if constexpr (UNIT > 1) {
                    for (int pair = lane; pair < h.half; pair += 64) {
                        float c, s;
                        turn(pair, c, s);
                        mine[pair] = float2{c, s};
                    }
                    // (a wave's own LDS operations are in order: only the compiler has to keep it)
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    const int first = at.pair[0] < 0 ? 0 : at.pair[0];
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const float2 x = mine[first + i];
                        cs[i] = x.x;
                        sn[i] = x.y;
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                } else {
#pragma unroll
                    for (int j = 0; j < N; j++) turn(at.pair[j] < 0 ? 0 : at.pair[j], cs[j], sn[j]);
                }
            }
        }
        const bool last = chunk + step >= chunks;
        const int r_next = last ? r + stride : r, chunk_next = last ? chunk0 : chunk + step;
#pragma unroll
        for (int i = 0; i < kIts; i++) {
            const int group = chunk * kIts + i, head = group * at_once + (lane >> log), kind = kind_of(head);
            const bool here = group < groups && head < all;
            float a[N], b[N];
            raw[i].values(a, b);
            if (r_next < int(it.n)) load(raw[i], r_next, chunk_next * kIts + i);
            if (h.normed) {
                norm(a, b, here && (h.normed >> kind & 1), log, inv_dim, h.eps);
                if (here && at.any) weigh<UNIT>(weights[kind], at, a, b);
            }
            if (!here || !at.any) continue;
            if (h.half && kind < 2) {
                if constexpr (UNIT > 1) {
                    if (at.pair[0] >= 0) {
                        if (h.pairs) {  // neighbours: pairs i of a and N / 2 + i of b
#pragma unroll
                            for (int j = 0; j < N; j += 2) {
                                turn_pair(a[j], a[j + 1], cs[j / 2], sn[j / 2]);
                                turn_pair(b[j], b[j + 1], cs[N / 2 + j / 2], sn[N / 2 + j / 2]);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < N; j++) turn_pair(a[j], b[j], cs[j], sn[j]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < N; j++)
                        if (at.pair[j] >= 0) turn_pair(a[j], b[j], cs[j], sn[j]);
                }
                if (h.gain != 1.0f) {
#pragma unroll
                    for (int j = 0; j < N; j++)
                        if (at.pair[UNIT > 1 ? 0 : j] >= 0) {
                            a[j] *= h.gain;
                            b[j] *= h.gain;
                        }
                }
            }
            const size_t number = size_t(number_of(head, kind));
            uint16_t* p;
            if (kind == 0)
                p = h.q_out + row * size_t(h.q_out_stride) + number * size_t(h.head_dim);
            else if constexpr (APPEND)
                p = (kind == 1 ? h.k_out : h.v_out) + page_at + (number << h.page_shift) * size_t(h.head_dim);
            else
                p = h.k_out + row * size_t(h.k_out_stride) + number * size_t(h.head_dim);
            store<O, UNIT>(p, at, a, b);
        }
        r = r_next;
        chunk = chunk_next;
    }
}

template <typename I, typename O, int UNIT>
__global__ __launch_bounds__(256, 4) void rotate_heads_kernel(const HeadsArgs h) {
    const int row0 = int(blockIdx.x) * h.rows_each;
    const AppendItem it{uint32_t(row0), uint32_t(min(h.rows_each, h.rows - row0)), 0, 0, 0};
    heads_body<I, O, UNIT, false>(h, it);
}

template <typename I, typename O, int UNIT>
__global__ __launch_bounds__(256, 4) void append_kernel(const HeadsArgs h, const AppendInline in) {
    auto scalar = [](uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); };
    AppendItem it;
    if (h.items) {
        const AppendItem* const p = h.items + blockIdx.x;
        it = AppendItem{scalar(p->row0), scalar(p->n), scalar(p->slot), scalar(p->first), blockIdx.x};
    } else {
        // the last item that begins at or before this workgroup
        const bool each = h.workgroups == h.n_items;
        int at = each ? int(blockIdx.x) : 0;
        for (int n = each ? 1 : h.n_items; n > 1;) {
            const int half = n / 2;
            if (in.items[at + half].group0 <= blockIdx.x) {
                at += half;
                n -= half;
            } else {
                n = half;
            }
        }
        const uint32_t skip = (blockIdx.x - in.items[at].group0) * uint32_t(h.rows_each);
        it = AppendItem{in.items[at].row0 + skip, min(in.items[at].n - skip, uint32_t(h.rows_each)), in.items[at].slot, in.items[at].first + skip, blockIdx.x};
    }
    heads_body<I, O, UNIT, true>(h, it);
}

__global__ __launch_bounds__(256) void table_set_kernel(int32_t* table, const uint2* entries, int n) {
    const int i = int(blockIdx.x) * 256 + int(threadIdx.x);
    if (i < n) table[entries[i].x] = int32_t(entries[i].y);
}

bool heads_ok(const HeadsArgs& a) {
    return a.heads >= 0 && a.kv_heads >= 0 && a.heads + a.kv_heads > 0 && a.head_dim > 0 && a.head_dim <= 512 && a.head_dim % 2 == 0 &&
           a.half >= 0 && a.half <= a.head_dim / 2 && a.rows >= 0;
}

template <typename I, typename O, int UNIT>
hipError_t run_rotate(hipStream_t s, const HeadsArgs& a) {
    launch_kernel(rotate_heads_kernel<I, O, UNIT>, dim3(uint32_t((int64_t(a.rows) + a.rows_each - 1) / a.rows_each)), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <typename I, typename O>
hipError_t run_rotate(hipStream_t s, const HeadsArgs& a, int unit) {
    switch (unit) {
        case 8: return run_rotate<I, O, 8>(s, a);
        case 4: return run_rotate<I, O, 4>(s, a);
        case 2: return run_rotate<I, O, 2>(s, a);
        default: return run_rotate<I, O, 1>(s, a);
    }
}

template <typename I, typename O, int UNIT>
hipError_t run_append(hipStream_t s, const HeadsArgs& a, const AppendInline& in) {
    launch_kernel(append_kernel<I, O, UNIT>, dim3(uint32_t(a.workgroups)), dim3(256), 0, s, a, in);
    return hipGetLastError();
}

template <typename I, typename O>
hipError_t run_append(hipStream_t s, const HeadsArgs& a, const AppendInline& in, int unit) {
    switch (unit) {
        case 8: return run_append<I, O, 8>(s, a, in);
        case 4: return run_append<I, O, 4>(s, a, in);
        case 2: return run_append<I, O, 2>(s, a, in);
        default: return run_append<I, O, 1>(s, a, in);
    }
}

}  // namespace

hipError_t launch_rotate_heads(hipStream_t s, const HeadsArgs& a, bool in_f32, bool bf16, int unit) {
    if (!heads_ok(a) || !heads_unit_ok(a.head_dim, a.half, unit) || a.rows_each <= 0 || (a.half && !a.positions)) return hipErrorInvalidValue;
    if (a.rows == 0) return hipSuccess;
    if (in_f32) return bf16 ? run_rotate<F32, BF16>(s, a, unit) : run_rotate<F32, F16>(s, a, unit);
    return bf16 ? run_rotate<BF16, BF16>(s, a, unit) : run_rotate<F16, F16>(s, a, unit);
}

hipError_t launch_append(hipStream_t s, const HeadsArgs& a, const AppendInline& in, bool in_f32, bool bf16, int unit) {
    if (!heads_ok(a) || !heads_unit_ok(a.head_dim, a.half, unit) || a.n_items < 0 || a.workgroups < a.n_items || uint64_t(a.workgroups) * 256 >> 32 || a.rows_each <= 0 ||
        (a.items ? a.workgroups != a.n_items : a.n_items > kAppendInlineItems))
        return hipErrorInvalidValue;
    if (a.n_items == 0) return hipSuccess;
    if (in_f32) return bf16 ? run_append<F32, BF16>(s, a, in, unit) : run_append<F32, F16>(s, a, in, unit);
    return bf16 ? run_append<BF16, BF16>(s, a, in, unit) : run_append<F16, F16>(s, a, in, unit);
}

hipError_t launch_table_set(hipStream_t s, int32_t* table, const uint2* entries, int n) {
    if (n <= 0) return n < 0 ? hipErrorInvalidValue : hipSuccess;
    launch_kernel(table_set_kernel, dim3(uint32_t((n + 255) / 256)), dim3(256), 0, s, table, entries, n);
    return hipGetLastError();
}

}  // namespace ge
