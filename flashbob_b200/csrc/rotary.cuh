// Rotary positions: y = m R(position * frequency) x over the first 2 * pairs elements of a head, the others unchanged.
//
// Pair i turns elements (i, i + pairs) or, interleaved, (2 i, 2 i + 1) by position * frequency_i.  The gradient is the
// same map with the angles negated, so one kernel serves forward and every order of backward.
//
// Angles: a frequency is kept as the 64-bit fraction of a turn per position.  position * fraction modulo 2^64 is then
// the angle modulo a turn in one integer product, off by 2^-64 turns per position (8e-10 radians at position 2^31), and a sine
// needs no range reduction; position * frequency in fp32 is off by 0.004 radians at position 100,000.
//
// What bounds it: one read and one write of every element.  A thread turns the same 16 elements (8 pairs) of HPT heads of
// a token, so its 8 sines and cosines are shared by them and their loads are in flight together.  They are the special-
// function unit's, off by 2^-21.4 and 2^-21.2, of an fp32 angle that is off by 4e-7: 8e-7 together, a six-hundredth of the
// result's rounding in fp16 (sincospif, with four times the instructions, took 31 us for 29.5 on 84 MB with one head a thread, 18 for 17.1 with four).  Measured now: 84 MB in 15.4 us, 5.4 TB/s.
#pragma once

#include "ptx.cuh"
#include "../../include/bob_sm100.h"

namespace bob {

// How a thread's 16 elements lie in a row.  kHalf: two 16-byte chunks, partners `pairs` elements apart (pairs a multiple of
// 8); kInterleaved: 16 elements in a row; kQuarter: as kHalf in four 8-byte pieces (pairs a multiple of 4); kScattered: the
// same for any number of pairs, element by element in shared memory (4 times as slow as the others: 103 us on 168 MB).
enum RotaryForm : int { kHalf = 0, kInterleaved = 1, kScattered = 2, kQuarter = 3 };

inline int rotary_form(const bob_sm100_rotary* r) {
    return r->interleaved ? kInterleaved : (r->pairs % 8 == 0 ? kHalf : (r->pairs % 4 == 0 ? kQuarter : kScattered));
}

__device__ __forceinline__ int64_t angle_of(int64_t position, uint64_t turn) {      // 2^-64 turns, in [-1/2, 1/2) turns
    return static_cast<int64_t>(static_cast<uint64_t>(position) * turn);
}
__device__ __forceinline__ void turn_factors(int64_t position, uint64_t turn, float& s, float& c) {
    // the upper 32 bits, 7e-10 radians; in fp32 and times 2 pi / 2^32 off by up to 4e-7
    const float x = static_cast<float>(static_cast<int32_t>(angle_of(position, turn) >> 32)) * 1.4629180792671596e-9f;      // 2 pi / 2^32
    s = __sinf(x);
    c = __cosf(x);
}

// Sine and cosine of a whole turn's 256 parts.
struct TurnTable { double2 at[256]; };
constexpr double sine_series(double x) {
    double term = x, sum = x;
    for (int k = 1; k < 14; ++k) { term *= -x * x / ((2 * k) * (2 * k + 1)); sum += term; }
    return sum;
}
constexpr double cosine_series(double x) {
    double term = 1, sum = 1;
    for (int k = 1; k < 14; ++k) { term *= -x * x / ((2 * k - 1) * (2 * k)); sum += term; }
    return sum;
}
constexpr TurnTable make_turn_table() {
    TurnTable t = {};
    for (int i = 0; i < 256; ++i) {
        const int octant = i / 32, j = i % 32;           // 45 degrees each: series of at most pi / 4
        const double x = 0.024543692606170259675489401 * (octant % 2 ? 32 - j : j);        // 2 pi / 256
        const double s = sine_series(x), c = cosine_series(x);
        const double ss[8] = {s, c, c, s, -s, -c, -c, -s}, cc[8] = {c, s, -s, -c, -c, -s, s, c};
        t.at[i].x = ss[octant];
        t.at[i].y = cc[octant];
    }
    return t;
}
__device__ const TurnTable kTurnTable = make_turn_table();

// In 64 bits: the part of a turn from the table, the rest (at most 2^-9 of a turn, x = 0.0123) by the series
// x - x^3/6 + x^5/120 and 1 - x^2/2 + x^4/24 - x^6/720, which end below 1e-17.
__device__ __forceinline__ void turn_factors(int64_t position, uint64_t turn, double& s, double& c) {
    const uint64_t a = static_cast<uint64_t>(angle_of(position, turn)) + (1ull << 55);      // to the nearest of 256
    const double2 t = kTurnTable.at[a >> 56];
    const double x = static_cast<double>(static_cast<int64_t>(a & ((1ull << 56) - 1)) - (1ll << 55)) * 3.4061215800210806e-19;     // 2 pi / 2^64
    const double x2 = x * x;
    const double sx = fma(x * x2, fma(x2, 1.0 / 120, -1.0 / 6), x), cx = fma(x2, fma(x2, fma(x2, -1.0 / 720, 1.0 / 24), -0.5), 1.0);
    s = fma(t.x, cx, t.y * sx);
    c = fma(t.y, cx, -(t.x * sx));
}

// Frequencies 2 i and 2 i + 1 of a rotation that is a kernel parameter, by its address: read as constants, which a warp takes
// one address at a time, the eight frequencies of every thread took most of the kernel's time (84 MB with one head a
// thread 29.5 us, with them as ordinary loads 21.1; with four heads a thread 17.1 and 15.4).
__device__ __forceinline__ ulonglong2 turn_pair(const bob_sm100_rotary& r, int i) {
    ulonglong2 x;
    asm("ld.v2.u64 {%0, %1}, [%2];" : "=l"(x.x), "=l"(x.y) : "l"(r.turns + 2 * i));
    return x;
}

// Two 16-byte chunks of a row, as they are loaded.
struct Chunks { uint4 a, b; };

// The place of thread `c` of a row (its pairs are 8 c ... 8 c + 7) for a row of D elements.
template <int FORM>
struct RowPlace {
    int first, second;            // elements of the two chunks (kHalf, kInterleaved)
    int c, pairs;
    __device__ __forceinline__ RowPlace(int c_, int pairs_) : c(c_), pairs(pairs_) {
        if (FORM == kHalf) {
            const bool turning = 8 * c < pairs;
            first = turning ? 8 * c : 16 * c;                // behind the turned elements: 2 pairs + 16 (c - pairs / 8)
            second = turning ? first + pairs : first + 8;
        } else {
            first = 16 * c;
            second = first + 8;
        }
    }
    // kScattered, kQuarter: the elements of pair 8 c + j
    __device__ __forceinline__ int element(int j, bool partner) const {
        const int i = 8 * c + j;
        if (FORM == kQuarter) return i < pairs ? i + (partner ? pairs : 0) : 2 * i + (partner ? 4 : 0);     // (j = 0 or 4)
        return i < pairs ? i + (partner ? pairs : 0) : 2 * i + (partner ? 1 : 0);
    }
    __device__ __forceinline__ Chunks load(const uint16_t* row) const {
        Chunks x;
        if constexpr (FORM == kScattered) {
            uint32_t w[8];
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = row[element(2 * j, false)] | static_cast<uint32_t>(row[element(2 * j + 1, false)]) << 16;
                w[4 + j] = row[element(2 * j, true)] | static_cast<uint32_t>(row[element(2 * j + 1, true)]) << 16;
            }
            x.a = make_uint4(w[0], w[1], w[2], w[3]);
            x.b = make_uint4(w[4], w[5], w[6], w[7]);
        } else if constexpr (FORM == kQuarter) {
            const uint2 a0 = *reinterpret_cast<const uint2*>(row + element(0, false)), a1 = *reinterpret_cast<const uint2*>(row + element(4, false));
            const uint2 b0 = *reinterpret_cast<const uint2*>(row + element(0, true)), b1 = *reinterpret_cast<const uint2*>(row + element(4, true));
            x.a = make_uint4(a0.x, a0.y, a1.x, a1.y);
            x.b = make_uint4(b0.x, b0.y, b1.x, b1.y);
        } else {
            x.a = *reinterpret_cast<const uint4*>(row + first);
            x.b = *reinterpret_cast<const uint4*>(row + second);
        }
        return x;
    }
    __device__ __forceinline__ void store(uint16_t* row, const Chunks& x) const {
        if constexpr (FORM == kScattered) {
            const uint32_t w[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                row[element(2 * j, false)] = static_cast<uint16_t>(w[j]);
                row[element(2 * j + 1, false)] = static_cast<uint16_t>(w[j] >> 16);
                row[element(2 * j, true)] = static_cast<uint16_t>(w[4 + j]);
                row[element(2 * j + 1, true)] = static_cast<uint16_t>(w[4 + j] >> 16);
            }
        } else if constexpr (FORM == kQuarter) {
            *reinterpret_cast<uint2*>(row + element(0, false)) = make_uint2(x.a.x, x.a.y);
            *reinterpret_cast<uint2*>(row + element(4, false)) = make_uint2(x.a.z, x.a.w);
            *reinterpret_cast<uint2*>(row + element(0, true)) = make_uint2(x.b.x, x.b.y);
            *reinterpret_cast<uint2*>(row + element(4, true)) = make_uint2(x.b.z, x.b.w);
        } else {
            *reinterpret_cast<uint4*>(row + first) = x.a;
            *reinterpret_cast<uint4*>(row + second) = x.b;
        }
    }
};

template <bool BF16>
__device__ __forceinline__ void widen8(const uint4 a, float* v) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
}
template <bool BF16>
__device__ __forceinline__ uint4 narrow8(const float* v) {
    return make_uint4(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]), pack2<BF16>(v[4], v[5]), pack2<BF16>(v[6], v[7]));
}

// A 64-bit value in 16 bits, through fp32 as tensor conversions go.
template <bool BF16>
__device__ __forceinline__ uint32_t narrow(double x) {
    const float f = __double2float_rn(x);
    if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
    else return __half_as_ushort(__float2half_rn(f));
}

// The turning of a thread's 8 pairs, with its sines and cosines; T = float, or double where the result's last bit matters.
template <int FORM, bool BF16, class T>
struct Turner {
    T s[8], c[8];
    int active;                   // how many of the 8 pairs turn
    __device__ __forceinline__ void set(const bob_sm100_rotary& r, int place, int64_t position) {
        active = min(8, max(0, r.pairs - 8 * place));
        if (active == 0) return;
        #pragma unroll
        for (int j = 0; j < 8; j += 2) {                     // (those that do not turn are not used)
            const ulonglong2 turn = turn_pair(r, 4 * place + j / 2);         // (64 of them are there)
            turn_factors(position, turn.x, s[j], c[j]);
            turn_factors(position, turn.y, s[j + 1], c[j + 1]);
        }
        if (r.factor != 1.0) {
            #pragma unroll
            for (int j = 0; j < 8; ++j) { s[j] *= static_cast<T>(r.factor); c[j] *= static_cast<T>(r.factor); }
        }
    }
    static constexpr int STEP = FORM == kInterleaved ? 2 : 1, PARTNER = FORM == kInterleaved ? 1 : 8;
    // The 16 elements in fp32, turned.
    __device__ __forceinline__ void values(const Chunks& x, float (&v)[16]) const {
        widen8<BF16>(x.a, v);
        widen8<BF16>(x.b, v + 8);
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = v[STEP * j], b = v[STEP * j + PARTNER];
            if (j < active) {                                // (elements that do not turn keep their bits)
                v[STEP * j] = a * c[j] - b * s[j];
                v[STEP * j + PARTNER] = b * c[j] + a * s[j];
            }
        }
    }
    __device__ __forceinline__ Chunks operator()(const Chunks& x) const {
        if (active == 0) return x;
        float v[16];
        if constexpr (sizeof(T) == 4) {
            values(x, v);
            return Chunks{narrow8<BF16>(v), narrow8<BF16>(v + 8)};
        } else {
            widen8<BF16>(x.a, v);
            widen8<BF16>(x.b, v + 8);
            uint32_t w[16];
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const T a = v[STEP * j], b = v[STEP * j + PARTNER];
                w[STEP * j] = narrow<BF16>(j < active ? a * c[j] - b * s[j] : a);
                w[STEP * j + PARTNER] = narrow<BF16>(j < active ? b * c[j] + a * s[j] : b);
            }
            Chunks y;
            y.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
            y.b = make_uint4(w[8] | w[9] << 16, w[10] | w[11] << 16, w[12] | w[13] << 16, w[14] | w[15] << 16);
            return y;
        }
    }
};

// Turns a row's 16 elements that were loaded in order (kScattered: through `stage`, the row's place in shared memory; the
// lanes of a row are in one warp, and all lanes call this) or as `place` loads them.
template <int FORM, class TURN>
__device__ __forceinline__ Chunks turned(const TURN& turn, const RowPlace<FORM>& place, const RowPlace<kInterleaved>& plain, Chunks x, uint16_t* stage) {
    if constexpr (FORM == kScattered) {
        plain.store(stage, x);
        __syncwarp();
        const Chunks y = turn(place.load(stage));
        __syncwarp();
        place.store(stage, y);
        __syncwarp();
        x = plain.load(stage);
        __syncwarp();
        return x;
    } else {
        return turn(x);
    }
}
// The place of the 16 elements that a thread loads from, and stores to, global memory.
template <int FORM>
__device__ __forceinline__ auto outer_place(const RowPlace<FORM>& place, const RowPlace<kInterleaved>& plain) {
    if constexpr (FORM == kScattered) return plain; else return place;
}

struct RotateTensor {
    const uint16_t* in; long long in_sb, in_sh, in_sn;      // element strides: batch, head, row
    uint16_t* out;                                          // contiguous [B, H, N, D]
    int H;
};

struct alignas(16) RotateParams {
    bob_sm100_rotary rotary;      // (first: its frequencies are 16-byte aligned)
    RotateTensor t[2];
    int B, N, D;
    const void* positions; int wide; long long pos_sb, pos_sn;   // int64 or int32; null: first + row
    int64_t first;
    int pack;                     // > 1: out is [B, H / pack, N, pack, D]
    const int *lengths, *counts;  // not null: the positions of a paged call's rows (counts null: all N), not the above
};

constexpr int kRotateThreads = 256;

// blockIdx.y: HPT heads, numbered through both tensors.
template <int FORM, bool BF16, int HPT>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(const __grid_constant__ RotateParams p) {
    const int per_row = p.D / 16;
    const long long id = (long long)blockIdx.x * kRotateThreads + threadIdx.x;
    const long long token = id / per_row;
    const bool there = token < (long long)p.B * p.N;             // (the others stay for their warp)
    const int c = static_cast<int>(id % per_row), b = there ? static_cast<int>(token / p.N) : 0, n = there ? static_cast<int>(token % p.N) : 0;
    __shared__ __align__(16) uint16_t stage[FORM == kScattered ? kRotateThreads * 16 : 8];
    const RowPlace<FORM> place(c, p.rotary.pairs);
    const RowPlace<kInterleaved> plain(c, 0);                    // 16 elements in a row
    const auto outer = outer_place(place, plain);
    const int h0 = blockIdx.y * HPT;
    Chunks x[HPT];
    #pragma unroll
    for (int k = 0; k < HPT; ++k) {
        const int h = h0 + k;
        const bool second = h >= p.t[0].H;
        const RotateTensor& t = p.t[second];
        const int th = second ? h - p.t[0].H : h;
        x[k] = Chunks{};
        if (there && th < t.H) x[k] = outer.load(t.in + b * t.in_sb + th * t.in_sh + n * t.in_sn);
    }
    int64_t position = p.first + n;
    if (p.lengths) {
        position = __ldg(p.lengths + b) - (p.counts ? __ldg(p.counts + b) : p.N) + n;
    } else if (p.positions) {
        const long long at = b * p.pos_sb + n * p.pos_sn;
        position = p.wide ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    Turner<FORM, BF16, float> turn;
    turn.set(p.rotary, c, position);
    #pragma unroll
    for (int k = 0; k < HPT; ++k) {
        const int h = h0 + k;
        const bool second = h >= p.t[0].H;
        const RotateTensor& t = p.t[second];
        const int th = second ? h - p.t[0].H : h;
        const Chunks y = turned<FORM>(turn, place, plain, x[k], stage + threadIdx.x / per_row * p.D);
        if (there && th < t.H) outer.store(t.out + ((((long long)b * (t.H / p.pack) + th / p.pack) * p.N + n) * p.pack + th % p.pack) * p.D, y);
    }
}

}  // namespace bob
