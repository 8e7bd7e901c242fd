// Rotary positions: y = m R(position * frequency) x over the first 2 * pairs elements of a head, the others unchanged.
//
// Pair i turns elements (i, i + pairs) or, interleaved, (2 i, 2 i + 1) by position * frequency_i.  The gradient is the
// same map with the angles negated, so one kernel serves forward and every order of backward.
//
// Angles: a frequency is kept as the 64-bit fraction of a turn per position.  position * fraction modulo 2^64 is then
// the exact angle modulo a turn, for any position, in one integer product, and sincospi needs no range reduction;
// position * frequency in fp32 is off by 0.004 radians at position 100,000.
//
// What bounds it: one read and one write of every element.  A thread turns the same 16 elements (8 pairs) of HPT heads of
// a token, so its 8 sines and cosines (about 300 instructions) are shared by them and their loads are in flight together.
#pragma once

#include "ptx.cuh"
#include "../../include/bob_sm100.h"

namespace bob {

// How a thread's 16 elements lie in a row.  kHalf: two 16-byte chunks, partners `pairs` elements apart (pairs a multiple of
// 8); kInterleaved: 16 elements in a row; kScattered: as kHalf for any number of pairs, element by element.
enum RotaryForm : int { kHalf = 0, kInterleaved = 1, kScattered = 2 };

inline int rotary_form(const bob_sm100_rotary* r) {
    return r->interleaved ? kInterleaved : (r->pairs % 8 ? kScattered : kHalf);
}

__device__ __forceinline__ int64_t angle_of(int64_t position, uint64_t turn) {      // 2^-64 turns, in [-1/2, 1/2) turns
    return static_cast<int64_t>(static_cast<uint64_t>(position) * turn);
}
__device__ __forceinline__ void turn_factors(int64_t position, uint64_t turn, float factor, float& s, float& c) {
    // the upper 32 bits: 2^-33 of a turn, 7e-10 radians, far below the rounding of a sine in fp32
    sincospif(static_cast<float>(static_cast<int32_t>(angle_of(position, turn) >> 32)) * 0x1p-31f, &s, &c);
    s *= factor;
    c *= factor;
}
__device__ __forceinline__ void turn_factors(int64_t position, uint64_t turn, double factor, double& s, double& c) {
    sincospi(static_cast<double>(angle_of(position, turn)) * 0x1p-63, &s, &c);
    s *= factor;
    c *= factor;
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
    // kScattered: the elements of pair 8 c + j
    __device__ __forceinline__ int element(int j, bool partner) const {
        const int i = 8 * c + j;
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
        } else {
            x.a = __ldg(reinterpret_cast<const uint4*>(row + first));
            x.b = __ldg(reinterpret_cast<const uint4*>(row + second));
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
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = 0; c[j] = 1;
            if (j < active) turn_factors(position, r.turns[8 * place + j], static_cast<T>(r.factor), s[j], c[j]);
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

struct RotateTensor {
    const uint16_t* in; long long in_sb, in_sh, in_sn;      // element strides: batch, head, row
    uint16_t* out;                                          // contiguous [B, H, N, D]
    int H;
};

struct RotateParams {
    bob_sm100_rotary rotary;
    RotateTensor t[2];
    int B, N, D;
    const void* positions; int wide; long long pos_sb, pos_sn;   // int64 or int32; null: first + row
    int64_t first;
    const int *lengths, *counts;  // not null: the positions of a paged call's rows (counts null: all N), not the above
};

constexpr int kRotateThreads = 256;

// blockIdx.y: HPT heads, numbered through both tensors.
template <int FORM, bool BF16, int HPT>
__global__ void __launch_bounds__(kRotateThreads) rotate_kernel(const __grid_constant__ RotateParams p) {
    const int per_row = p.D / 16;
    const long long id = (long long)blockIdx.x * kRotateThreads + threadIdx.x;
    const long long token = id / per_row;
    if (token >= (long long)p.B * p.N) return;
    const int c = static_cast<int>(id % per_row), b = static_cast<int>(token / p.N), n = static_cast<int>(token % p.N);
    const RowPlace<FORM> place(c, p.rotary.pairs);
    const int h0 = blockIdx.y * HPT;
    Chunks x[HPT];
    #pragma unroll
    for (int k = 0; k < HPT; ++k) {
        const int h = h0 + k;
        const bool second = h >= p.t[0].H;
        const RotateTensor& t = p.t[second];
        const int th = second ? h - p.t[0].H : h;
        x[k] = Chunks{};
        if (th < t.H) x[k] = place.load(t.in + b * t.in_sb + th * t.in_sh + n * t.in_sn);
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
        if (th < t.H) place.store(t.out + (((long long)b * t.H + th) * p.N + n) * p.D, turn(x[k]));
    }
}

}  // namespace bob
