// What the attention kernels share: vector types, what a query sees, which rows a sequence of a batch has.
#pragma once
#include "sequence.h"

#include <type_traits>

namespace fynhip {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr float kNone = -__builtin_huge_valf();

// The positions that one query sees: [lo, hi) and [0, first).
struct Sight {
    int lo, hi, first;
    __device__ bool sees(int j) const { return (j >= lo && j < hi) || j < first; }
};

__device__ __forceinline__ Sight sight_of(int pos, int len, int causal, int window, int sinks) {
    Sight s;
    const int last = causal ? min(pos + 1, len) : len;
    s.lo = 0; s.hi = last; s.first = 0;
    if (window > 0) {
        s.lo = max(0, pos - window + 1);
        s.hi = (int)min((int64_t)last, (int64_t)pos + window);
        s.first = min(sinks, last);
    }
    return s;
}

template <class T, int N> struct Vec;
template <> struct Vec<_Float16, 8> { typedef h8 type; };
template <> struct Vec<_Float16, 4> { typedef h4 type; };
template <> struct Vec<_Float16, 2> { typedef h2 type; };
template <> struct Vec<float, 4> { typedef f4 type; };
template <> struct Vec<float, 2> { typedef f2 type; };

__device__ __forceinline__ bool finite(_Float16 x) { return (__builtin_bit_cast(unsigned short, x) & 0x7c00) != 0x7c00; }
__device__ __forceinline__ bool finite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000) != 0x7f800000; }

// Four values of a result, of which some are NaN though no score is.  A weight that a key's score gives is above zero, but 32 or 16 bits may
// hold it as zero, or what rounding took from it is zero or below: then an infinite value makes NaN where the sum is infinite.  Here it is
// looked up again: what the query sees of the positions [from, to) and [from2, to2) are infinities of one sign, or not (NaN among them).
// src(j): where the four values of position j are.
template <class T, class Src>
__device__ __forceinline__ f4 with_infinities(f4 o, const Sight& see, int from, int to, int from2, int to2, Src src) {
    unsigned odd = 0, nan = 0, up = 0, down = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) odd |= o[e] != o[e] ? 1u << e : 0u;
    for (int part = 0; part < 2; part++) {
        const int a = part ? from2 : from, z = part ? to2 : to;
        for (int j = a; j < z && (odd & ~(nan | (up & down))); j += 8) {
            typename Vec<T, 4>::type x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = *reinterpret_cast<const typename Vec<T, 4>::type*>(src(min(j + i, z - 1)));
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const T v = x[i][e];
                    if (finite(v) || j + i >= z || !see.sees(j + i)) continue;
                    (v > (T)0 ? up : v < (T)0 ? down : nan) |= 1u << e;
                }
        }
    }
    const float inf = __builtin_huge_valf();
#pragma unroll
    for (int e = 0; e < 4; e++)
        if ((odd & ~(nan | (up & down)) & (up | down)) >> e & 1) o[e] = up >> e & 1 ? inf : -inf;
    return o;
}

// A sequence of the batch: its tokens, and its queries: `count` rows from row0 of q and the result, the first of them at
// position pos0.
struct Batched {
    int seq, len, count, row0, pos0;
};

template <bool PAGED>
__device__ __forceinline__ Batched batched(const AttnParams& p, int b) {
    Batched s{b, 0, 0, 0, 0};
    if (PAGED) {
        // (everything that does not wait for another is asked for at once; b is within the tables)
        const int n = p.words.first[p.words.sequences + 1], seq = p.words.batch[b], row0 = p.words.first[b], end = p.words.first[b + 1];
        const int len = p.words.len[seq];
        if (b >= n) return s;
        s.seq = seq;
        s.len = len;
        s.row0 = row0;
        s.count = min(end, p.tokens) - s.row0;
        s.pos0 = s.len - (end - s.row0);
    } else {
        s.len = p.lengths ? min(max(p.lengths[b], 0), p.tokens) : p.tokens;
        s.count = p.tokens;   // (rows behind the length see nothing: zero)
    }
    return s;
}

}  // namespace fynhip
