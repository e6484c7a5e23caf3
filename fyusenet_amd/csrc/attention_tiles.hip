// Attention of many tokens: 128 or 64 queries of one head a workgroup, keys and values in tiles through shared memory.
//
// Each of the four waves has 32 queries as columns.  Per 32 keys
//     S^T [keys x queries]  = K Q^T          K from LDS, Q in registers for the whole run
//     O^T [dims x queries] += V^T P^T        V^T from LDS, P^T as S^T's registers hold it
// with the 32x32 matrix instructions.  Their result has the rows 8i + 4h + 0..3 (i = 0..3) in the lanes of half h, and the inner
// index of the second product is ordered by that, so that the weights go from one product to the next without leaving the
// lane.  Of a query everything, running maximum and sum too, is in two lanes.  With 64 queries two waves have the same ones, each takes
// 32 others of the tile's keys, and their sums are joined at the end.
//
// The next tile goes from memory straight into the other half of the LDS while a tile is worked on: one barrier a tile.  Its rows
// lie as they are in memory, their sixteen-byte pieces exchanged by a pattern of the row's number, so that the sixteen lanes that
// read one piece of sixteen rows (keys), or pieces side by side of eight rows (values), find them in different banks.  Values in
// 16 bits are turned by the LDS as they are read: four keys of a dim to a lane, which had four dims of a key.
//
// In 16 bits a weight goes into the second product as two numbers (22 bits of it; one alone, 11 bits, is 2.6e-4 off the formula in 64
// bits where two are 1.9e-4, which is the result's own rounding), so that a unit of 32 keys by 32 queries, 128 dims, has 24 matrix
// instructions, 768 cycles, and about 720 of vector ones.  By counters a SIMD's two waves take turns with them more than they overlap:
// 16384 tokens, 16 heads of 128, causal, fp16 take 1.63 to 1.69 ms (1.24 with one number), of which the matrix unit is busy 50 %, the
// vector unit 54 %, LDS 17 % (no conflicts), at 1.9 GHz.  Of larger tiles and other orders, with one number, 4096 tokens, 16 heads of 128:
// 32 keys a wave 159 us, 64 keys 166; through registers and turned there 172; the next unit's first product in front of this one's
// exponentials 192 (its registers spill).  fp32, whose matrix instructions are a sixteenth as fast: 4096 tokens, 8 heads of 128, 763 us,
// 90 TFLOP/s (library: 154).
#include "attention_common.h"

namespace fynhip {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

template <class T, int DIMS, int QW>
struct TileShape {
    static constexpr bool F16 = std::is_same<T, _Float16>::value;
    static constexpr int KW = 4 / QW;                                            // waves with the same queries
    static constexpr int TILE = 32 * KW;                                         // keys: each wave has 32 of them at once
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int PIECES = DIMS / VEC;                                    // of a row
    static constexpr int PITCH = PIECES <= 4 ? 4 : PIECES <= 8 ? 8 : PIECES <= 16 ? 16 : 32;   // ... in LDS
    static constexpr int ALL = TILE * PITCH;                                     // pieces of a tile's keys, or values
    static constexpr int LOADS = (ALL + 255) / 256;                              // of a lane, for the keys as for the values
    static_assert(ALL % 256 == 0 || ALL < 256, "whole waves load");
    static constexpr int HALF = 2 * TILE * PITCH * 16;                           // bytes of a tile: keys, then values
    static constexpr int DIM_TILES = DIMS / 32;
    static constexpr int LEAST = DIMS == 256 ? 128 : DIMS - 32;                  // fewer dims than any head of the class has
    static_assert(KW == 1 || HALF >= 2 * DIM_TILES * 4096, "sums of two waves in the place of a tile");
    static constexpr int LDS = 2 * HALF;
    static_assert(LDS + 2048 <= 160 * 1024, "a CU's LDS");
    // Weights are 2^SHIFT times as large as relative to the running maximum, which may be LAG binary orders of magnitude behind the true
    // one.  (In 32 bits the exponent's argument is 1 at most: the larger it is, the fewer bits it has behind the point.)
    static constexpr float SHIFT = F16 ? 6.f : 0.f, LAG = F16 ? 8.f : 1.f;
    static constexpr int WAVES = DIMS <= (F16 ? 128 : 64) && LDS <= 64 * 1024 ? 2 : 1;   // workgroups that share a CU (their registers)
};

// Place of a piece of a row.  (Rows side by side in 256 bytes, the banks' width, are exchanged alike.)
template <int PITCH>
__device__ __forceinline__ int pattern(int row) {
    if (PITCH >= 16) return (row & 3) << 2 | (row >> 2 & 3);
    if (PITCH == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    return row >> 2 & 3;
}
template <int PITCH>
__device__ __forceinline__ int row_piece(int row, int piece) { return row * PITCH + (piece ^ pattern<PITCH>(row)); }

// The larger of a lane's value and that of its other half's.
__device__ __forceinline__ float across(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned a = both[0], b = both[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

template <class T, int DIMS, bool PAGED, int QW>
__global__ __launch_bounds__(256, (TileShape<T, DIMS, QW>::WAVES)) void attend_tiles(const AttnParams p) {
    typedef TileShape<T, DIMS, QW> S;
    typedef typename Vec<T, S::VEC>::type KVec;
    constexpr bool F16 = S::F16;
    constexpr int QUERIES = 32 * QW, V_AT = S::HALF / 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, c = lane & 31, mates = wave / QW, queries = wave % QW;
    // (two arrays: the compiler then knows that a tile that is read is not the one that arrives)
    __shared__ __attribute__((aligned(16))) char tile_a[S::HALF], tile_b[S::HALF];
    __shared__ int odd_values[4];   // a wave found infinities or NaN among a tile's values

    // The last queries first: under a causal mask theirs are the longest runs.  Heads that share keys lie eight workgroups apart
    // where there are eight key heads, on one XCD and its L2.
    const int units = p.batch * p.heads, rounds = (units + 7) / 8, id = blockIdx.x;
    const int unit = id / 8 % rounds * 8 + id % 8, tile = p.tiles - 1 - id / 8 / rounds;
    if (unit >= units) return;
    const int b = p.first_batch + unit / p.heads, kv_head = unit % p.heads % p.kv_heads, head = kv_head * (p.heads / p.kv_heads) + unit % p.heads / p.kv_heads;
    const Batched in = batched<PAGED>(p, b);
    if (tile * QUERIES >= in.count) return;
    const int seen_rows = PAGED ? in.count : min(in.count, in.len);   // (padded rows see nothing)

    // what this lane's query sees, all of the wave's, and all of the workgroup's
    auto sight = [&](int tok) { return sight_of(in.pos0 + tok, in.len, p.causal, p.window, p.sinks); };
    const int tok = tile * QUERIES + queries * 32 + c;
    Sight mine = sight(tok), any, all, group, whole;   // (some query of the wave, all of them; some of the workgroup, all of them)
    if (tok >= seen_rows) mine.lo = mine.hi = mine.first = 0;
    {
        const int a = tile * QUERIES, z = min(a + QUERIES - 1, seen_rows - 1), wa = a + queries * 32, wz = min(wa + 31, seen_rows - 1);
        group = sight(a);
        const Sight last = sight(z), first = sight(wa), wlast = sight(wz);
        whole = Sight{last.lo, group.hi, group.first};
        group.hi = last.hi; group.first = last.first;
        if (z < a) group.lo = group.hi = group.first = whole.lo = whole.hi = whole.first = 0;
        any = Sight{first.lo, wlast.hi, wlast.first};
        all = Sight{wlast.lo, first.hi, first.first};
        if (wz < wa) any.lo = any.hi = any.first = all.lo = all.hi = all.first = 0;
    }
    const int a_steps = (group.first + S::TILE - 1) / S::TILE, b_first = max(group.lo / S::TILE, a_steps);
    const int steps = a_steps + max(0, (group.hi + S::TILE - 1) / S::TILE - b_first);
    const int most = max(group.hi, group.first);

    KVec q[S::PIECES / 2];
    {
        const T* src = reinterpret_cast<const T*>(p.q.p) + (PAGED ? 0 : b * p.q.seq) + (int64_t)(in.row0 + tok) * p.q.tok + (int64_t)head * p.q.head;
#pragma unroll
        for (int s = 0; s < S::PIECES / 2; s++) {
            const int d = (2 * s + half) * S::VEC;
            q[s] = tok < in.count && d < p.dim ? *reinterpret_cast<const KVec*>(src + d) : KVec{};
            if (p.scale_log2 < 0) q[s] = -q[s];   // (the factor is positive below)
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);   // here, and not wherever in the loop the queries are looked at: that would be a wait for the next tile's loads
    }
    const float scale = fabsf(p.scale_log2);

    const char *kbase, *vbase;
    const int* table = nullptr;
    if (PAGED) {
        kbase = p.pages.pool + kv_head * p.pages.head_bytes;
        vbase = kbase + p.pages.values;
        table = p.words.table + (int64_t)in.seq * p.words.table_pitch;
    } else {
        kbase = p.k.p + (b * p.k.seq + kv_head * p.k.head) * (int64_t)sizeof(T);
        vbase = p.v.p + (b * p.v.seq + kv_head * p.v.head) * (int64_t)sizeof(T);
    }
    // The key at + r, `bytes` into it; nothing behind the last visible one is read.
    auto row = [&](const char* base, int64_t tok_pitch, int at, int r, int bytes) -> const char* {
        const int j = min(at + r, most - 1);
        if (PAGED) return base + table[j >> p.pages.shift] * p.pages.page_bytes + ((j & ((1 << p.pages.shift) - 1)) * p.dim * (int)sizeof(T) + bytes);
        return base + (int64_t)j * tok_pitch * (int64_t)sizeof(T) + bytes;
    };
    auto at_of = [&](int st) { return (st < a_steps ? st : b_first + st - a_steps) * S::TILE; };

    // A tile on its way: a lane's sixteen bytes go to the place that its number says, so the exchange of pieces is one of what it
    // asks for.  (Pieces behind a head's last value are taken from within it: of the keys they are zero in the first product, as
    // the queries are, because zero times an infinity of the head's own would not be; of the values they end in dims that nobody stores.)
    const int row_bytes = p.dim * (int)sizeof(T);
    constexpr int ROWS = 64 / S::PITCH;   // of a load
    const int lane_row = lane / S::PITCH, lane_piece = lane % S::PITCH;
    const unsigned k_lane = (unsigned)(lane_row * (int)p.k.tok * (int)sizeof(T)), v_lane = (unsigned)(lane_row * (int)p.v.tok * (int)sizeof(T));
    auto arrive = [&](char* dst, const char* k, const char* v) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)k, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)v, (__attribute__((address_space(3))) void*)(dst + V_AT), 16, 0, 0);
    };
    auto fetch = [&](char* dst, int at) {
        const bool inside = !PAGED && at + S::TILE <= most;
        const char* kb = kbase + (int64_t)at * p.k.tok * (int64_t)sizeof(T);
        const char* vb = vbase + (int64_t)at * p.v.tok * (int64_t)sizeof(T);
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            const int first = (wave * S::LOADS + i) * ROWS, bytes = min((lane_piece ^ pattern<S::PITCH>(first + lane_row)) * 16, row_bytes - 16);
            if (S::ALL < 256 && first >= S::TILE) break;
            char* to = dst + first * S::PITCH * 16;
            if (inside)   // (scalar bases and 32 bits of offset: the host has seen to that)
                arrive(to, kb + (int64_t)first * p.k.tok * (int64_t)sizeof(T) + (k_lane + bytes), vb + (int64_t)first * p.v.tok * (int64_t)sizeof(T) + (v_lane + bytes));
            else
                arrive(to, row(kbase, p.k.tok, at, first + lane_row, bytes), row(vbase, p.v.tok, at, first + lane_row, bytes));
        }
    };
    // A tile that not all of the workgroup's queries see whole: infinities and NaN among its values are left out, and those who
    // see them are told.
    auto clean = [&](char* tile) {
        u4* vl = reinterpret_cast<u4*>(tile + V_AT);
        bool found = false;
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            if (S::ALL < 256 && tid >= S::ALL) break;
            u4 x = vl[i * 256 + tid];
            bool any_odd = false;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned y = x[e];
                if constexpr (F16) {   // (an exponent of all ones carries into the sign's place)
                    const unsigned odd = ((y & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
                    any_odd = any_odd || odd;
                    x[e] = y & ~((odd << 1) - (odd >> 15));
                } else {
                    const bool odd = (y & 0x7f800000u) == 0x7f800000u;
                    any_odd = any_odd || odd;
                    x[e] = odd ? 0 : y;
                }
            }
            if (any_odd) vl[i * 256 + tid] = x;
            found = found || any_odd;
        }
        found = __any(found);
        if (lane == 0) odd_values[wave] = found;
    };
    auto is_partial = [&](int at) { return !((at >= whole.lo && at + S::TILE <= whole.hi) || at + S::TILE <= whole.first); };

    f16v acc[S::DIM_TILES];
#pragma unroll
    for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[d][r] = 0.f;
    float m = kNone, l = 0;   // (l: of this lane's keys only)

    auto work = [&](char* tile, char* other, int st) {
        const int from = at_of(st), at = from + mates * 32;   // (the wave's keys)
        __builtin_amdgcn_s_waitcnt(0x0f70);   // (the wave's part of the tile has arrived)
        __syncthreads();                      // the tile is in LDS, and nobody reads the other any more
        if (st + 1 < steps) fetch(other, at_of(st + 1));
        __builtin_amdgcn_sched_barrier(0);
        const bool partial = is_partial(from);
        if (partial) {
            clean(tile);
            __syncthreads();
        }
        if ((at < any.hi && at + 32 > any.lo) || at < any.first) {
            const char* kl = tile;
            const char* vl = tile + V_AT;
            f16v sc;
#pragma unroll
            for (int r = 0; r < 16; r++) sc[r] = 0.f;
            // (All pieces of the keys are asked for before the first is needed, where there are registers for them: left to itself the
            // compiler asks for each in front of its use, and the use waits.)
            constexpr bool AHEAD = DIMS <= 128;
            KVec kf[S::PIECES / 2];
#pragma unroll
            for (int s = 0; s < S::PIECES / 2; s++) kf[s] = *reinterpret_cast<const KVec*>(kl + 16 * row_piece<S::PITCH>(mates * 32 + c, 2 * s + half));
            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
            // (Pieces behind the head are zero.  In 32 bits in front of the products, for heads that have such: 8 heads of 128, 4096 tokens,
            // 763 us, and 783 with a select for each product; in 16 bits, heads of 256, 2048 tokens, the branch spills: 222 us and 160.)
            if (!F16 && p.dim < DIMS) {
#pragma unroll
                for (int s = 0; s < S::PIECES / 2; s++)
                    if ((2 * s + 2) * S::VEC > S::LEAST && (2 * s + half) * S::VEC >= p.dim) kf[s] = KVec{};
            }
#pragma unroll
            for (int s = 0; s < S::PIECES / 2; s++) {
                if constexpr (F16) {
                    const KVec piece = (2 * s + 2) * S::VEC <= S::LEAST || (2 * s + half) * S::VEC < p.dim ? kf[s] : KVec{};
                    sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(piece, q[s], sc, 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) sc = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[s][e], q[s][e], sc, 0, 0, 0);
                }
            }
            if (!((at >= all.lo && at + 32 <= all.hi) || at + 32 <= all.first)) {
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!mine.sees(at + (r & 3) + 8 * (r >> 2) + 4 * half)) sc[r] = kNone;
            }
            // Dims 32 d + c, keys 4 half .. + 3 of the sixteen t, and those 8 further on.  A lane names what it has before they are
            // turned: key lane / 4 % 4 of the four, and the dims from 16 (c / 16) + 4 (lane % 4) on.
            auto value = [&](int t, int d) {
                h8 v;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int key = mates * 32 + 16 * t + 8 * e + 4 * half + (lane >> 2 & 3), dim = 32 * d + 16 * (c >> 4) + 4 * (lane & 3);
                    const h4 four = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s4*)(vl + 16 * row_piece<S::PITCH>(key, dim / 8) + dim % 8 * 2)));
#pragma unroll
                    for (int i = 0; i < 4; i++) v[4 * e + i] = four[i];
                }
                return v;
            };
            h8 vf[F16 ? S::DIM_TILES : 1];
            if constexpr (F16) {
#pragma unroll
                for (int d = 0; d < S::DIM_TILES; d++) vf[d] = value(0, d);
                if (AHEAD) __builtin_amdgcn_sched_barrier(0);
            }
            float top = kNone;
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, sc[r]);
            top = across(top) * scale;
            // The sums are relative to a maximum that may be the true one's 2^-LAG (in 16 bits with weights up to 2^14 then): it follows where
            // a query is further off, which after the first tiles is seldom.  (fp32, 4096 tokens, 8 heads of 128: 786 us, and 798 if it always
            // follows.)
            if (__any(top > m + S::LAG)) {
                const float m_new = top > m + S::LAG ? top : m, alpha = m == kNone ? 0.f : __builtin_amdgcn_exp2f(m - m_new);   // (by each query alone)
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[d][r] *= alpha;
            }
            // In 16 bits a weight is 2^6 times as large as relative to m, and two numbers: what the first one's rounding takes from it
            // is the second, 22 bits of it in all down to 2^-9 of the largest weight, and never off by more than 2^-31 of that one.
            const float base = m == kNone ? 0.f : m - S::SHIFT;
#pragma unroll
            for (int r = 0; r < 16; r++) sc[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], scale, -base));
            float sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < 16; r++) sum[r & 3] += sc[r];
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if constexpr (F16) {
                h8 w[2], rest[2];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        w[t][e] = (_Float16)sc[t * 8 + e];
                        rest[t][e] = (_Float16)(sc[t * 8 + e] - (float)w[t][e]);
                    }
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int d = 0; d < S::DIM_TILES; d++) {
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], w[t], acc[d], 0, 0, 0);
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], rest[t], acc[d], 0, 0, 0);
                        if (t == 0) {
                            vf[d] = value(1, d);
                            if (AHEAD) __builtin_amdgcn_sched_barrier(0);
                        }
                    }
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++)
#pragma unroll
                    for (int d = 0; d < S::DIM_TILES; d++) {
                        const int key = mates * 32 + (r & 3) + 8 * (r >> 2) + 4 * half, dim = 32 * d + c;
                        const float v = *reinterpret_cast<const float*>(vl + 16 * row_piece<S::PITCH>(key, dim / 4) + dim % 4 * 4);
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[r], acc[d], 0, 0, 0);
                    }
            }
            // Values that were left out: whoever sees them has them in the result (a weight is never negative).
            if (partial && (odd_values[0] | odd_values[1] | odd_values[2] | odd_values[3])) {
                for (int key = 0; key < 32; key++) {
                    const T* v = reinterpret_cast<const T*>(row(vbase, p.v.tok, at, key, 0));
                    const bool sees = mine.sees(at + key);
                    int h4 = 4 * half;
                    asm volatile("" : "+v"(h4));   // (no address is kept over the loop, whose registers the products need)
#pragma unroll
                    for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const T x = v[min(32 * d + (r & 3) + 8 * (r >> 2) + h4, p.dim - 1)];
                            if (sees && !finite(x)) acc[d][r] += (float)x;
                            __builtin_amdgcn_sched_barrier(0);
                        }
                }
            }
        }
    };
    if (steps > 0) fetch(tile_a, at_of(0));
    for (int st = 0; st < steps; st += 2) {
        work(tile_a, tile_b, st);
        if (st + 1 < steps) work(tile_b, tile_a, st + 1);
    }

    l += __shfl_xor(l, 32);
    if constexpr (S::KW > 1) {
        // The sums of the waves with the same queries, as they lie in the registers; each wave joins its share of the dims.
        __shared__ float tops[4][32], totals[4][32];
        if (half == 0) {
            tops[wave][c] = m;
            totals[wave][c] = l;
        }
        __syncthreads();   // (the last tile has been read, too)
        float top = kNone, total = 0;
#pragma unroll
        for (int k = 0; k < S::KW; k++) top = fmaxf(top, tops[k * QW + queries][c]);
#pragma unroll
        for (int k = 0; k < S::KW; k++) total += top == kNone ? 0.f : totals[k * QW + queries][c] * __builtin_amdgcn_exp2f(tops[k * QW + queries][c] - top);
        const float f = top == kNone ? 0.f : __builtin_amdgcn_exp2f(m - top);
        auto sums = [&](int w, int d, int r) -> float& { return reinterpret_cast<float*>(w < 2 ? tile_a : tile_b)[(((w & 1) * S::DIM_TILES + d) * 16 + r) * 64 + lane]; };
#pragma unroll
        for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) sums(wave, d, r) = acc[d][r] * f;
        __syncthreads();
#pragma unroll
        for (int d = 0; d < S::DIM_TILES; d++)
            if (d % S::KW == mates)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float sum = 0;
#pragma unroll
                    for (int k = 0; k < S::KW; k++) sum += sums(k * QW + queries, d, r);
                    acc[d][r] = sum;
                }
        l = total;
    }
    if (tok >= in.count) return;
    const bool zero = tok >= seen_rows;
    bool odd = false;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = reinterpret_cast<T*>(p.out.p) + (PAGED ? 0 : b * p.out.seq) + (int64_t)(in.row0 + tok) * p.out.tok + (int64_t)head * p.out.head;
#pragma unroll
    for (int d = 0; d < S::DIM_TILES; d++) {
        if (d % S::KW != mates) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int dim = 32 * d + 8 * j + 4 * half;
            typename Vec<T, 4>::type t;
#pragma unroll
            for (int e = 0; e < 4; e++) t[e] = zero ? (T)0 : (T)(acc[d][4 * j + e] * inv);
            if (dim < p.dim) {
                *reinterpret_cast<typename Vec<T, 4>::type*>(dst + dim) = t;
#pragma unroll
                for (int e = 0; e < 4; e++) odd = odd || t[e] != t[e];
            }
        }
    }
    // (seldom: from what has been stored, so that no sum is kept for it)
    if (odd && l == l)
        for (int dim = 4 * half; dim < p.dim; dim += 8) {
            if (dim / 32 % S::KW != mates) continue;
            auto& at = *reinterpret_cast<typename Vec<T, 4>::type*>(dst + dim);
            const typename Vec<T, 4>::type t = at;
            if (t[0] == t[0] && t[1] == t[1] && t[2] == t[2] && t[3] == t[3]) continue;
            const f4 o = with_infinities<T>(f4{(float)t[0], (float)t[1], (float)t[2], (float)t[3]}, mine, 0, mine.first, mine.lo, mine.hi,
                                            [&](int j) { return reinterpret_cast<const T*>(row(vbase, p.v.tok, j, 0, 0)) + dim; });
            at = typename Vec<T, 4>::type{(T)o[0], (T)o[1], (T)o[2], (T)o[3]};
        }
}

template <class T, int DIMS, int QW>
static hipError_t launch_tiles(const AttnParams& p, unsigned blocks, hipStream_t s) {
    return start(p.paged ? attend_tiles<T, DIMS, true, QW> : attend_tiles<T, DIMS, false, QW>, blocks, s, p);
}

#if FYN_ATTN_HALF
typedef _Float16 Stored;
#define FYN_ATTN_NAME launch_tiles_f16
#else
typedef float Stored;
#define FYN_ATTN_NAME launch_tiles_f32
#endif

template <int QW>
static int launch_class(const AttnParams& p, unsigned blocks, hipStream_t s) {
    hipError_t e;
    if (p.dim <= 32) e = launch_tiles<Stored, 32, QW>(p, blocks, s);
    else if (p.dim <= 64) e = launch_tiles<Stored, 64, QW>(p, blocks, s);
    else if (p.dim <= 96) e = launch_tiles<Stored, 96, QW>(p, blocks, s);
    else if (p.dim <= 128) e = launch_tiles<Stored, 128, QW>(p, blocks, s);
#if FYN_ATTN_HALF
    else e = launch_tiles<Stored, 256, QW>(p, blocks, s);
#else
    else return -1;   // (queries and sums of 32 bits: more registers than a wave has)
#endif
    return e == hipSuccess ? 0 : -1;
}

int FYN_ATTN_NAME(const AttnParams& p, unsigned blocks, hipStream_t s) { return p.tiled == 128 ? launch_class<4>(p, blocks, s) : launch_class<2>(p, blocks, s); }

}  // namespace fynhip
