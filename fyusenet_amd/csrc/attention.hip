// Attention over a sequence's keys and values, dense or in the pages of a cache.
//
// For a query at position i of a sequence of n tokens the visible positions are
//     j < n,  j <= i (causal),  |i - j| < window or j < sinks (window > 0)
// and with s_j = scale <q, k_j> the result is  sum_j exp(s_j) v_j / sum_j exp(s_j)  over them, zero where there are none.
//
// One pass over the keys: a running maximum m and, relative to it, the running sum of the weights and of the weighted
// values; where m grows both are multiplied with exp(m_old - m_new).  All of that is held in 32 bits.
#include "attention_common.h"

#include <algorithm>

namespace fynhip {

// ---------------------------------------------------------------------------------------------------------------------
// Columns of queries against steps of keys, without shared memory on the way.
//
// A workgroup has sixteen columns: one token's heads of one key head (a group shares its keys), or sixteen tokens of one
// head.  Its four waves take the steps of 16 or 32 keys in turn and join their sums at the end.  In a step
//     S^T [keys x columns]  = K Q^T         K straight from memory as the matrix instruction's first operand
//     O^T [dims x columns] += V^T P^T       V^T likewise, P^T is what S^T's registers hold already
// The instruction multiplies with any order of its inner index, as long as both operands have the same one.  The lanes
// l/16 = g hold rows 4g..4g+3 of S^T, so the inner index of the second product is ordered by them: a lane loads the
// values of the keys 4g..4g+3 of each sixteen, a few neighbouring dims at a time, and P^T never leaves its registers.
// A dim's keys are brought together by byte permutes of the lane's own registers (half a one for each value).
//
// Memory bound where a group's heads are the columns: every key and value is read once, in rows of 16 bytes a lane.  The next
// step's loads are under way while a step is worked on (in the registers that its products have freed).  64 sequences of 32768
// tokens, 8 key heads of 128, fp16: 1.24 ms, 6.9 TB/s of the 7.1 that reading alone reaches; 24 ragged ones of up to 5000: 57 to 67 us
// (3.9 to 4.6 TB/s: a workgroup's start, its joins, the unequal lengths and the parts' short rests weigh there); 16 with a window of 4096,
// 8 heads of 96, fp32: 72 to 74 us (4.8 TB/s).  Over pages that all sequences of a batch begin with, the columns are heads of several
// sequences.  Sixteen tokens as columns serve short prompts: 12 heads of 197 tokens take 7.1 us, 8.7 in tiles.
// ---------------------------------------------------------------------------------------------------------------------
template <class T, int DIMS>
struct Shape {
    static constexpr bool F16 = std::is_same<T, _Float16>::value;
    static constexpr int VEC = 16 / sizeof(T);                    // elements of a lane's load of K
    static constexpr int KLOADS = DIMS / (4 * VEC);               // ... for one key: 4 lanes side by side
    static constexpr int TILES = (!F16 && DIMS > 128) ? 1 : 2;    // sixteens of keys in a step
    static constexpr int STEP = 16 * TILES;
    static constexpr int WAVES = F16 && DIMS <= 128 ? 3 : DIMS <= 64 ? 3 : DIMS <= 128 ? 2 : 1;   // workgroups that share a CU
    static constexpr int LEAST = DIMS == 32 ? 0 : DIMS == 256 ? 128 : DIMS - 32;   // fewer dims than any head of the class has
    static constexpr int E = DIMS / 16 < VEC ? DIMS / 16 : VEC;   // dims that a lane loads of V at once
    static constexpr int BLOCKS = (DIMS + 16 * E - 1) / (16 * E);
    static constexpr int PITCH = BLOCKS * 16 * E + 4;             // of the joined sums in LDS (floats)
};
// (the classes of dims: DIMS = 32, 64, 96, 128, 256; E = 2, 4, 8 (6 would not be a power of two), 8, 8 of fp16 and
// 2, 4, 4, 4, 4 of fp32)
template <class T>
struct Shape<T, 96> {
    static constexpr bool F16 = std::is_same<T, _Float16>::value;
    static constexpr int VEC = 16 / sizeof(T), KLOADS = 96 / (4 * VEC), TILES = 2, STEP = 32, LEAST = 64, WAVES = F16 ? 3 : 2, E = F16 ? 8 : 4, BLOCKS = F16 ? 1 : 2, PITCH = 132;
};

template <bool ONCE, class V>
__device__ __forceinline__ V load(const void* p) {
    return ONCE ? __builtin_nontemporal_load(reinterpret_cast<const V*>(p)) : *reinterpret_cast<const V*>(p);
}

template <class T, int DIMS, bool PAGED, bool BY_TOKEN, bool ONCE>
__global__ __launch_bounds__(256, (Shape<T, DIMS>::WAVES)) void attend_steps(const AttnParams p) {
    typedef Shape<T, DIMS> S;
    typedef typename Vec<T, S::VEC>::type KVec;
    typedef typename Vec<T, S::E>::type VVec;
    constexpr bool F16 = S::F16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;

    // Which part of which columns.  Workgroups that read the same keys for different sequences (branches of one sequence
    // share pages) or columns lie eight apart, which is on one XCD and its L2, one behind the other.
    constexpr bool BRANCHES = PAGED && !BY_TOKEN && !ONCE;   // some tokens may be those of all sequences (AttnParams::common)
    const int group = p.heads / p.kv_heads, across = BY_TOKEN ? p.heads : p.kv_heads;
    const int common_blocks = BRANCHES && p.common ? (across * p.common_parts + 7) / 8 * 8 * p.common_tiles : 0;
    const bool together = BRANCHES && (int)blockIdx.x < common_blocks;
    const int columns = together ? p.common_tiles : p.tiles * p.batch, parts = together ? p.common_parts : p.parts - (BRANCHES ? p.common_parts : 0);
    const int id = (int)blockIdx.x - (together ? 0 : common_blocks), x = (id / (8 * columns)) * 8 + id % 8, col_tile = id / 8 % columns;
    if (x >= across * parts) return;
    const int part = x / across, who = x % across, b = together ? 0 : p.first_batch + col_tile / p.tiles, tile = together ? 0 : col_tile % p.tiles;
    const int kv_head = BY_TOKEN ? who / group : who;

    const Batched in = batched<PAGED>(p, b);
    const int len = in.len, count = in.count, row0 = in.row0, seq = in.seq, pos0 = in.pos0;
    const int token_tile = BY_TOKEN ? tile : tile / ((group + 15) / 16);
    if ((BY_TOKEN ? token_tile * 16 : token_tile) >= count) return;
    // a column's row of the queries (from row0 on) and its head; whether there is such a column
    const int first_head = BY_TOKEN ? 0 : tile % ((group + 15) / 16) * 16;
    auto row_of = [&](int col) { return together ? (col_tile * 16 + col) / group : BY_TOKEN ? token_tile * 16 + col : token_tile; };
    auto head_of = [&](int col) { return together ? kv_head * group + (col_tile * 16 + col) % group : BY_TOKEN ? who : kv_head * group + first_head + col; };
    auto exists = [&](int col) { return together ? col_tile * 16 + col < min(p.batch, p.tokens) * group : BY_TOKEN ? token_tile * 16 + col < count : first_head + col < group; };
    const int tok = row_of(c), head = head_of(c);
    const bool valid = exists(c);
    const bool inside = PAGED || pos0 + tok < len;   // (a padded row sees nothing)

    // what the columns see, one by one and together
    Sight mine, any, all;
    if (together) {
        mine = any = all = Sight{0, p.common, 0};
    } else {
        mine = sight_of(pos0 + tok, len, p.causal, p.window, p.sinks);
        const int tok_a = BY_TOKEN ? token_tile * 16 : token_tile, tok_b = BY_TOKEN ? min(tok_a + 15, (PAGED ? count : min(count, len)) - 1) : token_tile;
        any = all = sight_of(pos0 + tok_a, len, p.causal, p.window, p.sinks);
        if (tok_b < tok_a || (!PAGED && pos0 + tok_a >= len)) {
            any.lo = any.hi = any.first = 0;
            all = any;
        } else if (BY_TOKEN) {
            const Sight last = sight_of(pos0 + tok_b, len, p.causal, p.window, p.sinks);
            any.hi = last.hi; any.first = last.first;
            all.lo = last.lo;
        }
        if (BRANCHES && p.common) mine.lo = any.lo = all.lo = p.common;
    }
    if (!valid || !inside) mine.lo = mine.hi = mine.first = 0;
    const int a_steps = (any.first + S::STEP - 1) / S::STEP, b_first = max(any.lo / S::STEP, a_steps);
    const int b_steps = max(0, (any.hi + S::STEP - 1) / S::STEP - b_first), steps = a_steps + b_steps;
    // (parts of as many steps for every row, and what is left as its last one: those of long and short sequences take equally long)
    const int chunk = max(together ? p.common_chunk : p.chunk, (steps + parts - 1) / parts), begin = part * chunk, end = min(steps, begin + chunk);
    if (begin > 0 && begin >= end) return;
    const int most = max(any.hi, any.first);   // positions from here on are not read

    // queries: operand of the first product
    KVec q[S::KLOADS];
    {
        const T* src = reinterpret_cast<const T*>(p.q.p) + (PAGED ? 0 : b * p.q.seq) + (int64_t)(row0 + tok) * p.q.tok + (int64_t)head * p.q.head;
#pragma unroll
        for (int s = 0; s < S::KLOADS; s++) {
            const int d = (s * 4 + g) * S::VEC;
            q[s] = valid && d < p.dim ? *reinterpret_cast<const KVec*>(src + d) : KVec{};
        }
    }
    f4 acc[S::BLOCKS][S::E];
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
        for (int n = 0; n < S::E; n++) acc[i][n] = f4{0, 0, 0, 0};
    float m = kNone, l = 0;   // (l: of this lane's keys only)

    const char *kbase, *vbase;
    if (PAGED) {
        kbase = p.pages.pool + kv_head * p.pages.head_bytes;
        vbase = kbase + p.pages.values;
    } else {
        kbase = p.k.p + (b * p.k.seq + kv_head * p.k.head) * (int64_t)sizeof(T);
        vbase = p.v.p + (b * p.v.seq + kv_head * p.v.head) * (int64_t)sizeof(T);
    }
    const int* table = PAGED ? p.words.table + (int64_t)seq * p.words.table_pitch : nullptr;

    // Where a step's keys and values are for this lane: those of key 16 t + c, piece g, and of the keys 16 t + 4 g .. + 3,
    // dims from c E on.  Pages have eight tokens or more: half a sixteen lies in one.  A list is not read behind its last page;
    // what is read behind the last visible key is within a page (or, nothing paged, the last visible key again).
    struct Where {
        const char *k[S::TILES], *v[S::TILES];
        int rows[S::TILES];   // nothing paged: how many keys from the lane's first value's there are, less one
    };
    const int row_bytes = p.dim * (int)sizeof(T);
    auto at_of = [&](int st) { return (st < a_steps ? st : b_first + st - a_steps) * S::STEP; };
    auto where = [&](int at) {
        Where w;
        if (PAGED) {
            const int top = (most - 1) >> p.pages.shift, mask = (1 << p.pages.shift) - 1;
#pragma unroll
            for (int t = 0; t < S::TILES; t++) {
                const int64_t a = table[min((at + 16 * t) >> p.pages.shift, top)] * p.pages.page_bytes, b = table[min((at + 16 * t + 8) >> p.pages.shift, top)] * p.pages.page_bytes;
                w.k[t] = kbase + (c < 8 ? a : b) + ((at + 16 * t + c) & mask) * row_bytes;
                w.v[t] = vbase + (g < 2 ? a : b) + ((at + 16 * t + 4 * g) & mask) * row_bytes;
                w.rows[t] = 3;
            }
        } else {
#pragma unroll
            for (int t = 0; t < S::TILES; t++) {
                w.k[t] = kbase + min(at + 16 * t + c, most - 1) * p.k.tok * (int64_t)sizeof(T);
                const int j = min(at + 16 * t + 4 * g, most - 1);
                w.v[t] = vbase + j * p.v.tok * (int64_t)sizeof(T);
                w.rows[t] = most - 1 - j;
            }
        }
        return w;
    };
    const int64_t v_pitch = PAGED ? row_bytes : p.v.tok * (int64_t)sizeof(T);
    KVec k[S::TILES][S::KLOADS];
    VVec v[S::TILES][4][S::BLOCKS];
    // Pieces behind a head's last value are taken from within it.  Of the values they end in dims that nobody stores; of the keys they are
    // zero in the product, as the queries are (zero times an infinity of the head's own would not be).
    auto load_keys = [&](const Where& w) {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int s = 0; s < S::KLOADS; s++) {
                const int at = (s * 4 + g) * 16;
                k[t][s] = load<ONCE, KVec>(w.k[t] + ((s + 1) * 4 * S::VEC <= S::LEAST ? at : min(at, row_bytes - 16)));
            }
    };
    auto load_values = [&](const Where& w) {
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < S::BLOCKS; i++) {
                    const int at = (i * 16 + c) * S::E * (int)sizeof(T);
                    v[t][r][i] = load<ONCE, VVec>(w.v[t] + min(r, w.rows[t]) * v_pitch + min(at, row_bytes - S::E * (int)sizeof(T)));
                }
    };
    // The next step's keys are asked for when this one's have gone through the first product, its values when these have gone
    // through the second.
    if (begin + wave < end) {
        const Where w = where(at_of(begin + wave));
        load_keys(w);
        load_values(w);
    }
    for (int st = begin + wave; st < end; st += 4) {
        const int at = at_of(st);
        const Where next = where(at_of(min(st + 4, end - 1)));
        // scores
        if (p.dim < DIMS) {
#pragma unroll
            for (int s = 0; s < S::KLOADS; s++)
#pragma unroll
                for (int t = 0; t < S::TILES; t++)
                    if ((s + 1) * 4 * S::VEC > S::LEAST && (s * 4 + g) * S::VEC >= p.dim) k[t][s] = KVec{};
        }
        f4 sc[S::TILES];
#pragma unroll
        for (int t = 0; t < S::TILES; t++) {
            sc[t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S::KLOADS; s++) {
                if constexpr (F16) {
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][s], q[s], sc[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][s][e], q[s][e], sc[t], 0, 0, 0);
                }
            }
            sc[t] *= p.scale_log2;
        }
        if (st + 4 < end) load_keys(next);
        // Whether every column sees every key of the step; if not, what a column does not see weighs nothing, whatever
        // the memory holds there.
        const bool whole = (at >= all.lo && at + S::STEP <= all.hi) || at + S::STEP <= all.first;
        bool fix = false;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = at + 16 * t + 4 * g + r;
                    if (!mine.sees(j)) sc[t][r] = kNone;
                    const bool used = any.sees(j);
#pragma unroll
                    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                        for (int n = 0; n < S::E; n++) {
                            if (!used) v[t][r][i][n] = 0;
                            if (BY_TOKEN && !finite(v[t][r][i][n])) {   // a value that one column sees and another does not
                                v[t][r][i][n] = 0;
                                fix = true;
                            }
                        }
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) top = fmaxf(top, sc[t][r]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m_new = fmaxf(m, top), base = m_new == kNone ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - base);   // (m = none: 0)
        m = m_new;
        // In 16 bits weights are kept 2^14 times as large: they then have their full precision down to 2^-28 of the largest, and
        // what rounding takes from them is a second operand of the product.  (In 32 bits nothing is gained by that, and the
        // exponent's argument would lose three bits: 14 has steps of 2^-20.)
        constexpr float shift = F16 ? 14.f : 0.f;
        f4 w[S::TILES];
        float sum = 0;
#pragma unroll
        for (int t = 0; t < S::TILES; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                w[t][r] = __builtin_amdgcn_exp2f(sc[t][r] - base + shift);
                sum += w[t][r];
            }
        l = l * alpha + sum;
#pragma unroll
        for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
            for (int n = 0; n < S::E; n++) acc[i][n] *= alpha;
        if constexpr (F16) {
            h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                hi[e] = (_Float16)w[e / 4][e % 4];
                lo[e] = (_Float16)(w[e / 4][e % 4] - (float)hi[e]);
            }
#pragma unroll
            for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                for (int n = 0; n < S::E; n++) {
                    h8 vt;
#pragma unroll
                    for (int e = 0; e < 8; e++) vt[e] = v[e / 4][e % 4][i][n];
                    acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, hi, acc[i][n], 0, 0, 0);
                    acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, lo, acc[i][n], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int t = 0; t < S::TILES; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                        for (int n = 0; n < S::E; n++) acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t][r][i][n], w[t][r], acc[i][n], 0, 0, 0);
        }
        // Infinities and NaN among the values of such a step: only for the columns that see them.
        if (BY_TOKEN && __any(fix)) {
            for (int off = 0; off < S::STEP; off++) {
                const int t = off / 16, owner = off % 16 / 4, r = off % 4;
                float weight = 0;
#pragma unroll
                for (int tt = 0; tt < S::TILES; tt++)
#pragma unroll
                    for (int rr = 0; rr < 4; rr++)
                        if (tt == t && rr == r) weight = w[tt][rr];
                weight = __shfl(weight, owner * 16 + c);
                const int j = min(at + off, most - 1);
                const T* src = reinterpret_cast<const T*>(PAGED ? vbase + table[j >> p.pages.shift] * p.pages.page_bytes + (j & ((1 << p.pages.shift) - 1)) * row_bytes
                                                                : vbase + j * p.v.tok * (int64_t)sizeof(T));
#pragma unroll
                for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
                    for (int n = 0; n < S::E; n++)
#pragma unroll
                        for (int rr = 0; rr < 4; rr++) {
                            const int d = (i * 16 + 4 * g + rr) * S::E + n;
                            if (d < p.dim && mine.sees(at + off)) {
                                const T val = src[d];
                                if (!finite(val)) acc[i][n][rr] += weight * (float)val;
                            }
                        }
            }
        }
        if (st + 4 < end) load_values(next);
    }

    // the four waves' sums: each has a maximum of its own
    __shared__ __attribute__((aligned(16))) float sums[4][16][S::PITCH];
    __shared__ float tops[4][16], totals[4][16];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        tops[wave][c] = m;
        totals[wave][c] = l;
    }
    // (sums[][column][dim]: register n of block i, row 4g+r is dim (16 i + 4g + r) E + n)
#pragma unroll
    for (int i = 0; i < S::BLOCKS; i++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int n = 0; n < S::E; n++) sums[wave][c][(i * 16 + 4 * g + r) * S::E + n] = acc[i][n][r];
    __syncthreads();
    // (sixteen threads for a column)
    const int col = threadIdx.x >> 4, sub = threadIdx.x & 15;
    const int o_tok = row_of(col), o_head = head_of(col);
    if (!exists(col)) return;
    float mm = kNone;
    for (int w = 0; w < 4; w++) mm = fmaxf(mm, tops[w][col]);
    const float base = mm == kNone ? 0.f : mm;
    float f[4], total = 0;
    for (int w = 0; w < 4; w++) {
        f[w] = __builtin_amdgcn_exp2f(tops[w][col] - base);
        total += totals[w][col] * f[w];
    }
    const bool only = steps <= chunk && !(BRANCHES && p.common);   // the row has one part
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const bool zero = !PAGED && o_tok >= len;   // (a padded row: its column took part in steps that all others see whole)
    const int64_t r_out = (int64_t)row0 + o_tok;
    T* dst = reinterpret_cast<T*>(p.out.p) + (PAGED ? 0 : b * p.out.seq) + r_out * p.out.tok + (int64_t)o_head * p.out.head;
    const int64_t cell = ((PAGED ? r_out : (int64_t)b * p.tokens + r_out) * p.heads + o_head) * p.parts + (BRANCHES && !together ? p.common_parts : 0) + part;
    for (int d = sub * 4; d < p.dim; d += 64) {
        f4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) o += *reinterpret_cast<const f4*>(&sums[w][col][d]) * f[w];
        if (!zero && total == total && (o[0] != o[0] || o[1] != o[1] || o[2] != o[2] || o[3] != o[3])) {
            Sight see = together ? any : sight_of(pos0 + o_tok, len, p.causal, p.window, p.sinks);
            if (BRANCHES && p.common && !together) see.lo = p.common;
            const int second = b_first - a_steps;   // (steps of the window are so many further on)
            o = with_infinities<T>(o, see, begin * S::STEP, min(min(end, a_steps) * S::STEP, most), (second + max(begin, a_steps)) * S::STEP, min((second + end) * S::STEP, most),
                                   [&](int j) { return reinterpret_cast<const T*>(PAGED ? vbase + table[j >> p.pages.shift] * p.pages.page_bytes + (j & ((1 << p.pages.shift) - 1)) * row_bytes
                                                                                        : vbase + j * p.v.tok * (int64_t)sizeof(T)) + d; });
        }
        if (only) {
            typename Vec<T, 4>::type t;
#pragma unroll
            for (int e = 0; e < 4; e++) t[e] = zero ? (T)0 : (T)(o[e] * inv);
            *reinterpret_cast<typename Vec<T, 4>::type*>(dst + d) = t;
        } else {
            *reinterpret_cast<f4*>(p.part_o + cell * p.dim + d) = o;
        }
    }
    if (!only && sub == 0) {
        p.part_ml[2 * cell] = mm;
        p.part_ml[2 * cell + 1] = total;
    }
}

// The parts of a row of a paged batch: a workgroup for a row and head.  LANES threads have a part's dims, four each, and 256 / LANES
// parts are added up side by side, those of each in their order, which makes the sums the same ones in every run.  Few bytes in
// a chain of loads that wait for each other (the batch, the length, the parts): what can be asked for early is.
// (47 parts for each of 64 rows of 128 dims: the call takes 17 us with both launches; 43 with a wave for a row that takes part after part.)
template <class T, int DIMS>
__global__ __launch_bounds__(256) void join_parts(const AttnParams p) {
    typedef Shape<T, DIMS> S;
    constexpr int LANES = DIMS == 32 ? 8 : DIMS == 64 ? 16 : DIMS <= 128 ? 32 : 64, SIDE = 256 / LANES;
    __shared__ f4 sums[256];
    const int lane = threadIdx.x & 63, cell = blockIdx.x, head = cell % p.heads, row = cell / p.heads;
    // the sequence whose rows this one is among: the one of that number where each has one new token
    const int* first = p.words.first;
    const int n = first[p.words.sequences + 1], guess = min(row, p.words.sequences - 1);
    const int guess_first = first[guess], guess_end = first[guess + 1], guess_seq = p.words.batch[guess];
    int end = guess_end, seq = guess_seq;
    if (n <= 0) return;
    if (guess >= n || row < guess_first || row >= guess_end) {
        if (row >= first[n]) return;
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= row) lo = mid;
            else hi = mid;
        }
        end = first[lo + 1];
        seq = p.words.batch[lo];
    }
    const int len = p.words.len[seq], pos = len - (end - row);
    // the parts that attend_steps made
    Sight see = sight_of(pos, len, p.causal, p.window, p.sinks);
    if (p.common) see.lo = p.common;
    const int a_steps = (see.first + S::STEP - 1) / S::STEP, b_first = max(see.lo / S::STEP, a_steps);
    const int steps = a_steps + max(0, (see.hi + S::STEP - 1) / S::STEP - b_first);
    const int most = p.parts - p.common_parts, chunk = max(p.chunk, (steps + most - 1) / most);
    if (steps <= chunk && !p.common) return;
    const int parts = p.common_parts + (steps + chunk - 1) / chunk;
    const float* ml = p.part_ml + 2 * (int64_t)cell * p.parts;
    const int d = (int)threadIdx.x % LANES * 4, side = (int)threadIdx.x / LANES;
    const float* from = p.part_o + (int64_t)cell * p.parts * p.dim + d;
    const bool has = d < p.dim;
    auto part = [&](int i) { return has && i < parts ? *reinterpret_cast<const f4*>(from + (int64_t)i * p.dim) : f4{0, 0, 0, 0}; };
    constexpr int AHEAD = 4;
    f4 ahead[AHEAD];
#pragma unroll
    for (int t = 0; t < AHEAD; t++) ahead[t] = part(side + t * SIDE);
    // (every wave has the maximum and the sum for itself)
    float m = kNone;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, ml[2 * i]);
    for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x));
    const float base = m == kNone ? 0.f : m;
    float total = 0;
    for (int i = lane; i < parts; i += 64) total += __builtin_amdgcn_exp2f(ml[2 * i] - base) * ml[2 * i + 1];
    for (int x = 1; x < 64; x *= 2) total += __shfl_xor(total, x);
    f4 o = {0, 0, 0, 0};
    for (int i = side; i < parts; i += AHEAD * SIDE) {
#pragma unroll
        for (int t = 0; t < AHEAD; t++) {
            if (i + t * SIDE < parts) {
                const float f = __builtin_amdgcn_exp2f(ml[2 * (i + t * SIDE)] - base);
                // (a part's infinity stays one, however little the part weighs; a part without weights has none)
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] += f == 0.f && __builtin_isinf(ahead[t][e]) ? ahead[t][e] : ahead[t][e] * f;
            }
            ahead[t] = part(i + (AHEAD + t) * SIDE);
        }
    }
    sums[threadIdx.x] = o;
    __syncthreads();
    if (side > 0 || !has) return;
    f4 all = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < SIDE; t++) all += sums[t * LANES + threadIdx.x];
    const float inv = total == 0.f ? 0.f : 1.f / total;
    typename Vec<T, 4>::type t;
#pragma unroll
    for (int e = 0; e < 4; e++) t[e] = (T)(all[e] * inv);
    *reinterpret_cast<typename Vec<T, 4>::type*>(reinterpret_cast<T*>(p.out.p) + (int64_t)row * p.out.tok + (int64_t)head * p.out.head + d) = t;
}

template <class T, int DIMS>
static hipError_t launch_steps(const AttnParams& p, unsigned blocks, hipStream_t s) {
    const auto kernel = !p.paged ? attend_steps<T, DIMS, false, true, false> : p.by_token ? attend_steps<T, DIMS, true, true, false>
                        : p.once ? attend_steps<T, DIMS, true, false, true> : attend_steps<T, DIMS, true, false, false>;
    const hipError_t e = start(kernel, blocks, s, p);
    return e != hipSuccess || p.parts <= 1 ? e : start(join_parts<T, DIMS>, (unsigned)(p.tokens * p.heads), s, p);
}

int attention_step(int f16, int dim) { return !f16 && dim > 128 ? 16 : 32; }

static int64_t steps_blocks(const AttnParams& p) {
    const int64_t across = p.by_token ? p.heads : p.kv_heads;
    return (across * (p.parts - p.common_parts) + 7) / 8 * 8 * (int64_t)p.tiles * p.batch + (across * p.common_parts + 7) / 8 * 8 * (int64_t)p.common_tiles;
}

static int launch_once(const AttnParams& p, int64_t blocks, hipStream_t s) {
    if (blocks <= 0) return 0;
    if (p.tiled) return p.f16 ? launch_tiles_f16(p, (unsigned)blocks, s) : launch_tiles_f32(p, (unsigned)blocks, s);
    hipError_t e;
#define FYN_ATTN(T, D) e = launch_steps<T, D>(p, (unsigned)blocks, s)
    if (p.f16) {
        if (p.dim <= 32) FYN_ATTN(_Float16, 32);
        else if (p.dim <= 64) FYN_ATTN(_Float16, 64);
        else if (p.dim <= 96) FYN_ATTN(_Float16, 96);
        else if (p.dim <= 128) FYN_ATTN(_Float16, 128);
        else FYN_ATTN(_Float16, 256);
    } else {
        if (p.dim <= 32) FYN_ATTN(float, 32);
        else if (p.dim <= 64) FYN_ATTN(float, 64);
        else if (p.dim <= 96) FYN_ATTN(float, 96);
        else if (p.dim <= 128) FYN_ATTN(float, 128);
        else FYN_ATTN(float, 256);
    }
#undef FYN_ATTN
    return e == hipSuccess ? 0 : -1;
}

int launch_attention(const AttnParams& p, hipStream_t s) {
    // A launch has fewer than 2^32 threads: the batch in pieces where it would have more.
    constexpr int64_t kMost = 0xffffff;
    auto blocks = [](const AttnParams& q) { return q.tiled ? ((int64_t)q.batch * q.heads + 7) / 8 * 8 * q.tiles : steps_blocks(q); };
    AttnParams q = p;
    while (q.batch > 1 && blocks(q) > kMost) q.batch = (q.batch + 1) / 2;
    if (blocks(q) > kMost || (q.batch < p.batch && p.parts > 1)) return -2;   // (rows in parts are few)
    for (const int each = q.batch; q.first_batch < p.batch; q.first_batch += each) {
        q.batch = std::min(each, p.batch - q.first_batch);
        const int rc = launch_once(q, blocks(q), s);
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace fynhip
