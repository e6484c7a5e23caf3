// Attention of many tokens: 128, 64 or 32 queries of one head a workgroup, keys and values in tiles through shared memory.
//
// Each of the four waves has 32 queries as columns.  Per piece of 64 or 32 keys
//     S^T [keys x queries]  = K Q^T          K from LDS, Q in registers for the whole run
//     O^T [dims x queries] += V^T P^T        V^T from LDS, P^T as S^T's registers hold it
// with the 32x32 matrix instructions.  Their result has the rows 8i + 4h + 0..3 (i = 0..3) in the lanes of half h, and the inner
// index of the second product is ordered by that, so that the weights go from one product to the next without leaving the
// lane.  Of a query everything, running maximum and sum too, is in two lanes.  With fewer than 128 queries two or four waves have the
// same ones, each takes another piece of the tile's keys, and their sums are joined at the end.
//
// The next tile's loads are under way while a tile is worked on, and go to the other half of the LDS behind it: one barrier a tile.
// Values in 16 bits are turned in registers on the way (eight keys by four dims a thread) so that a dim's keys lie side by
// side as the second product wants them.  Sixteen-byte pieces of rows are placed with their number xored with the row's, so
// that the sixteen lanes that read one piece of sixteen rows find them in different banks.
#include "attention_common.h"

namespace fynhip {

typedef float f16v __attribute__((ext_vector_type(16)));
constexpr float kLag = 8.f;   // binary orders of magnitude
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

template <class T, int DIMS, int QW>
struct TileShape {
    static constexpr bool F16 = std::is_same<T, _Float16>::value;
    static constexpr int KW = 4 / QW;                                            // waves with the same queries
    static constexpr int KEYS = F16 && DIMS <= 128 && QW == 4 ? 64 : 32;         // of a wave
    static constexpr int TILE = KEYS * KW;
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int PIECES = DIMS / VEC;                                    // of a row
    static constexpr int PITCH = PIECES <= 4 ? 4 : PIECES <= 8 ? 8 : PIECES <= 16 ? 16 : 32;   // ... in LDS
    static constexpr int SPREAD = PITCH < 16 ? PITCH : 16;                       // pieces among which a row's are exchanged
    static constexpr int SHARE = 16 / SPREAD;                                    // rows side by side in 256 bytes
    static constexpr int LOADS = (TILE * PITCH + 255) / 256;                     // of a thread, for the keys
    static constexpr int QUADS = DIMS / 4, GROUPS = TILE / 8;
    static constexpr int TURNS = F16 ? (QUADS * GROUPS + 255) / 256 : LOADS;     // ... for the values
    static constexpr int K_BYTES = TILE * PITCH * 16, V_BYTES = F16 ? DIMS * TILE * 2 : K_BYTES;
    static constexpr int DIM_TILES = DIMS / 32, KEY_TILES = KEYS / 32;
    static constexpr int JOIN_BYTES = KW > 1 ? 4 * DIM_TILES * 4096 : 0;         // sums of four waves
    static constexpr int LDS = 2 * (K_BYTES + V_BYTES) > JOIN_BYTES ? 2 * (K_BYTES + V_BYTES) : JOIN_BYTES;
    static constexpr bool FITS = LDS + 2048 <= 160 * 1024;
    static constexpr int WAVES = DIMS <= (F16 ? 128 : 64) && LDS <= 64 * 1024 ? 2 : 1;   // workgroups that share a CU (their registers)
};

__device__ __forceinline__ int row_piece(int row, int piece, int pitch, int spread, int share) { return row * pitch + (piece ^ (row / share % spread)); }

// Place of the eight keys (group) of a dim.
template <int GROUPS>
__device__ __forceinline__ int dim_piece(int dim, int group) {
    if (GROUPS >= 16) return dim * GROUPS + (group ^ (dim & 15));
    if (GROUPS == 8) return dim * 8 + (group ^ ((dim >> 1 & 7) ^ (dim >> 4 & 1)));
    return dim * 4 + (group ^ ((dim >> 2 & 3) ^ (dim >> 4 & 1)));
}

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
    constexpr int QUERIES = 32 * QW, HALF = S::K_BYTES + S::V_BYTES;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, c = lane & 31, mates = wave / QW, queries = wave % QW;
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    __shared__ int odd_values[2][4];   // a wave found infinities or NaN among a tile's values

    // The last queries first: under a causal mask theirs are the longest runs.  Heads that share keys lie eight workgroups apart
    // where there are eight key heads, on one XCD and its L2.
    const int units = p.batch * p.heads, rounds = (units + 7) / 8, id = blockIdx.x;
    const int unit = id / 8 % rounds * 8 + id % 8, tile = p.tiles - 1 - id / 8 / rounds;
    if (unit >= units) return;
    const int b = unit / p.heads, kv_head = unit % p.heads % p.kv_heads, head = kv_head * (p.heads / p.kv_heads) + unit % p.heads / p.kv_heads;
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

    u4 kreg[S::LOADS];
    u2 vreg[F16 ? S::TURNS : 1][F16 ? 8 : 1];
    u4 vreg32[F16 ? 1 : S::LOADS];
    // (Pieces behind a head's last value are taken from within it: in the first product they meet queries that are zero
    // there, in the second they end in dims that nobody stores.)
    const int k_piece = tid % S::PITCH, k_row = tid / S::PITCH, k_bytes = min(k_piece * 16, (p.dim - S::VEC) * (int)sizeof(T));
    auto v_quad = [&](int i) { return (tid + i * 256) % S::QUADS; };
    auto v_group = [&](int i) { return S::GROUPS * S::QUADS % 256 == 0 ? (tid + i * 256) / S::QUADS : min((tid + i * 256) / S::QUADS, S::GROUPS - 1); };
    auto v_bytes = [&](int i) { return min(v_quad(i) * 8, (p.dim - 4) * 2); };
    auto fetch = [&](int at) {
        if (!PAGED && at + S::TILE <= most) {
            // A thread's rows are a fixed distance from its first: one offset of 32 bits (the host has seen to that) to scalar bases.
            const char* kb = kbase + (int64_t)at * p.k.tok * (int64_t)sizeof(T);
            const char* vb = vbase + (int64_t)at * p.v.tok * (int64_t)sizeof(T);
            const unsigned k_off = (unsigned)(k_row * (int)p.k.tok * (int)sizeof(T) + k_bytes);
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) kreg[i] = *reinterpret_cast<const u4*>(kb + (int64_t)i * (256 / S::PITCH) * p.k.tok * (int64_t)sizeof(T) + k_off);
            if constexpr (F16) {
#pragma unroll
                for (int i = 0; i < S::TURNS; i++) {
                    const int g = v_group(i);
                    const unsigned v_off = (unsigned)((g / 2 * 16 + g % 2 * 4) * (int)p.v.tok * 2 + v_bytes(i));
#pragma unroll
                    for (int e = 0; e < 8; e++) vreg[i][e] = *reinterpret_cast<const u2*>(vb + (int64_t)(e / 4 * 8 + e % 4) * p.v.tok * 2 + v_off);
                }
            } else {
                const unsigned v_off = (unsigned)(k_row * (int)p.v.tok * (int)sizeof(T) + k_bytes);
#pragma unroll
                for (int i = 0; i < S::LOADS; i++) vreg32[i] = *reinterpret_cast<const u4*>(vb + (int64_t)i * (256 / S::PITCH) * p.v.tok * (int64_t)sizeof(T) + v_off);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) kreg[i] = *reinterpret_cast<const u4*>(row(kbase, p.k.tok, at, k_row + i * (256 / S::PITCH), k_bytes));
        if constexpr (F16) {
#pragma unroll
            for (int i = 0; i < S::TURNS; i++) {
                const int g = v_group(i);
#pragma unroll
                for (int e = 0; e < 8; e++) vreg[i][e] = *reinterpret_cast<const u2*>(row(vbase, p.v.tok, at, g / 2 * 16 + e / 4 * 8 + g % 2 * 4 + e % 4, v_bytes(i)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) vreg32[i] = *reinterpret_cast<const u4*>(row(vbase, p.v.tok, at, k_row + i * (256 / S::PITCH), k_bytes));
        }
    };
    // `partial`: not all of the workgroup's queries see all of the tile.  Infinities and NaN among its values are left out then,
    // and those who see them are told.
    auto place = [&](int buf, bool partial) {
        u4* kl = reinterpret_cast<u4*>(lds + buf * HALF);
        u4* vl = reinterpret_cast<u4*>(lds + buf * HALF + S::K_BYTES);
#pragma unroll
        for (int i = 0; i < S::LOADS; i++) {
            const int r = k_row + i * (256 / S::PITCH);
            if (r < S::TILE) kl[row_piece(r, k_piece, S::PITCH, S::SPREAD, S::SHARE)] = kreg[i];
        }
        if (partial) {
            bool found = false;
            if constexpr (F16) {
#pragma unroll
                for (int i = 0; i < S::TURNS; i++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const unsigned x = vreg[i][e / 2][e % 2], odd = ((x & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;   // (an exponent of all ones carries into the sign's place)
                        found = found || odd;
                        vreg[i][e / 2][e % 2] = x & ~((odd << 1) - (odd >> 15));
                    }
            } else {
#pragma unroll
                for (int i = 0; i < S::LOADS; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const unsigned x = vreg32[i][e];
                        const bool odd = (x & 0x7f800000u) == 0x7f800000u;
                        found = found || odd;
                        vreg32[i][e] = odd ? 0 : x;
                    }
            }
            found = __any(found);
            if (lane == 0) odd_values[buf][wave] = found;
        }
        if constexpr (F16) {
#pragma unroll
            for (int i = 0; i < S::TURNS; i++) {
                const int quad = v_quad(i), g = (tid + i * 256) / S::QUADS;
                if (g < S::GROUPS)
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        u4 t;
#pragma unroll
                        for (int e = 0; e < 4; e++) t[e] = __builtin_amdgcn_perm(vreg[i][2 * e + 1][d / 2], vreg[i][2 * e][d / 2], d % 2 ? 0x07060302u : 0x05040100u);
                        vl[dim_piece<S::GROUPS>(quad * 4 + d, g)] = t;
                    }
            }
        } else {
#pragma unroll
            for (int i = 0; i < S::LOADS; i++) {
                const int r = k_row + i * (256 / S::PITCH);
                if (r < S::TILE) vl[row_piece(r, k_piece, S::PITCH, S::SPREAD, S::SHARE)] = vreg32[i];
            }
        }
    };
    auto is_partial = [&](int at) { return !((at >= whole.lo && at + S::TILE <= whole.hi) || at + S::TILE <= whole.first); };

    f16v acc[S::DIM_TILES];
#pragma unroll
    for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[d][r] = 0.f;
    float m = kNone, l = 0;   // (l: of this lane's keys only)

    if (steps > 0) {
        fetch(at_of(0));
        place(0, is_partial(at_of(0)));
    }
    for (int st = 0; st < steps; st++) {
        const int from = at_of(st), buf = st & 1, at = from + mates * S::KEYS;   // (the wave's piece)
        __syncthreads();   // the tile is in LDS, and nobody reads the other half any more
        if (st + 1 < steps) fetch(at_of(st + 1));
        if ((at < any.hi && at + S::KEYS > any.lo) || at < any.first) {
            const char* kl = lds + buf * HALF;
            const char* vl = kl + S::K_BYTES;
            f16v sc[S::KEY_TILES];
#pragma unroll
            for (int t = 0; t < S::KEY_TILES; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) sc[t][r] = 0.f;
#pragma unroll
            for (int s = 0; s < S::PIECES / 2; s++) {
#pragma unroll
                for (int t = 0; t < S::KEY_TILES; t++) {
                    const KVec k = *reinterpret_cast<const KVec*>(kl + 16 * row_piece(mates * S::KEYS + 32 * t + c, 2 * s + half, S::PITCH, S::SPREAD, S::SHARE));
                    if constexpr (F16) {
                        sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[s], sc[t], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[s][e], sc[t], 0, 0, 0);
                    }
                }
            }
            if (!((at >= all.lo && at + S::KEYS <= all.hi) || at + S::KEYS <= all.first)) {
#pragma unroll
                for (int t = 0; t < S::KEY_TILES; t++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (!mine.sees(at + 32 * t + (r & 3) + 8 * (r >> 2) + 4 * half)) sc[t][r] = kNone;
            }
            float top = kNone;
#pragma unroll
            for (int t = 0; t < S::KEY_TILES; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, sc[t][r]);
            top = across(top) * scale;
            // The sums are relative to a maximum that may be the true one's 2^-8 (with weights up to 2^14 then): it follows where a
            // query is further off, which after the first tiles is seldom.
            if (__any(top > m + kLag)) {
                const float m_new = top > m + kLag ? top : m, alpha = m == kNone ? 0.f : __builtin_amdgcn_exp2f(m - m_new);   // (by each query alone)
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[d][r] *= alpha;
            }
            // Weights 2^6 times as large as relative to m: 16 bits hold them to full precision down to 2^-20 of it.
            // They are rounded to 16 bits for the second product, and it is the rounded ones that are summed up.
            const float base = m == kNone ? 0.f : m - 6.f;
#pragma unroll
            for (int t = 0; t < S::KEY_TILES; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) sc[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][r], scale, -base));
            if constexpr (F16) {
                h8 w[2 * S::KEY_TILES];
#pragma unroll
                for (int t = 0; t < 2 * S::KEY_TILES; t++)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const h2 two = {(_Float16)sc[t / 2][t % 2 * 8 + e], (_Float16)sc[t / 2][t % 2 * 8 + e + 1]};
                        l = __builtin_amdgcn_fdot2(two, h2{(_Float16)1, (_Float16)1}, l, false);
                        w[t][e] = two[0];
                        w[t][e + 1] = two[1];
                    }
#pragma unroll
                for (int t = 0; t < 2 * S::KEY_TILES; t++)
#pragma unroll
                    for (int d = 0; d < S::DIM_TILES; d++) {
                        const h8 v = *reinterpret_cast<const h8*>(vl + 16 * dim_piece<S::GROUPS>(32 * d + c, mates * (S::KEYS / 8) + 2 * t + half));
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w[t], acc[d], 0, 0, 0);
                    }
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) l += sc[0][r];
#pragma unroll
                for (int r = 0; r < 16; r++)
#pragma unroll
                    for (int d = 0; d < S::DIM_TILES; d++) {
                        const int key = mates * S::KEYS + (r & 3) + 8 * (r >> 2) + 4 * half, dim = 32 * d + c;
                        const float v = *reinterpret_cast<const float*>(vl + 16 * row_piece(key, dim / 4, S::PITCH, S::SPREAD, S::SHARE) + dim % 4 * 4);
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[0][r], acc[d], 0, 0, 0);
                    }
            }
            // Values that were left out: whoever sees them has them in the result (a weight is never negative).
            if (is_partial(from) && (odd_values[buf][0] | odd_values[buf][1] | odd_values[buf][2] | odd_values[buf][3])) {
                for (int key = 0; key < S::KEYS; key++) {
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
        if (st + 1 < steps) place(buf ^ 1, is_partial(at_of(st + 1)));
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
        float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int d = 0; d < S::DIM_TILES; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) sums[((wave * S::DIM_TILES + d) * 16 + r) * 64 + lane] = acc[d][r] * f;
        __syncthreads();
#pragma unroll
        for (int d = 0; d < S::DIM_TILES; d++)
            if (d % S::KW == mates)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    float sum = 0;
#pragma unroll
                    for (int k = 0; k < S::KW; k++) sum += sums[(((k * QW + queries) * S::DIM_TILES + d) * 16 + r) * 64 + lane];
                    acc[d][r] = sum;
                }
        l = total;
    }
    if (tok >= in.count) return;
    const bool zero = tok >= seen_rows;
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
            if (dim < p.dim) *reinterpret_cast<typename Vec<T, 4>::type*>(dst + dim) = t;
        }
    }
}

template <class T, int DIMS, int QW>
static bool launch_tiles(const AttnParams& p, unsigned blocks, hipStream_t s) {
    if constexpr (TileShape<T, DIMS, QW>::FITS) {
        if (p.paged) hipLaunchKernelGGL((attend_tiles<T, DIMS, true, QW>), dim3(blocks), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((attend_tiles<T, DIMS, false, QW>), dim3(blocks), dim3(256), 0, s, p);
        return true;
    }
    return false;
}

#if FYN_ATTN_HALF
typedef _Float16 Stored;
#define FYN_ATTN_NAME launch_tiles_f16
#define FYN_ATTN_FITS tiles_fit_f16
#else
typedef float Stored;
#define FYN_ATTN_NAME launch_tiles_f32
#define FYN_ATTN_FITS tiles_fit_f32
#endif

template <int QW>
static int launch_class(const AttnParams& p, hipStream_t s) {
    const int64_t blocks = ((int64_t)p.batch * p.heads + 7) / 8 * 8 * p.tiles;
    if (blocks <= 0) return 0;
    if (blocks > 0x7fffffff) return -1;
    bool done = false;
    if (p.dim <= 32) done = launch_tiles<Stored, 32, QW>(p, (unsigned)blocks, s);
    else if (p.dim <= 64) done = launch_tiles<Stored, 64, QW>(p, (unsigned)blocks, s);
    else if (p.dim <= 96) done = launch_tiles<Stored, 96, QW>(p, (unsigned)blocks, s);
    else if (p.dim <= 128) done = launch_tiles<Stored, 128, QW>(p, (unsigned)blocks, s);
#if FYN_ATTN_HALF
    else done = launch_tiles<Stored, 256, QW>(p, (unsigned)blocks, s);
#endif
    return done && hipGetLastError() == hipSuccess ? 0 : -1;
}

int FYN_ATTN_NAME(const AttnParams& p, hipStream_t s) {
    return p.tiled == 128 ? launch_class<4>(p, s) : p.tiled == 64 ? launch_class<2>(p, s) : launch_class<1>(p, s);
}

template <int QW>
static bool fits(int dim) {
    if (dim <= 32) return TileShape<Stored, 32, QW>::FITS;
    if (dim <= 64) return TileShape<Stored, 64, QW>::FITS;
    if (dim <= 96) return TileShape<Stored, 96, QW>::FITS;
    if (dim <= 128) return TileShape<Stored, 128, QW>::FITS;
#if FYN_ATTN_HALF
    return TileShape<Stored, 256, QW>::FITS;
#else
    return false;   // (queries and sums of 32 bits: more registers than a wave has)
#endif
}

bool FYN_ATTN_FITS(int dim, int queries) { return queries == 128 ? fits<4>(dim) : queries == 64 ? fits<2>(dim) : fits<1>(dim); }

}  // namespace fynhip
