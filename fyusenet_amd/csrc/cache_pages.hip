// The pages of a cache of keys and values: the words that say where they are, copies of pages, and tokens between pages and
// tensors.  All of it is bound by memory; nothing is computed.  Copies of pages run at 6.1 TB/s read and written together (480 pages
// of 512 KB: 83 us), reading tokens into tensors at 4.9 (885 MB each way: 358 us: a look-up in the list for every 16 bytes); few
// pages or tokens take the time of a launch, 2 to 5 us.
#include "sequence.h"

#include <algorithm>

namespace fynhip {

typedef unsigned u4 __attribute__((ext_vector_type(4)));

template <int WORDS>
struct ChangeArgument {
    int runs, singles, lists, moves, source, entries;
    int w[WORDS];
};

// One launch for all that a call changes.  Workgroup 0 writes the words, the next ones the lists, the others copy pages, each a
// part of one: 16 KB, four vectors of 16 bytes a thread.
constexpr int kPart = 16 << 10;
template <int WORDS>
__global__ __launch_bounds__(256) void change_cache(const CacheMemory m, const ChangeArgument<WORDS> c, const int parts) {
    int b = blockIdx.x;
    if (b == 0) {
        for (int i = threadIdx.x; i < c.singles; i += 256) m.words[c.w[c.runs + 2 * i]] = c.w[c.runs + 2 * i + 1];
        for (int i = 0; i < c.runs;) {
            const int at = c.w[i], n = c.w[i + 1];
            for (int k = threadIdx.x; k < n; k += 256) m.words[at + k] = c.w[i + 2 + k];
            i += 2 + n;
        }
        return;
    }
    b -= 1;
    const int lists = c.runs + 2 * c.singles;
    if (b < c.lists) {
        const int* src = m.table + (int64_t)c.source * m.pitch;
        int* dst = m.table + (int64_t)c.w[lists + b] * m.pitch;
        for (int i = threadIdx.x; i < c.entries; i += 256) dst[i] = src[i];
        return;
    }
    b -= c.lists;
    const int pair = b / parts;
    const int64_t at = (int64_t)(b % parts) * kPart;
    const int moves = lists + c.lists;
    const char* src = m.pool + c.w[moves + 2 * pair] * m.page_bytes + at;
    char* dst = m.pool + c.w[moves + 2 * pair + 1] * m.page_bytes + at;
    const int64_t left = m.page_bytes - at;
    u4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if ((i * 256 + threadIdx.x) * 16 < left) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(src + (i * 256 + threadIdx.x) * 16));
#pragma unroll
    for (int i = 0; i < 4; i++)
        if ((i * 256 + threadIdx.x) * 16 < left) __builtin_nontemporal_store(v[i], reinterpret_cast<u4*>(dst + (i * 256 + threadIdx.x) * 16));
}

template <int WORDS>
static hipError_t launch_change(const CacheMemory& m, const CacheChange& c, hipStream_t s) {
    ChangeArgument<WORDS> a;
    a.runs = c.runs; a.singles = c.singles; a.lists = c.lists; a.moves = c.moves; a.source = c.source; a.entries = c.entries;
    for (int i = 0; i < c.used(); i++) a.w[i] = c.w[i];
    const int64_t parts = (m.page_bytes + kPart - 1) / kPart;
    return start(change_cache<WORDS>, (unsigned)(1 + c.lists + c.moves * parts), s, m, a, (int)parts);
}

hipError_t launch_cache_change(const CacheMemory& m, const CacheChange& c, hipStream_t s) {
    return c.used() <= 48 ? launch_change<48>(m, c, s) : c.used() <= 240 ? launch_change<240>(m, c, s) : launch_change<kChangeWords>(m, c, s);
}

// where the head's keys of a token of a sequence are
__device__ __forceinline__ char* token_at(const CacheRows& p, int seq, int pos, int head, int size) {
    const int page = p.words.table[(int64_t)seq * p.words.table_pitch + (pos >> p.pages.shift)];
    return p.pages.pool + page * p.pages.page_bytes + head * p.pages.head_bytes + (int64_t)(pos & ((1 << p.pages.shift) - 1)) * p.dim * size;
}

// A thread moves 16 bytes of a key and of its value.  Threads run over vectors of a head, heads, tokens; a launch has fewer than
// 2^31 of them (the host divides what is more).  What is read is not read again: it does not stay in the caches.
struct Item {
    int vec, head, row;
    bool any;
};
__device__ __forceinline__ Item item_of(const CacheRows& p, int vecs) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x, row_head = i / vecs;
    return Item{(int)(i - row_head * vecs), (int)(row_head % p.kv_heads), (int)(row_head / p.kv_heads), row_head / p.kv_heads < (unsigned)p.rows};
}

// The entry of first[0 .. n-1], which ascend, that `row` belongs to.
__device__ __forceinline__ int find(const int* first, int n, int row) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(256) void write_tokens(const CacheRows p, const int from) {
    const int size = p.f16 ? 2 : 4;
    const Item it = item_of(p, p.dim * size / 16);
    const int batch = p.words.first[p.words.sequences + 1], row = from + it.row;
    if (!it.any || batch <= 0 || row >= p.words.first[batch]) return;
    const u4 k = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p.k.p + (it.row * p.k.tok + it.head * p.k.head) * size + it.vec * 16));
    const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p.v.p + (it.row * p.v.tok + it.head * p.v.head) * size + it.vec * 16));
    const int b = find(p.words.first, batch, row), seq = p.words.batch[b], pos = p.words.len[seq] - (p.words.first[b + 1] - row);
    char* dst = token_at(p, seq, pos, it.head, size) + it.vec * 16;
    *reinterpret_cast<u4*>(dst) = k;
    *reinterpret_cast<u4*>(dst + p.pages.values) = v;
}

__global__ __launch_bounds__(256) void read_tokens(const CacheRows p, const CacheRead r, const int from) {
    const int size = p.f16 ? 2 : 4;
    const Item it = item_of(p, p.dim * size / 16);
    if (!it.any) return;
    const int row = from + it.row, b = find(r.first, r.n, row);
    const char* src = token_at(p, r.sequence[b], row - r.first[b], it.head, size) + it.vec * 16;
    const u4 k = __builtin_nontemporal_load(reinterpret_cast<const u4*>(src));
    const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(src + p.pages.values));
    __builtin_nontemporal_store(k, reinterpret_cast<u4*>(p.k.p + (it.row * p.k.tok + it.head * p.k.head) * size + it.vec * 16));
    __builtin_nontemporal_store(v, reinterpret_cast<u4*>(p.v.p + (it.row * p.v.tok + it.head * p.v.head) * size + it.vec * 16));
}

// Launches over rows from, from + 1, ..: as many at once as 32 bits count.
template <class F>
static hipError_t over_rows(CacheRows p, F&& launch) {
    const int size = p.f16 ? 2 : 4;
    const int64_t each = (int64_t)p.kv_heads * (p.dim * size / 16), most = std::max<int64_t>(1, 0x7f000000 / each);
    const int rows = p.rows;
    hipError_t e = hipSuccess;
    for (int64_t from = 0; from < rows && e == hipSuccess; from += most) {
        p.rows = (int)std::min<int64_t>(most, rows - from);
        e = launch(p, (unsigned)((p.rows * each + 255) / 256), (int)from);
        p.k.p += p.rows * p.k.tok * size;
        p.v.p += p.rows * p.v.tok * size;
    }
    return e;
}

hipError_t launch_cache_write(const CacheRows& p, hipStream_t s) {
    return over_rows(p, [&](const CacheRows& q, unsigned blocks, int from) { return start(write_tokens, blocks, s, q, from); });
}

hipError_t launch_cache_read(const CacheRows& p, const CacheRead& r, hipStream_t s) {
    return over_rows(p, [&](const CacheRows& q, unsigned blocks, int from) { return start(read_tokens, blocks, s, q, r, from); });
}

}  // namespace fynhip
