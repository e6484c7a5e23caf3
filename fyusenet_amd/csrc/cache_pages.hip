// The pages of a cache of keys and values: the words that say where they are, copies of pages, and tokens between pages and
// tensors.  All of it is bound by memory; nothing is computed.
#include "sequence.h"

namespace fynhip {

typedef unsigned u4 __attribute__((ext_vector_type(4)));

template <int WORDS>
struct ChangeArgument {
    int update, lists, moves, source, entries;
    int w[WORDS];
};

// One launch for all that a call changes.  Workgroup 0 writes the words, the next ones the lists, the others copy pages, each a
// part of one: 16 KB, four vectors of 16 bytes a thread.
constexpr int kPart = 16 << 10;
template <int WORDS>
__global__ __launch_bounds__(256) void change_cache(const CacheMemory m, const ChangeArgument<WORDS> c, const int parts) {
    int b = blockIdx.x;
    if (b == 0) {
        for (int i = 0; i < c.update;) {
            const int at = c.w[i], n = c.w[i + 1];
            for (int k = threadIdx.x; k < n; k += 256) m.words[at + k] = c.w[i + 2 + k];
            i += 2 + n;
        }
        return;
    }
    b -= 1;
    if (b < c.lists) {
        const int* src = m.table + (int64_t)c.source * m.pitch;
        int* dst = m.table + (int64_t)c.w[c.update + b] * m.pitch;
        for (int i = threadIdx.x; i < c.entries; i += 256) dst[i] = src[i];
        return;
    }
    b -= c.lists;
    const int pair = b / parts;
    const int64_t at = (int64_t)(b % parts) * kPart;
    const char* src = m.pool + c.w[c.update + c.lists + 2 * pair] * m.page_bytes + at;
    char* dst = m.pool + c.w[c.update + c.lists + 2 * pair + 1] * m.page_bytes + at;
    const int64_t left = m.page_bytes - at;
    u4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if ((i * 256 + threadIdx.x) * 16 < left) v[i] = *reinterpret_cast<const u4*>(src + (i * 256 + threadIdx.x) * 16);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if ((i * 256 + threadIdx.x) * 16 < left) *reinterpret_cast<u4*>(dst + (i * 256 + threadIdx.x) * 16) = v[i];
}

template <int WORDS>
static void launch_change(const CacheMemory& m, const CacheChange& c, hipStream_t s) {
    ChangeArgument<WORDS> a;
    a.update = c.update; a.lists = c.lists; a.moves = c.moves; a.source = c.source; a.entries = c.entries;
    const int n = c.update + c.lists + 2 * c.moves;
    for (int i = 0; i < n; i++) a.w[i] = c.w[i];
    const int64_t parts = (m.page_bytes + kPart - 1) / kPart;
    hipLaunchKernelGGL(change_cache<WORDS>, dim3((unsigned)(1 + c.lists + c.moves * parts)), dim3(256), 0, s, m, a, (int)parts);
}

void launch_cache_change(const CacheMemory& m, const CacheChange& c, hipStream_t s) {
    const int n = c.update + c.lists + 2 * c.moves;
    if (n <= 48) launch_change<48>(m, c, s);
    else launch_change<kChangeWords>(m, c, s);
}

// where the head's keys of a token of a sequence are
__device__ __forceinline__ char* token_at(const CacheRows& p, int seq, int pos, int head, int size) {
    const int page = p.words.table[(int64_t)seq * p.words.table_pitch + (pos >> p.pages.shift)];
    return p.pages.pool + page * p.pages.page_bytes + head * p.pages.head_bytes + (int64_t)(pos & ((1 << p.pages.shift) - 1)) * p.dim * size;
}

// A thread moves 16 bytes of a key and of its value.  Threads run over vectors of a head, heads, tokens.
__global__ __launch_bounds__(256) void write_tokens(const CacheRows p) {
    const int size = p.f16 ? 2 : 4, vecs = p.dim * size / 16;
    const int64_t n = (int64_t)p.rows * p.kv_heads * vecs;
    const int batch = p.words.first[p.words.sequences + 1];
    if (batch <= 0) return;
    const int rows = min(p.rows, p.words.first[batch]);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int vec = (int)(i % vecs), head = (int)(i / vecs % p.kv_heads), row = (int)(i / ((int64_t)vecs * p.kv_heads));
        if (row >= rows) return;
        int lo = 0, hi = batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.words.first[mid] <= row) lo = mid;
            else hi = mid;
        }
        const int seq = p.words.batch[lo], pos = p.words.len[seq] - (p.words.first[lo + 1] - row);
        char* dst = token_at(p, seq, pos, head, size) + vec * 16;
        *reinterpret_cast<u4*>(dst) = *reinterpret_cast<const u4*>(p.k.p + (row * p.k.tok + head * p.k.head) * size + vec * 16);
        *reinterpret_cast<u4*>(dst + p.pages.values) = *reinterpret_cast<const u4*>(p.v.p + (row * p.v.tok + head * p.v.head) * size + vec * 16);
    }
}

static unsigned blocks_for(const CacheRows& p) {
    const int64_t n = ((int64_t)p.rows * p.kv_heads * (p.dim * (p.f16 ? 2 : 4) / 16) + 255) / 256;
    return (unsigned)(n > 8192 ? 8192 : n);
}

void launch_cache_write(const CacheRows& p, hipStream_t s) {
    if (p.rows > 0) hipLaunchKernelGGL(write_tokens, dim3(blocks_for(p)), dim3(256), 0, s, p);
}

__global__ __launch_bounds__(256) void read_tokens(const CacheRows p, const CacheRead r) {
    const int size = p.f16 ? 2 : 4, vecs = p.dim * size / 16;
    const int64_t n = (int64_t)p.rows * p.kv_heads * vecs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int vec = (int)(i % vecs), head = (int)(i / vecs % p.kv_heads), row = (int)(i / ((int64_t)vecs * p.kv_heads));
        int lo = 0, hi = r.n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (r.first[mid] <= row) lo = mid;
            else hi = mid;
        }
        const char* src = token_at(p, r.sequence[lo], row - r.first[lo], head, size) + vec * 16;
        *reinterpret_cast<u4*>(p.k.p + (row * p.k.tok + head * p.k.head) * size + vec * 16) = *reinterpret_cast<const u4*>(src);
        *reinterpret_cast<u4*>(p.v.p + (row * p.v.tok + head * p.v.head) * size + vec * 16) = *reinterpret_cast<const u4*>(src + p.pages.values);
    }
}

void launch_cache_read(const CacheRows& p, const CacheRead& r, hipStream_t s) {
    if (p.rows > 0) hipLaunchKernelGGL(read_tokens, dim3(blocks_for(p)), dim3(256), 0, s, p, r);
}

}  // namespace fynhip
