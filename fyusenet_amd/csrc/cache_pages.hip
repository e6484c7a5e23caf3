// The pages of a cache of keys and values: the words that say where they are, copies of pages, and tokens between pages and
// tensors.  All of it is bound by memory; nothing is computed.
#include "sequence.h"

namespace fynhip {

typedef unsigned u4 __attribute__((ext_vector_type(4)));

// Changed words travel as the launch's argument: no host memory has to outlive the call, and nothing is copied between
// host and device on the way.
__global__ __launch_bounds__(256) void update_words(int* __restrict__ words, const CacheUpdate u) {
    for (int i = 0; i < u.n;) {
        const int at = u.w[i], n = u.w[i + 1];
        for (int k = threadIdx.x; k < n; k += 256) words[at + k] = u.w[i + 2 + k];
        i += 2 + n;
    }
}

void launch_cache_update(int* words, const CacheUpdate& u, hipStream_t s) {
    hipLaunchKernelGGL(update_words, dim3(1), dim3(256), 0, s, words, u);
}

__global__ __launch_bounds__(256) void copy_rows(int* __restrict__ table, int pitch, int from, const RowCopies r) {
    const int* src = table + (int64_t)from * pitch;
    int* dst = table + (int64_t)r.to[blockIdx.y] * pitch;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < r.words; i += gridDim.x * 256) dst[i] = src[i];
}

void launch_row_copies(int* table, int pitch, int from, const RowCopies& r, hipStream_t s) {
    const unsigned x = (unsigned)min((r.words + 255) / 256, 64);
    hipLaunchKernelGGL(copy_rows, dim3(x, (unsigned)r.n), dim3(256), 0, s, table, pitch, from, r);
}

__global__ __launch_bounds__(256) void copy_pages(char* __restrict__ pool, int64_t page_bytes, const PageCopies c) {
    const u4* src = reinterpret_cast<const u4*>(pool + c.from[blockIdx.y] * page_bytes);
    u4* dst = reinterpret_cast<u4*>(pool + c.to[blockIdx.y] * page_bytes);
    const int64_t n = page_bytes / 16;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) dst[i] = src[i];
}

void launch_page_copies(char* pool, int64_t page_bytes, const PageCopies& c, hipStream_t s) {
    const int64_t x = (page_bytes / 16 + 1023) / 1024;   // four vectors a thread
    hipLaunchKernelGGL(copy_pages, dim3((unsigned)(x < 1 ? 1 : x > 256 ? 256 : x), (unsigned)c.n), dim3(256), 0, s, pool, page_bytes, c);
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
