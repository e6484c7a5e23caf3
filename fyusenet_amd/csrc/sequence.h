// Parameter blocks and host-side launchers of the kernels on sequences: attention (attention.hip) and the pages of a cache
// of keys and values (cache_pages.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>

namespace fynhip {

constexpr int kMaxHeadDim = 256;

// One launch, with its own result.  (The thread's last error may be that of an earlier call of somebody else's, and stays what it is.)
template <class... P, class... A>
inline hipError_t start(void (*kernel)(P...), unsigned blocks, hipStream_t s, const A&... a) {
    std::tuple<P...> given(a...);
    return std::apply([&](auto&... x) {
        void* at[] = {const_cast<void*>(static_cast<const void*>(&x))...};
        const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3(256), at, 0, s);
        if (e != hipSuccess) (void)hipGetLastError();
        return e;
    }, given);
}

// Rows of a tensor [sequence, token, head, dim], distances in elements; dim is dense.
struct SeqRows {
    char* p;
    int64_t seq, tok, head;
};

// Where a cache keeps its int32 words on the device (page_book.h writes them): tokens of each sequence, the sequences of
// the current batch, the rows at which their new tokens begin (one more than there are sequences), and the lists of pages.
struct CacheWords {
    const int* len;
    const int* batch;
    const int* first;
    const int* table;
    int table_pitch;   // entries per sequence
    int sequences;     // entries of batch; `first` has one more, and the number of sequences in the batch stands behind it
};

// Pages: [page][layer][keys or values][kv head][token][dim].
struct PageLayout {
    char* pool;             // (with the offset of the layer)
    int64_t page_bytes;     // all layers
    int64_t values;         // bytes from a head's keys to its values
    int64_t head_bytes;
    int shift;              // log2 of the tokens of a page
};

struct AttnParams {
    SeqRows q, k, v, out;   // (k, v: where nothing is paged)
    PageLayout pages;
    CacheWords words;
    const int* lengths;     // nothing paged: tokens of each sequence, or null
    int paged, f16;
    int first_batch;        // of one launch: the sequences [first_batch, first_batch + batch) of the batch
    int batch, tokens;      // nothing paged: rows of each sequence; paged: rows of q in all
    int heads, kv_heads, dim;
    int causal, window, sinks;
    float scale_log2;       // softmax scale times log2(e)
    // rows of one launch
    int tiled;              // attention_tiles.hip: tokens of a head that a workgroup has (128 or 64), or 0: attention.hip
    int by_token;           // a workgroup's columns: 1 sixteen tokens of a head, 0 one token and up to sixteen heads of a group
    int tiles;              // column tiles per sequence and (by_token) head or (else) key head
    // the long axis in parts
    int once;               // no key is read by two workgroups
    int chunk;              // key steps of one part
    int parts;              // most parts of a row
    // Sequences that begin with the same `common` tokens (a multiple of 32, in the same pages), one new token each: columns are heads
    // of all of them over those tokens, divided into the first `common_parts` of each row's parts.
    int common, common_parts, common_chunk, common_tiles;
    float* part_o;          // [row * heads + head][part][dim]
    float* part_ml;         // ... [2]: maximum and sum
};

// 0, -1 where a launch failed, -2 where one sequence would have more workgroups than a launch can.
int launch_attention(const AttnParams& p, hipStream_t s);
int launch_tiles_f16(const AttnParams& p, unsigned blocks, hipStream_t s);   // (called by it)
int launch_tiles_f32(const AttnParams& p, unsigned blocks, hipStream_t s);   // ... up to 128 dims
int attention_step(int f16, int dim);   // keys of one step of the kernel (AttnParams::chunk counts them)

// What the host changes of a cache in one launch.  It travels as the kernel's argument (at most 4 KB, and 256 bytes where it is
// little: the argument's size is part of a launch's time): no memory of the host's has to outlive the call.
// Runs of words {first word, number of words, words ...} ...; single words; lists of pages that become copies of another's first
// entries; pages that are copied.  They stand one kind behind the other in w.
constexpr int kChangeWords = 960;
struct CacheChange {
    int runs;               // words that the runs take
    int singles;            // {word, value}
    int lists;              // sequences whose lists become copies of the first `entries` of `source`'s
    int moves;              // {from, to}
    int source, entries;
    int w[kChangeWords];
    int used() const { return runs + 2 * singles + lists + 2 * moves; }
};
struct CacheMemory {
    int* words;
    int* table;
    int pitch;
    char* pool;
    int64_t page_bytes;
};
hipError_t launch_cache_change(const CacheMemory& m, const CacheChange& c, hipStream_t s);

struct CacheRows {          // tokens between a cache and tensors
    SeqRows k, v;
    PageLayout pages;
    CacheWords words;
    int rows, kv_heads, dim, f16;
};
hipError_t launch_cache_write(const CacheRows& p, hipStream_t s);
constexpr int kReadSequences = 400;
struct CacheRead {
    int n;
    int sequence[kReadSequences], first[kReadSequences + 1];   // rows of the tensors, of this launch
};
hipError_t launch_cache_read(const CacheRows& p, const CacheRead& r, hipStream_t s);

}  // namespace fynhip
