// A cache of keys and values in pages, and attention over it (fyn_cache_* of the C ABI).
#pragma once
#include <memory>
#include <mutex>

#include "engine.h"
#include "page_book.h"
#include "sequence.h"

namespace fynhip {

class Cache : public std::enable_shared_from_this<Cache> {
  public:
    Cache(int device, const fyn_cache_desc& d);
    ~Cache();
    void extend(int n, const int* seqs, const int* counts, hipStream_t s);
    void write(int layer, const fyn_rows& k, const fyn_rows& v, int rows, hipStream_t s);
    void attend(int layer, const fyn_attend_desc& a, hipStream_t s);
    void read(int n, const int* seqs, int layer, const fyn_rows& k, const fyn_rows& v, int rows, hipStream_t s);
    void fork(int source, int n, const int* targets, int tokens, hipStream_t s);
    void copy(int n, const int* sources, const int* targets, hipStream_t s);
    void truncate(int n, const int* seqs, const int* tokens, hipStream_t s);
    void compact(int* used, hipStream_t s);
    void lengths(int n, const int* seqs, int* tokens);
    void pages(int* used, int* free);
    // A pass over the batch follows on this stream, for so many new tokens.  -> the rows at which its sequences begin
    std::vector<int> expect(int rows, hipStream_t s);
    void order(hipStream_t s);   // what has been queued on the stream that the cache was used on last comes before what follows on this one

    const int device;
    const fyn_cache_desc d;
    void check_layer(int layer) const { (void)layout(layer); }

  private:
    std::mutex mu_;
    PageBook book_;
    char* pool_ = nullptr;
    int* words_ = nullptr;
    float* parts_ = nullptr;
    int64_t part_cells_ = 0;
    int64_t head_bytes_ = 0, layer_bytes_ = 0, page_bytes_ = 0;
    hipStream_t last_ = nullptr;
    bool used_ = false;
    hipEvent_t between_ = nullptr;

    void release();
    bool enter(hipStream_t s);     // -> the stream is being captured
    void settle(hipStream_t s);    // no capture: what changes on the host cannot be replayed
    void join_streams(hipStream_t s);
    CacheMemory memory() const { return CacheMemory{words_, words_ + book_.table_at(), book_.pitch(), pool_, page_bytes_}; }
    void carry_out(const PageBook::Moves& moves, hipStream_t s, int source = 0, int n = 0, const int* lists = nullptr);
    PageLayout layout(int layer) const;
    CacheWords words() const;
};

// Attention over dense tensors.
void attention(const fyn_attention_desc& a, hipStream_t s);
void run_attention(const AttnParams& p, hipStream_t s);
bool attention_params(const fyn_attention_desc& a, AttnParams& p, int& device);   // checked; false: nothing to do

// The current device for the length of a call.
class OnDevice {
  public:
    explicit OnDevice(int device);
    ~OnDevice();
  private:
    int was_ = -1;
};

// Checks of a tensor's memory: where it is and how it is aligned.  -> the device that has it.
int check_rows(const char* what, const fyn_rows& r, int f16);

}  // namespace fynhip

struct fyn_cache {
    std::shared_ptr<fynhip::Cache> impl;
};
