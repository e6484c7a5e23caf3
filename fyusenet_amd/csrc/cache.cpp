// Host side of attention and of the cache of keys and values: checks, launches, order between streams.
#include "cache.h"

#include <algorithm>
#include <cmath>
#include <iterator>

namespace fynhip {

OnDevice::OnDevice(int device) {
    FYN_HIP(hipGetDevice(&was_));
    if (was_ != device) FYN_HIP(hipSetDevice(device));
    else was_ = -1;
}
OnDevice::~OnDevice() {
    if (was_ >= 0) (void)hipSetDevice(was_);
}

int check_rows(const char* what, const fyn_rows& r, int f16) {
    if (!r.data) fail(FYN_ERR_INVALID, "%s: null pointer", what);
    const int64_t unit = f16 ? 8 : 4;
    if (reinterpret_cast<uintptr_t>(r.data) % 16 || r.sequence_pitch % unit || r.token_pitch % unit || r.head_pitch % unit)
        fail(FYN_ERR_INVALID, "%s: address and pitches have to be multiples of 16 bytes", what);
    if (r.sequence_pitch < 0 || r.token_pitch < 0 || r.head_pitch < 0) fail(FYN_ERR_INVALID, "%s: negative pitch", what);
    hipPointerAttribute_t at;
    const hipError_t e = hipPointerGetAttributes(&at, r.data);
    if (e != hipSuccess || at.type != hipMemoryTypeDevice) {
        (void)hipGetLastError();
        fail(FYN_ERR_INVALID, "%s: not device memory", what);
    }
    return at.device;
}

// Rows that are written: no two of them may share memory.
static void check_apart(const char* what, const fyn_rows& r, int64_t sequences, int64_t tokens, int64_t heads, int dim) {
    std::pair<int64_t, int64_t> axes[] = {{r.head_pitch, heads}, {r.token_pitch, tokens}, {r.sequence_pitch, sequences}};
    std::sort(std::begin(axes), std::end(axes));
    __int128 span = dim;   // of what the axes so far reach over
    for (auto [pitch, n] : axes) {
        if (n <= 1) continue;
        if (pitch < span) fail(FYN_ERR_INVALID, "%s: rows of %d values at distances of %lld overlap", what, dim, (long long)pitch);
        span += (__int128)(n - 1) * pitch;
    }
}

static SeqRows rows_of(const fyn_rows& r) { return SeqRows{static_cast<char*>(r.data), r.sequence_pitch, r.token_pitch, r.head_pitch}; }

static float scale_log2(float scale, int dim) { return (scale == 0.f ? 1.f / std::sqrt((float)dim) : scale) * 1.44269504f; }

static void check_sight(int window, int sinks, float scale) {
    if (window < 0 || sinks < 0) fail(FYN_ERR_INVALID, "attention: window %d and sinks %d must not be negative", window, sinks);
    if (!std::isfinite(scale * 1.44269504f)) fail(FYN_ERR_INVALID, "attention: the scale is not finite, or too large");
}

static void check_heads(int heads, int kv_heads, int dim) {
    if (kv_heads < 1 || heads < 1 || heads > 65536 || heads % kv_heads) fail(FYN_ERR_INVALID, "attention: %d heads cannot share %d key heads", heads, kv_heads);
    if (dim < 8 || dim > kMaxHeadDim || dim % 8) fail(FYN_ERR_UNSUPPORTED, "attention: heads of %d values (multiples of 8 up to %d are supported)", dim, kMaxHeadDim);
}

static void check_storage(int storage) {
    if (storage != FYN_STORAGE_F32 && storage != FYN_STORAGE_F16) fail(FYN_ERR_INVALID, "unknown storage type %d", storage);
}

// How many of the `tokens` tokens of a head a workgroup of the kernel with tiles in shared memory gets; 0: the call is not for it.
static int tiled(const AttnParams& p, int tokens) {
    if (p.dim > 128 && !p.f16) return 0;
    if (!p.paged && std::max(p.k.tok, p.v.tok) * (p.f16 ? 2 : 4) > (1 << 24)) return 0;      // (32 bits of offset within a tile)
    // Large workgroups read keys and values the fewest times, small ones are more: 128 queries where that gives two workgroups
    // for each CU (16 heads of 4096 tokens, both ways: 222 us, against 243 with 64; causal, with runs of unequal length, 153 against 138;
    // half as many workgroups, 8 heads of 2048 tokens, two sequences: 71 us, against 49 with 64), 64 where it gives them for three quarters of
    // the CUs (12 heads of 197 tokens, four sequences: 8.9 us, against 11.4 without tiles; 8 heads of 1024 tokens of 64 values, fp32, which is
    // half of the CUs: 53 us, against 27).  Sequences count as long as the longest: of many short ones beside a long one most workgroups are
    // empty or have few queries.
    const int64_t units = (int64_t)p.batch * p.heads;
    if (units * ((tokens + 127) / 128) >= 512) return 128;
    if (units * ((tokens + 63) / 64) >= 192) return 64;
    return 0;
}

bool attention_params(const fyn_attention_desc& a, AttnParams& p, int& device) {
    check_storage(a.storage);
    check_heads(a.heads, a.kv_heads, a.head_dim);
    check_sight(a.window, a.sinks, a.scale);
    if (a.batch < 0 || a.tokens < 0 || (int64_t)a.batch * a.tokens > 0x7fffffff - 65536) fail(FYN_ERR_INVALID, "attention: %d sequences of %d tokens", a.batch, a.tokens);
    if (a.batch == 0 || a.tokens == 0) return false;
    const int f16 = a.storage == FYN_STORAGE_F16;
    check_apart("result", a.result, a.batch, a.tokens, a.heads, a.head_dim);
    device = check_rows("queries", a.queries, f16);
    if (check_rows("keys", a.keys, f16) != device || check_rows("values", a.values, f16) != device || check_rows("result", a.result, f16) != device)
        fail(FYN_ERR_INVALID, "attention: the tensors are on different devices");
    if (a.lengths) {
        hipPointerAttribute_t at;
        if (reinterpret_cast<uintptr_t>(a.lengths) % 4 || hipPointerGetAttributes(&at, a.lengths) != hipSuccess || at.type != hipMemoryTypeDevice || at.device != device) {
            (void)hipGetLastError();
            fail(FYN_ERR_INVALID, "lengths: not memory of the tensors' device");
        }
    }
    p = AttnParams{};
    p.q = rows_of(a.queries); p.k = rows_of(a.keys); p.v = rows_of(a.values); p.out = rows_of(a.result);
    p.lengths = a.lengths;
    p.f16 = f16;
    p.batch = a.batch; p.tokens = a.tokens;
    p.heads = a.heads; p.kv_heads = a.kv_heads; p.dim = a.head_dim;
    p.causal = a.causal != 0; p.window = a.window; p.sinks = a.sinks;
    p.scale_log2 = scale_log2(a.scale, a.head_dim);
    p.by_token = 1;
    p.chunk = 0x7fffffff;
    p.parts = 1;
    p.tiled = tiled(p, a.tokens);
    const int columns = p.tiled ? p.tiled : 16;
    p.tiles = (a.tokens + columns - 1) / columns;
    return true;
}

void run_attention(const AttnParams& p, hipStream_t s) {
    const int rc = launch_attention(p, s);
    if (rc == -2) fail(FYN_ERR_INVALID, "attention: more heads and tokens of one sequence than a launch takes");
    if (rc != 0) fail(FYN_ERR_DEVICE, "attention: launch failed");
}

void attention(const fyn_attention_desc& a, hipStream_t s) {
    AttnParams p;
    int device;
    if (!attention_params(a, p, device)) return;
    OnDevice on(device);
    run_attention(p, s);
}

// ---------------------------------------------------------------------------------------------------------------------
static const fyn_cache_desc& checked(const fyn_cache_desc& d) {
    check_storage(d.storage);
    check_heads(d.heads, d.kv_heads, d.head_dim);
    if (d.layers < 1 || d.layers > 65536) fail(FYN_ERR_INVALID, "cache: %d layers", d.layers);
    if (d.page_tokens < 8 || d.page_tokens > 1024 || (d.page_tokens & (d.page_tokens - 1)))
        fail(FYN_ERR_UNSUPPORTED, "cache: pages of %d tokens (powers of two from 8 to 1024 are supported)", d.page_tokens);
    if (d.pages < 1 || d.sequences < 1 || d.sequences > (1 << 20)) fail(FYN_ERR_INVALID, "cache: %d pages, %d sequences", d.pages, d.sequences);
    if ((int64_t)d.pages * d.page_tokens > 0x7fffffff - 65536) fail(FYN_ERR_INVALID, "cache: %d pages of %d tokens hold more tokens than can be counted", d.pages, d.page_tokens);
    if (d.most_tokens < 0 || d.most_tokens > d.pages * d.page_tokens) fail(FYN_ERR_INVALID, "cache: sequences of up to %d tokens do not fit into %d pages", d.most_tokens, d.pages);
    // (a page has up to 2^53 bytes)
    const int64_t page_bytes = (int64_t)d.layers * 2 * d.kv_heads * d.page_tokens * d.head_dim * (d.storage == FYN_STORAGE_F16 ? 2 : 4);
    if (page_bytes > (INT64_MAX >> 2) / d.pages) fail(FYN_ERR_INVALID, "cache: %d pages of %lld bytes are more than can be addressed", d.pages, (long long)page_bytes);
    const int64_t pitch = (d.most_tokens ? d.most_tokens + d.page_tokens - 1 : d.pages * d.page_tokens) / d.page_tokens;
    if (pitch * d.sequences > (1 << 30)) fail(FYN_ERR_INVALID, "cache: lists of %lld pages for each of %d sequences; give the most tokens of one (most_tokens)", (long long)pitch, d.sequences);
    return d;
}

Cache::Cache(int dev, const fyn_cache_desc& desc)
    : device(dev), d(checked(desc)), book_(desc.pages, desc.sequences, desc.page_tokens, desc.most_tokens ? desc.most_tokens : desc.pages * desc.page_tokens) {
    int count = 0;
    FYN_HIP(hipGetDeviceCount(&count));
    if (dev < 0 || dev >= count) fail(FYN_ERR_DEVICE, "device %d not present (%d devices)", dev, count);
    OnDevice on(dev);
    const int64_t size = d.storage == FYN_STORAGE_F16 ? 2 : 4;
    head_bytes_ = d.page_tokens * d.head_dim * size;
    layer_bytes_ = 2 * d.kv_heads * head_bytes_;
    page_bytes_ = d.layers * layer_bytes_;
    // sums of parts of rows that are read by several workgroups: enough for the parts of whole batches (attend())
    const int64_t most = (int64_t)book_.pitch() * d.page_tokens;
    part_cells_ = std::min<int64_t>(65536, (int64_t)d.sequences * 16 * d.heads * (most / 64 + 1));
    try {
        FYN_HIP(hipMalloc(&pool_, (size_t)(page_bytes_ * d.pages)));
        FYN_HIP(hipMalloc(&words_, book_.words.size() * sizeof(int)));
        FYN_HIP(hipMalloc(&parts_, (size_t)(part_cells_ * (d.head_dim + 2)) * sizeof(float)));
        FYN_HIP(hipEventCreateWithFlags(&between_, hipEventDisableTiming));
        FYN_HIP(hipMemset(words_, 0, book_.words.size() * sizeof(int)));
        FYN_HIP(hipStreamSynchronize(nullptr));
    } catch (...) {
        release();
        throw;
    }
}

void Cache::release() {
    if (pool_) (void)hipFree(pool_);   // (waits for what uses it)
    if (words_) (void)hipFree(words_);
    if (parts_) (void)hipFree(parts_);
    if (between_) (void)hipEventDestroy(between_);
}

Cache::~Cache() {
    int was = -1;
    (void)hipGetDevice(&was);
    (void)hipSetDevice(device);
    (void)hipDeviceSynchronize();
    release();
    if (was >= 0) (void)hipSetDevice(was);
}

static bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) == hipSuccess) return st != hipStreamCaptureStatusNone;
    (void)hipGetLastError();
    return false;
}

void Cache::join_streams(hipStream_t s) {
    if (used_ && last_ != s) {
        // (its work from before the capture could not be waited for without becoming part of the capture)
        if (capturing(last_)) fail(FYN_ERR_STATE, "cache: the stream that it was used on last is being captured");
        // (a stream that is gone cannot be asked: everything on the device then)
        if (hipEventRecord(between_, last_) == hipSuccess) {
            FYN_HIP(hipStreamWaitEvent(s, between_, 0));
        } else {
            (void)hipGetLastError();
            FYN_HIP(hipDeviceSynchronize());
        }
    }
    last_ = s;
    used_ = true;
}

bool Cache::enter(hipStream_t s) {
    if (capturing(s)) return true;
    join_streams(s);
    return false;
}

void Cache::settle(hipStream_t s) {
    if (capturing(s)) fail(FYN_ERR_STATE, "cache: sequences and pages cannot change while the stream is being captured");
    join_streams(s);
}

void Cache::order(hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    OnDevice on(device);
    if (capturing(s)) fail(FYN_ERR_STATE, "cache: a stream that is being captured is not put in order (the stream that replays is, in front of the replay)");
    join_streams(s);
}

std::vector<int> Cache::expect(int rows, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    if (rows != book_.batch_rows()) fail(FYN_ERR_INVALID, "cache: the batch has %d new tokens, the layer %d positions", book_.batch_rows(), rows);
    OnDevice on(device);
    enter(s);
    const int* first = book_.words.data() + book_.first_at();
    return std::vector<int>(first, first + book_.batch_size() + 1);
}

// What the book has changed, on the device: words, lists that are copies of another's, pages that are copied; in as few launches
// as their arguments hold.  The parts of a launch run in any order.  That is sound: a call changes no word twice, no page is
// copied from and to, a list that is copied from or to has no words changed in the same call, and copies do not look at words.
void Cache::carry_out(const PageBook::Moves& moves, hipStream_t s, int source, int n, const int* lists) {
    const CacheMemory m = memory();
    CacheChange c;
    auto clear = [&] { c.runs = c.singles = c.lists = c.moves = 0; };
    auto send = [&] {
        if (c.used()) FYN_HIP(launch_cache_change(m, c, s));
        clear();
    };
    clear();
    c.source = source;
    c.entries = n > 0 ? (int)book_.list(lists[0]).size() : 0;
    constexpr size_t kFew = 4;   // words of a run that go one by one: all at once then, where runs wait for each other's lengths
    for (auto [at, end] : book_.changes()) {
        if (end - at <= kFew) continue;
        while (at < end) {
            if (c.used() + 3 > kChangeWords) send();
            const int k = (int)std::min<size_t>(end - at, kChangeWords - c.used() - 2);
            c.w[c.runs] = (int)at;
            c.w[c.runs + 1] = k;
            std::copy_n(book_.words.begin() + at, k, c.w + c.runs + 2);
            c.runs += 2 + k;
            at += k;
        }
    }
    for (auto [at, end] : book_.changes()) {
        if (end - at > kFew) continue;
        for (; at < end; at++) {
            if (c.used() + 2 > kChangeWords) send();
            c.w[c.used()] = (int)at;
            c.w[c.used() + 1] = book_.words[at];
            c.singles++;
        }
    }
    book_.changes_taken();
    for (int i = 0; i < n && c.entries > 0; i++) {
        if (c.used() + 1 > kChangeWords) send();
        c.w[c.used()] = lists[i];
        c.lists++;
    }
    // (a launch has at most 2^31 workgroups)
    const int64_t most = std::max<int64_t>(1, (int64_t)0x7fff0000 / (page_bytes_ / 16384 + 1));
    for (const auto& x : moves) {
        if (c.used() + 2 > kChangeWords || c.moves >= most) send();
        c.w[c.used()] = x.first;
        c.w[c.used() + 1] = x.second;
        c.moves++;
    }
    send();
}

PageLayout Cache::layout(int layer) const {
    if (layer < 0 || layer >= d.layers) fail(FYN_ERR_INVALID, "cache: there is no layer %d", layer);
    PageLayout l;
    l.pool = pool_ + layer * layer_bytes_;
    l.page_bytes = page_bytes_;
    l.values = d.kv_heads * head_bytes_;
    l.head_bytes = head_bytes_;
    l.shift = __builtin_ctz(d.page_tokens);
    return l;
}

CacheWords Cache::words() const {
    return CacheWords{words_, words_ + book_.batch_at(), words_ + book_.first_at(), words_ + book_.table_at(), book_.pitch(), d.sequences};
}

template <class F>
static auto booked(F&& f) {
    try {
        return f();
    } catch (const PageBook::Refused& r) {
        fail(r.full ? FYN_ERR_STATE : FYN_ERR_INVALID, "cache: %s", r.why.c_str());
    }
}

void Cache::extend(int n, const int* seqs, const int* counts, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    if (n > 0 && !counts) fail(FYN_ERR_INVALID, "cache: no numbers of tokens given");
    OnDevice on(device);
    settle(s);
    carry_out(booked([&] { return book_.extend(n, seqs, counts); }), s);
}

void Cache::fork(int source, int n, const int* targets, int tokens, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    OnDevice on(device);
    settle(s);
    booked([&] { book_.fork(source, n, targets, tokens); return 0; });
    carry_out({}, s, source, n, targets);
}

void Cache::copy(int n, const int* sources, const int* targets, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    if (n > 0 && !sources) fail(FYN_ERR_INVALID, "cache: no sequences given");
    OnDevice on(device);
    settle(s);
    carry_out(booked([&] { return book_.copy(n, sources, targets); }), s);
}

void Cache::truncate(int n, const int* seqs, const int* tokens, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    OnDevice on(device);
    settle(s);
    booked([&] { book_.truncate(n, seqs, tokens); return 0; });
    carry_out({}, s);
}

void Cache::compact(int* used, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    OnDevice on(device);
    settle(s);
    carry_out(book_.compact(), s);
    if (used) *used = book_.pages_used();
}

void Cache::lengths(int n, const int* seqs, int* tokens) {
    std::lock_guard<std::mutex> lock(mu_);
    if (n > 0 && (!seqs || !tokens)) fail(FYN_ERR_INVALID, "cache: null pointer");
    for (int i = 0; i < n; i++)
        if (seqs[i] < 0 || seqs[i] >= d.sequences) fail(FYN_ERR_INVALID, "cache: there is no sequence %d", seqs[i]);
    for (int i = 0; i < n; i++) tokens[i] = book_.length(seqs[i]);
}

void Cache::pages(int* used, int* free) {
    std::lock_guard<std::mutex> lock(mu_);
    if (used) *used = book_.pages_used();
    if (free) *free = book_.pages_free();
}

void Cache::write(int layer, const fyn_rows& k, const fyn_rows& v, int rows, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    const int f16 = d.storage == FYN_STORAGE_F16;
    CacheRows p{};
    p.pages = layout(layer);
    if (rows != book_.batch_rows()) fail(FYN_ERR_INVALID, "cache: the batch has %d new tokens, the tensors %d", book_.batch_rows(), rows);
    if (rows == 0) return;
    if (check_rows("keys", k, f16) != device || check_rows("values", v, f16) != device) fail(FYN_ERR_INVALID, "cache: keys or values are on another device");
    OnDevice on(device);
    enter(s);
    p.k = rows_of(k); p.v = rows_of(v);
    p.words = words();
    p.rows = rows; p.kv_heads = d.kv_heads; p.dim = d.head_dim; p.f16 = f16;
    FYN_HIP(launch_cache_write(p, s));
}

void Cache::read(int n, const int* seqs, int layer, const fyn_rows& k, const fyn_rows& v, int rows, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    const int f16 = d.storage == FYN_STORAGE_F16;
    CacheRows p{};
    p.pages = layout(layer);
    if (n < 0 || (n > 0 && !seqs)) fail(FYN_ERR_INVALID, "cache: no sequences given");
    int64_t total = 0;
    for (int i = 0; i < n; i++) {
        if (seqs[i] < 0 || seqs[i] >= d.sequences) fail(FYN_ERR_INVALID, "cache: there is no sequence %d", seqs[i]);
        total += book_.length(seqs[i]);
    }
    if (total != rows) fail(FYN_ERR_INVALID, "cache: the sequences have %lld tokens, the tensors %d", (long long)total, rows);
    if (rows == 0) return;
    check_apart("keys", k, 1, rows, d.kv_heads, d.head_dim);
    check_apart("values", v, 1, rows, d.kv_heads, d.head_dim);
    if (check_rows("keys", k, f16) != device || check_rows("values", v, f16) != device) fail(FYN_ERR_INVALID, "cache: keys or values are on another device");
    OnDevice on(device);
    settle(s);   // (which rows there are is settled on the host)
    p.words = words();
    p.kv_heads = d.kv_heads; p.dim = d.head_dim; p.f16 = f16;
    int64_t row = 0;
    CacheRead r;
    for (int i = 0; i < n;) {
        p.k = rows_of(k); p.v = rows_of(v);
        p.k.p += row * k.token_pitch * (f16 ? 2 : 4);
        p.v.p += row * v.token_pitch * (f16 ? 2 : 4);
        int at = 0;
        for (r.n = 0; r.n < kReadSequences && i < n; i++) {
            if (!book_.length(seqs[i])) continue;   // (a sequence without tokens has no rows)
            r.sequence[r.n] = seqs[i];
            r.first[r.n++] = at;
            at += book_.length(seqs[i]);
        }
        r.first[r.n] = at;
        p.rows = at;
        FYN_HIP(launch_cache_read(p, r, s));
        row += at;
    }
}

// Steps of keys that a token at `pos` of a sequence takes, as the kernel counts them.
static int64_t steps_of(int pos, int len, int window, int sinks, int step) {
    int64_t lo = 0, first = 0;
    const int64_t hi = std::min(pos + 1, len);
    if (window > 0) {
        lo = std::max(0, pos - window + 1);
        first = std::min<int64_t>(sinks, hi);
    }
    const int64_t a = (first + step - 1) / step, b = std::max(lo / step, a);
    return a + std::max<int64_t>(0, (hi + step - 1) / step - b);
}

void Cache::attend(int layer, const fyn_attend_desc& a, hipStream_t s) {
    std::lock_guard<std::mutex> lock(mu_);
    const int f16 = d.storage == FYN_STORAGE_F16;
    AttnParams p{};
    p.pages = layout(layer);
    check_sight(a.window, a.sinks, a.scale);
    if (a.rows != book_.batch_rows()) fail(FYN_ERR_INVALID, "cache: the batch has %d new tokens, the tensors %d", book_.batch_rows(), a.rows);
    if (a.rows == 0) return;
    check_apart("result", a.result, 1, a.rows, d.heads, d.head_dim);
    if (check_rows("queries", a.queries, f16) != device || check_rows("result", a.result, f16) != device) fail(FYN_ERR_INVALID, "cache: queries or result are on another device");
    OnDevice on(device);
    const bool captured = enter(s);
    p.q = rows_of(a.queries); p.out = rows_of(a.result);
    p.words = words();
    p.paged = 1; p.f16 = f16;
    p.batch = book_.batch_size(); p.tokens = a.rows;
    p.heads = d.heads; p.kv_heads = d.kv_heads; p.dim = d.head_dim;
    p.causal = 1; p.window = a.window; p.sinks = a.sinks;
    p.scale_log2 = scale_log2(a.scale, d.head_dim);
    const int group = d.heads / d.kv_heads, step = attention_step(f16, d.head_dim);
    const int* first = book_.words.data() + book_.first_at();
    int most_new = 0;
    for (int b = 0; b < p.batch; b++) most_new = std::max(most_new, first[b + 1] - first[b]);
    // Sixteen columns are a token's heads of a group, or sixteen tokens of a head: whichever reads the keys fewer times.
    const int by_group = most_new * ((group + 15) / 16), by_token = (most_new + 15) / 16 * group;
    if (by_token < by_group) {
        p.by_token = 1;
        p.tiled = tiled(p, most_new);
        const int columns = p.tiled ? p.tiled : 16;
        p.tiles = (most_new + columns - 1) / columns;
        p.chunk = 0x7fffffff;
        p.parts = 1;
    } else {
        p.tiles = by_group;
        // The keys of a row go to several workgroups, each of which takes as many steps wherever it is: 512 workgroups, two for
        // each CU, where the batch has work for them (64 sequences of 32768 tokens: 1.24 ms, and 1.27 with 1024), and at least two steps
        // for each of the four waves.  Up to four steps for each need no second launch to join them (230 tokens: 8.3 us, and
        // 11.4 with two parts).  A captured call is replayed when the sequences have grown: as many parts as the longest one would have.
        int64_t all = 0, longest = 0;
        const int64_t most = captured ? steps_of(book_.pitch() * d.page_tokens - 1, book_.pitch() * d.page_tokens, a.window, a.sinks, step) : 0;
        for (int b = 0; b < p.batch; b++) {
            const int len = book_.length(book_.words[book_.batch_at() + b]), n = first[b + 1] - first[b];
            if (!n) continue;
            const int64_t st = captured ? most : steps_of(len - 1, len, a.window, a.sinks, step);
            all += st * n;
            longest = std::max(longest, st);
        }
        all *= (int64_t)d.kv_heads * ((group + 15) / 16);
        const int64_t chunk = std::max<int64_t>(8, (all + 511) / 512);
        int64_t parts = longest <= 16 ? 1 : std::max<int64_t>(1, (longest + chunk - 1) / chunk);
        parts = std::max<int64_t>(1, std::min(parts, part_cells_ / ((int64_t)a.rows * d.heads)));
        p.chunk = (int)std::max(chunk, (longest + parts - 1) / parts);
        p.parts = (int)parts;
        // Branches of one sequence: over the pages that all of them have in front, sixteen columns are heads of several branches, which
        // reads those pages once for each sixteen instead of once for each branch (fp16, 32 heads of 128 dims in groups of 4, 12000
        // tokens in common: 39 us with 32 branches, and 114 without; 17.5 and 17.4 with two).  There is always a second launch
        // then, so that it takes 1024 such tokens, which have several parts anyway (260: 11.2 and 8.5 us with four branches;
        // 1040: 11.3 and 11.1, and with 32 of them 14 and 20).  A captured call is replayed when the sequences may have no pages in common.
        int shortest = book_.length(book_.words[book_.batch_at()]);
        for (int b = 0; b < p.batch; b++) shortest = std::min(shortest, book_.length(book_.words[book_.batch_at() + b]));
        const int common = std::min((int64_t)book_.common_pages() * d.page_tokens, (int64_t)shortest - 1) / 32 * 32, together = (p.batch * group + 15) / 16;
        if (!captured && most_new == 1 && a.rows == p.batch && a.window == 0 && common >= 1024 && together < p.batch) {
            const int64_t first_steps = common / step, own = longest - first_steps;
            const int64_t sum = (first_steps * together + own * p.batch) * d.kv_heads;
            int64_t each = std::max<int64_t>(8, (sum + 511) / 512);
            const int64_t room = part_cells_ / ((int64_t)a.rows * d.heads);
            while ((first_steps + each - 1) / each + (own + each - 1) / each > room && each < first_steps + own) each *= 2;
            const int64_t of_first = (first_steps + each - 1) / each, of_own = (own + each - 1) / each;
            if (of_first + of_own <= room) {
                p.common = common;
                p.common_tiles = together;
                p.common_parts = (int)of_first;
                p.common_chunk = (int)((first_steps + of_first - 1) / of_first);
                p.chunk = (int)((own + of_own - 1) / of_own);
                p.parts = (int)(of_first + of_own);
            }
        }
        p.once = p.tiles == 1 && !book_.shares();
        p.part_o = parts_;
        p.part_ml = parts_ + part_cells_ * d.head_dim;
    }
    run_attention(p, s);
}

}  // namespace fynhip
