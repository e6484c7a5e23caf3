// extern "C" surface declared in include/fynhip.h: translates C++ errors into status codes and a
// thread-local message (the text a FynException would have carried, common/fynexception.h).
#include <cstring>
#include <string>

#include "cache.h"
#include "engine.h"

struct fyn_net {
    fynhip::Net* impl;
};

static thread_local std::string g_last_error;

#define FYN_API_BEGIN try {
#define FYN_API_END                                     \
    }                                                   \
    catch (const fynhip::Error& e) {                    \
        g_last_error = e.what();                        \
        return e.code;                                  \
    }                                                   \
    catch (const std::bad_alloc&) {                     \
        g_last_error = "out of host memory";            \
        return FYN_ERR_DEVICE;                          \
    }                                                   \
    catch (const std::exception& e) {                   \
        g_last_error = e.what();                        \
        return FYN_ERR_INVALID;                         \
    }                                                   \
    return FYN_OK;

static fyn_layer_desc described(const fyn_layer_desc* desc) {
    if (!desc) fynhip::fail(FYN_ERR_INVALID, "No builder supplied to layer factory line");
    if (desc->struct_size != sizeof(fyn_layer_desc))
        fynhip::fail(FYN_ERR_INVALID, "fyn_layer_desc size mismatch (%u, library expects %zu)", desc->struct_size, sizeof(fyn_layer_desc));
    fyn_layer_desc d = *desc;
    d.name[FYN_NAME_LEN - 1] = 0;
    return d;
}

static fynhip::Net* N(fyn_net* n) {
    if (!n || !n->impl) fynhip::fail(FYN_ERR_INVALID, "null network handle");
    return n->impl;
}

static fynhip::Cache* C(fyn_cache* c) {
    if (!c || !c->impl) fynhip::fail(FYN_ERR_INVALID, "null cache handle");
    return c->impl.get();
}
template <class D>
static const D& sized(const D* d, const char* name) {
    if (!d) fynhip::fail(FYN_ERR_INVALID, "no %s given", name);
    if (d->struct_size != sizeof(D)) fynhip::fail(FYN_ERR_INVALID, "%s size mismatch (%u, library expects %zu)", name, d->struct_size, sizeof(D));
    return *d;
}
static const fyn_rows& given(const fyn_rows* r) {
    if (!r) fynhip::fail(FYN_ERR_INVALID, "no keys or values given");
    return *r;
}

extern "C" {

const char* fyn_last_error(void) { return g_last_error.c_str(); }

int fyn_device_info(int device, char* buf, size_t buflen) {
    FYN_API_BEGIN
    if (!buf || buflen == 0) fynhip::fail(FYN_ERR_INVALID, "null buffer");
    hipDeviceProp_t prop;
    FYN_HIP(hipGetDeviceProperties(&prop, device));
    snprintf(buf, buflen, "%s arch=%s CUs=%d clock=%dMHz mem=%.1fGiB lds/block=%zu", prop.name, prop.gcnArchName,
             prop.multiProcessorCount, prop.clockRate / 1000, (double)prop.totalGlobalMem / (1024.0 * 1024.0 * 1024.0),
             (size_t)prop.sharedMemPerBlock);
    FYN_API_END
}

int fyn_net_create(int device, int storage, fyn_net** out) {
    FYN_API_BEGIN
    if (!out) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    fynhip::Net* impl = new fynhip::Net(device, storage);
    *out = new fyn_net{impl};
    FYN_API_END
}

int fyn_net_destroy(fyn_net* net) {
    FYN_API_BEGIN
    if (net) {
        delete net->impl;
        delete net;
    }
    FYN_API_END
}

int fyn_net_add_layer(fyn_net* net, const fyn_layer_desc* desc) {
    FYN_API_BEGIN
    N(net)->add_layer(described(desc));
    FYN_API_END
}

int fyn_net_add_custom_layer(fyn_net* net, const fyn_layer_desc* desc, const fyn_custom_layer* impl) {
    FYN_API_BEGIN
    if (!impl) fynhip::fail(FYN_ERR_INVALID, "No builder supplied to layer factory line");
    N(net)->add_custom_layer(described(desc), *impl);
    FYN_API_END
}

int fyn_net_connect(fyn_net* net, int out_layer, int in_layer, int port) {
    FYN_API_BEGIN
    N(net)->connect(out_layer, in_layer, port);
    FYN_API_END
}

int fyn_layer_load_weights(fyn_net* net, int layer, const float* wb, size_t offset_floats) {
    FYN_API_BEGIN
    if (!wb) fynhip::fail(FYN_ERR_INVALID, "null weight pointer");
    fynhip::Layer* l = N(net)->layer(layer);
    if (l->d.type == FYN_LAYER_BATCHNORM) fynhip::fail(FYN_ERR_INVALID, "layer %s takes scale/bias, not weights", l->d.name);
    l->load_weights(wb + offset_floats);
    N(net)->weights_changed();
    FYN_API_END
}

int fyn_layer_load_scale_bias(fyn_net* net, int layer, const float* sb, size_t offset_floats) {
    FYN_API_BEGIN
    if (!sb) fynhip::fail(FYN_ERR_INVALID, "null scale/bias pointer");
    fynhip::Layer* l = N(net)->layer(layer);
    if (l->d.type != FYN_LAYER_BATCHNORM) fynhip::fail(FYN_ERR_INVALID, "layer %s is not a batchnorm layer", l->d.name);
    l->load_weights(sb + offset_floats);
    N(net)->weights_changed();
    FYN_API_END
}

int fyn_layer_weight_floats(fyn_net* net, int layer, size_t* count) {
    FYN_API_BEGIN
    if (!count) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    *count = N(net)->layer(layer)->weight_floats();
    FYN_API_END
}

int fyn_net_setup(fyn_net* net) {
    FYN_API_BEGIN
    N(net)->setup();
    FYN_API_END
}

int fyn_net_set_input(fyn_net* net, int layer, int port, const float* data, int order) {
    FYN_API_BEGIN
    N(net)->set_input(layer, port, data, order);
    FYN_API_END
}

int fyn_net_input_floats(fyn_net* net, int layer, int port, size_t* count) {
    FYN_API_BEGIN
    if (!count) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    *count = N(net)->input_floats(layer, port);
    FYN_API_END
}

int fyn_net_forward(fyn_net* net, uint64_t* seq_out) {
    FYN_API_BEGIN
    N(net)->forward(seq_out);
    FYN_API_END
}

int fyn_net_finish(fyn_net* net) {
    FYN_API_BEGIN
    N(net)->finish();
    FYN_API_END
}

int fyn_layer_copy_result(fyn_net* net, int layer, float* chw, int include_padding) {
    FYN_API_BEGIN
    if (!chw) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    N(net)->copy_result(layer, chw, include_padding);
    FYN_API_END
}

int fyn_layer_copy_result_noalloc(fyn_net* net, int layer, float* chw, int include_padding) {
    FYN_API_BEGIN
    if (!chw) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    N(net)->copy_result_static(layer, chw, include_padding);
    FYN_API_END
}

int fyn_layer_output_shape(fyn_net* net, int layer, int* channels, int* height, int* width, int* padding) {
    FYN_API_BEGIN
    fynhip::Layer* l = N(net)->layer(layer);
    if (channels) *channels = l->oc;
    if (height) *height = l->oh;
    if (width) *width = l->ow;
    // a pass-through (download) layer hands on its input tensor, halo included
    if (padding) *padding = (N(net)->is_setup && l->out >= 0) ? l->tout().v.pad : l->d.output_padding;
    FYN_API_END
}

int fyn_net_get_output(fyn_net* net, int layer, float* data, int order) {
    FYN_API_BEGIN
    if (!data) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    N(net)->get_output(layer, data, order);
    FYN_API_END
}

int fyn_layer_copy_argmax(fyn_net* net, int layer, int32_t* idx, float* val) {
    FYN_API_BEGIN
    N(net)->copy_argmax(layer, idx, val);
    FYN_API_END
}

int fyn_net_enable_timings(fyn_net* net, int enable) {
    FYN_API_BEGIN
    fynhip::Net* n = N(net);
    n->finish();
    n->timings = enable != 0;
    if (!enable) return FYN_OK;
    for (auto& kv : n->layers) {
        kv.second->ms_total = 0.f;
        kv.second->runs = 0;
    }
    FYN_API_END
}

int fyn_net_get_timing(fyn_net* net, int layer, float* ms_total, int* runs) {
    FYN_API_BEGIN
    fynhip::Net* n = N(net);
    n->finish();
    fynhip::Layer* l = n->layer(layer);
    if (ms_total) *ms_total = l->ms_total;
    if (runs) *runs = l->runs;
    FYN_API_END
}

int fyn_net_enable_intermediate_output(fyn_net* net, const char* dir) {
    FYN_API_BEGIN
    N(net)->dump_dir = dir ? dir : "";
    FYN_API_END
}

int fyn_net_set_buffer_reuse(fyn_net* net, int enable) {
    FYN_API_BEGIN
    fynhip::Net* n = N(net);
    if (n->is_setup) fynhip::fail(FYN_ERR_STATE, "buffer reuse must be chosen before setup");
    n->reuse_buffers = enable != 0;
    FYN_API_END
}

int fyn_net_use_graph(fyn_net* net, int enable) {
    FYN_API_BEGIN
    N(net)->use_graph(enable != 0);
    FYN_API_END
}

int fyn_net_time_forward(fyn_net* net, int iters, float* ms_total) {
    FYN_API_BEGIN
    if (!ms_total || iters < 1) fynhip::fail(FYN_ERR_INVALID, "invalid arguments");
    N(net)->time_forward(iters, ms_total);
    FYN_API_END
}

int fyn_net_time_steps(fyn_net* net, int iters, float* ms_each) {
    FYN_API_BEGIN
    if (!ms_each || iters < 1) fynhip::fail(FYN_ERR_INVALID, "need an output array and at least one step");
    N(net)->time_steps(iters, ms_each);
    FYN_API_END
}

int fyn_layer_time(fyn_net* net, int layer, int iters, float* ms_total) {
    FYN_API_BEGIN
    if (!ms_total || iters < 1) fynhip::fail(FYN_ERR_INVALID, "invalid arguments");
    N(net)->time_layer(layer, iters, ms_total);
    FYN_API_END
}

int fyn_net_async_begin(fyn_net* net, int in_layer, int in_port, int in_order, int out_layer, int out_order, int depth, int copy_streams) {
    FYN_API_BEGIN
    N(net)->async_begin(in_layer, in_port, in_order, out_layer, out_order, depth, copy_streams != 0);
    FYN_API_END
}

int fyn_net_async_submit(fyn_net* net, const float* in, float* out, uint64_t* ticket) {
    FYN_API_BEGIN
    N(net)->async_submit(in, out, ticket);
    FYN_API_END
}

int fyn_net_async_sizes(fyn_net* net, size_t* in_floats, size_t* out_floats) {
    FYN_API_BEGIN
    if (!in_floats || !out_floats) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    N(net)->async_sizes(in_floats, out_floats);
    FYN_API_END
}

int fyn_net_async_wait(fyn_net* net, uint64_t ticket) {
    FYN_API_BEGIN
    N(net)->async_wait(ticket);
    FYN_API_END
}

int fyn_net_async_end(fyn_net* net) {
    FYN_API_BEGIN
    N(net)->async_end();
    FYN_API_END
}

int fyn_host_acquire(size_t bytes, void** ptr) {
    FYN_API_BEGIN
    if (!ptr) fynhip::fail(FYN_ERR_INVALID, "null pointer");
    *ptr = fynhip::HostPool::acquire(bytes, true);
    FYN_API_END
}

int fyn_host_release(void* ptr) {
    FYN_API_BEGIN
    fynhip::HostPool::release(ptr);
    FYN_API_END
}

int fyn_net_device_allocations(fyn_net* net, size_t* calls, size_t* bytes) {
    FYN_API_BEGIN
    if (calls) *calls = N(net)->alloc_calls_;
    if (bytes) *bytes = N(net)->alloc_bytes_;
    FYN_API_END
}

int fyn_layer_kernel_info(fyn_net* net, int layer, char* buf, size_t buflen) {
    FYN_API_BEGIN
    if (!buf || buflen == 0) fynhip::fail(FYN_ERR_INVALID, "null buffer");
    std::string s = N(net)->layer(layer)->info();
    snprintf(buf, buflen, "%s", s.c_str());
    FYN_API_END
}

// ---- sequences ----
int fyn_attention(const fyn_attention_desc* desc, void* hip_stream) {
    FYN_API_BEGIN
    fynhip::attention(sized(desc, "fyn_attention_desc"), static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_create(int device, const fyn_cache_desc* desc, fyn_cache** out) {
    FYN_API_BEGIN
    if (!out) fynhip::fail(FYN_ERR_INVALID, "null output pointer");
    std::unique_ptr<fyn_cache> c(new fyn_cache);
    c->impl = std::make_shared<fynhip::Cache>(device, sized(desc, "fyn_cache_desc"));
    *out = c.release();
    FYN_API_END
}

int fyn_cache_destroy(fyn_cache* cache) {
    FYN_API_BEGIN
    delete cache;
    FYN_API_END
}

int fyn_cache_extend(fyn_cache* cache, int n, const int32_t* sequences, const int32_t* tokens, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->extend(n, sequences, tokens, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_write(fyn_cache* cache, int layer, const fyn_rows* keys, const fyn_rows* values, int rows, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->write(layer, given(keys), given(values), rows, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_attend(fyn_cache* cache, int layer, const fyn_attend_desc* desc, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->attend(layer, sized(desc, "fyn_attend_desc"), static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_read(fyn_cache* cache, int n, const int32_t* sequences, int layer, const fyn_rows* keys, const fyn_rows* values, int rows, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->read(n, sequences, layer, given(keys), given(values), rows, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_fork(fyn_cache* cache, int source, int n, const int32_t* targets, int tokens, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->fork(source, n, targets, tokens, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_copy(fyn_cache* cache, int n, const int32_t* sources, const int32_t* targets, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->copy(n, sources, targets, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_truncate(fyn_cache* cache, int n, const int32_t* sequences, const int32_t* tokens, void* hip_stream) {
    FYN_API_BEGIN
    if (n > 0 && !tokens) fynhip::fail(FYN_ERR_INVALID, "cache: no numbers of tokens given");
    C(cache)->truncate(n, sequences, tokens, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_free(fyn_cache* cache, int n, const int32_t* sequences, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->truncate(n, sequences, nullptr, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_compact(fyn_cache* cache, int* used, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->compact(used, static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

int fyn_cache_lengths(fyn_cache* cache, int n, const int32_t* sequences, int32_t* tokens) {
    FYN_API_BEGIN
    C(cache)->lengths(n, sequences, tokens);
    FYN_API_END
}

int fyn_cache_pages(fyn_cache* cache, int* used, int* free_pages) {
    FYN_API_BEGIN
    C(cache)->pages(used, free_pages);
    FYN_API_END
}

int fyn_net_add_attention_layer(fyn_net* net, const fyn_layer_desc* desc, const fyn_attention_layer* attention) {
    FYN_API_BEGIN
    N(net)->add_attention_layer(described(desc), sized(attention, "fyn_attention_layer"));
    FYN_API_END
}

int fyn_layer_bind_cache(fyn_net* net, int layer, fyn_cache* cache, int cache_layer) {
    FYN_API_BEGIN
    fynhip::Net* n = N(net);
    n->finish();   // (a pass that runs has what it was given)
    n->layer(layer)->bind_cache(cache ? C(cache)->shared_from_this() : nullptr, cache_layer);
    n->weights_changed();
    FYN_API_END
}

int fyn_cache_order(fyn_cache* cache, void* hip_stream) {
    FYN_API_BEGIN
    C(cache)->order(static_cast<hipStream_t>(hip_stream));
    FYN_API_END
}

}  // extern "C"
