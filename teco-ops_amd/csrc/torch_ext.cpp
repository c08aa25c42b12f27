// torch_ext.cpp — TORCH_LIBRARY(tecoops) registration of the operator path.
//
// Replaces the reference's pybind11 module api/torch_ext.cpp:208-215 (whose
// README claims a TORCH_LIBRARY registration it does not have) with real
// torch op schemas: the same op names and positional arguments
// (torch_ext.cpp:61-206), outputs mutated in place and annotated Tensor(a!),
// returning nothing.  Every op binds the current HIP stream of the calling
// thread (the reference never sets a stream, torch_ext.cpp:35-42) and calls
// the C ABI of libtecoops.so; a non-success status raises.
//
// Differences from the reference wrappers: flash_attn_varlen_func keeps
// cu_seqlens_q on the device (no host copy, torch_ext.cpp:119-126), honours
// softmax_scale / causal and takes the element type (fp16 or bf16) from q;
// causal_conv1d_fn_torch reads the [dim, tokens] layout in place instead of
// two transposing copies (torch_ext.cpp:186-205).
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>
#include <ATen/ATen.h>
#include <ATen/Tensor.h>

#include <algorithm>
#include <unordered_map>

#include "flash_attention.h"
#include "linear.h"
#include "tecoops.h"

namespace {

using at::Tensor;

// One handle per (thread, device), bound to that thread's current stream of
// the device on every call: threads never share a handle, so concurrent
// callers cannot race on its stream.
struct HandleCache {
    std::unordered_map<int, tecoopsHandle_t> by_device;
    ~HandleCache() {
        for (auto &kv : by_device) tecoopsDestroy(kv.second);
    }
};

tecoopsHandle_t handle_for(const Tensor &t) {
    thread_local HandleCache cache;
    const int dev = t.get_device();
    auto it = cache.by_device.find(dev);
    tecoopsHandle_t h;
    if (it == cache.by_device.end()) {
        TORCH_CHECK(tecoopsCreate(&h) == TECOOPS_STATUS_SUCCESS, "tecoopsCreate failed");
        cache.by_device.emplace(dev, h);
    } else {
        h = it->second;
    }
    tecoopsSetStream(h, c10::hip::getCurrentHIPStream(dev).stream());
    return h;
}

void check(tecoopsStatus_t st, const char *what) {
    TORCH_CHECK(st == TECOOPS_STATUS_SUCCESS, what, ": ", tecoopsGetErrorString(st));
}

tecoopsDataType_t dtype_of(const Tensor &t) {
    if (t.scalar_type() == at::kHalf) return TECOOPS_DATA_HALF;
    if (t.scalar_type() == at::kBFloat16) return TECOOPS_DATA_BFLOAT16;
    TORCH_CHECK(false, "tecoops: unsupported dtype ", t.scalar_type(), " (float16 or bfloat16)");
}

void need_cuda(std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        if (t && t->defined()) TORCH_CHECK(t->is_cuda(), "tecoops: tensors must be on the GPU");
}

// The C ABI takes plain pointers with packed row-major extents.
void need_contiguous(std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        if (t && t->defined())
            TORCH_CHECK(t->is_contiguous(), "tecoops: tensors must be contiguous");
}

void need_dtype(const Tensor &t, at::ScalarType st, const char *name) {
    TORCH_CHECK(t.scalar_type() == st, "tecoops: ", name, " must be ", st, ", got ",
                t.scalar_type());
}

struct Desc {
    tecoopsTensorDescriptor_t d = nullptr;
    Desc(const Tensor &t, tecoopsDataType_t dt) {
        check(tecoopsCreateTensorDescriptor(&d), "tecoopsCreateTensorDescriptor");
        std::vector<int> dims(t.dim()), strides(t.dim());
        for (int i = 0; i < t.dim(); ++i) {
            dims[i] = static_cast<int>(t.size(i));
            strides[i] = static_cast<int>(t.stride(i));
        }
        check(tecoopsSetTensorNdDescriptor(d, dt, t.dim(), dims.data(), strides.data()),
              "tecoopsSetTensorNdDescriptor");
    }
    ~Desc() { tecoopsDestroyTensorDescriptor(d); }
};

// reference torch_ext.cpp:61-79
void reshape_and_cache(const Tensor &key, const Tensor &value, const Tensor &slot_mapping,
                       Tensor &key_cache, Tensor &value_cache) {
    need_cuda({&key, &value, &slot_mapping, &key_cache, &value_cache});
    need_contiguous({&key, &value, &slot_mapping, &key_cache, &value_cache});
    TORCH_CHECK(slot_mapping.scalar_type() == at::kLong, "slot_mapping must be int64");
    TORCH_CHECK(key.dim() == 3 && key_cache.dim() == 4 && value.sizes() == key.sizes() &&
                    value_cache.sizes() == key_cache.sizes() &&
                    slot_mapping.numel() == key.size(0),
                "reshape_and_cache: key/value [T, Hkv, D], caches [blocks, Hkv, bs, D], "
                "slot_mapping [T]");
    check(tecoopsReshapeAndCacheEx(handle_for(key), key.data_ptr(), value.data_ptr(),
                                   slot_mapping.data_ptr<int64_t>(), key_cache.data_ptr(),
                                   value_cache.data_ptr(), key.size(0), key.size(1), key.size(2),
                                   key_cache.size(0), key_cache.size(2), dtype_of(key)),
          "reshape_and_cache");
}

// reference torch_ext.cpp:81-97
void rms_norm(const Tensor &input, const Tensor &weight, const c10::optional<Tensor> &residual,
              Tensor &output, const c10::optional<Tensor> &residual_out, double eps) {
    need_cuda({&input, &weight, &output});
    const Tensor *res = residual.has_value() ? &*residual : nullptr;
    const Tensor *res_out = residual_out.has_value() ? &*residual_out : nullptr;
    need_contiguous({&input, &weight, &output, res, res_out});
    // leading dimensions are rows, as in the plugin
    const int64_t D = input.size(-1);
    const int64_t N = D ? input.numel() / D : 0;
    const at::ScalarType st = input.scalar_type();
    need_dtype(weight, st, "weight");
    need_dtype(output, st, "output");
    TORCH_CHECK(weight.numel() == D && output.numel() == input.numel(),
                "rms_norm: weight must hold hidden_size elements and output match input");
    for (const Tensor *t : {res, res_out})
        if (t) {
            need_dtype(*t, st, "residual");
            TORCH_CHECK(t->numel() == input.numel(), "rms_norm: residual tensors must match input");
        }
    check(tecoopsRmsNormEx(handle_for(input), input.data_ptr(), weight.data_ptr(),
                           res ? res->data_ptr() : nullptr, output.data_ptr(),
                           res_out ? res_out->data_ptr() : nullptr, N, D,
                           static_cast<float>(eps), dtype_of(input)),
          "rms_norm");
}

// reference torch_ext.cpp:99-165
void flash_attn_varlen_func(const Tensor &q, const Tensor &k, const Tensor &v,
                            int64_t max_seqlen_q, const Tensor &cu_seqlens_q,
                            int64_t max_seqlen_k, const c10::optional<Tensor> &cu_seqlens_k,
                            const Tensor &seqused_k, double softmax_scale, bool causal,
                            const c10::optional<Tensor> &window_size, const Tensor &block_table,
                            bool return_softmax_lse, Tensor &out) {
    (void)cu_seqlens_k;
    (void)window_size;
    (void)return_softmax_lse;  // accepted and ignored, as in the reference
    need_cuda({&q, &k, &v, &cu_seqlens_q, &seqused_k, &block_table, &out});
    const tecoopsDataType_t dt = dtype_of(q);
    Desc bt(block_table, TECOOPS_DATA_INT32), qd(q, dt), kd(k, dt), vd(v, dt), od(out, dt);
    // The split-KV workspace comes from torch's allocator: stream-ordered like
    // any tensor, and taken from the graph's pool under CUDA-graph capture,
    // where the handle's own scratch (hipMalloc on a stream's first use) could
    // not be allocated.  The launch hints are the ones the library derives
    // without a workspace (mean q length; max_seqlen_k capped by the
    // block-table width * block size), so the plan and results are unchanged:
    // max_seqlen_q raised to the mean q length, max_seqlen_k capped by (or,
    // when <= 0, taken as) the block-table width * block size.
    int q_hint = static_cast<int>(max_seqlen_q), k_hint = static_cast<int>(max_seqlen_k);
    Tensor ws;
    if (q.dim() == 3 && k.dim() == 4 && block_table.dim() == 2 && block_table.size(0) > 0) {
        const int64_t batch = block_table.size(0);
        const int64_t cap = std::min<int64_t>(block_table.size(1) * k.size(2), 0x7fffffff);
        const int64_t q_mean = std::max<int64_t>(1, (q.size(0) + batch - 1) / batch);
        q_hint = static_cast<int>(std::min<int64_t>(std::max(max_seqlen_q, q_mean), 0x7fffffff));
        k_hint = static_cast<int>(max_seqlen_k > 0 ? std::min<int64_t>(max_seqlen_k, cap) : cap);
        // A workspace is for the decode route; a prefill uses the handle's scratch
        // where it splits its keys.  It is sized for this call's kv heads: for
        // any number of them 8 sequences of 1657 keys (32 heads over 8) took 1.7 MB
        // for 0.9, and above 1 MiB each captured graph's pool allocates a segment
        // of 20 MiB instead of 2 (preparing and capturing a decode step 1.92 ms
        // for 1.65).
        const int64_t H = q.size(1), Hkv = k.size(1);
        if (Hkv > 0 && H % Hkv == 0 && k_hint > 0) {
            const size_t bytes = tecoops::fa::workspace_bytes(static_cast<int>(batch), static_cast<int>(H),
                                                              static_cast<int>(Hkv), static_cast<int>(q.size(2)),
                                                              q_hint, k_hint);
            if (bytes > 0) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
        }
    }
    if (!ws.defined()) {
        q_hint = static_cast<int>(max_seqlen_q);
        k_hint = static_cast<int>(max_seqlen_k);
    }
    check(tecoopsFlashAttentionEx(handle_for(q), q_hint, k_hint, nullptr,
                                  cu_seqlens_q.data_ptr<int>(), seqused_k.data_ptr<int>(), bt.d,
                                  block_table.data_ptr(), qd.d, q.data_ptr(), kd.d, k.data_ptr(),
                                  vd.d, v.data_ptr(), od.d, out.data_ptr(),
                                  softmax_scale > 0 ? static_cast<float>(softmax_scale) : -1.0f,
                                  causal ? 1 : 0, ws.defined() ? ws.data_ptr() : nullptr),
          "flash_attn_varlen_func");
}

// reference torch_ext.cpp:167-206; x / out [dim, tokens], weight [width, dim]
void causal_conv1d_fn_torch(Tensor &out, Tensor &conv_states, const Tensor &x,
                            const Tensor &weight, const Tensor &query_start_loc,
                            const Tensor &cache_indices, const Tensor &has_initial_state,
                            int64_t pad_slot_id) {
    need_cuda({&out, &conv_states, &x, &weight, &query_start_loc, &cache_indices,
               &has_initial_state});
    const int dim = x.size(0), total = x.size(1);
    check(tecoopsCausalConv1dEx(handle_for(x), query_start_loc.size(0) - 1, total, dim,
                                weight.size(0), x.data_ptr(), 0, x.stride(1), x.stride(0),
                                out.data_ptr(), 0, out.stride(1), out.stride(0),
                                weight.data_ptr(), weight.stride(1), weight.stride(0), nullptr,
                                conv_states.data_ptr(), conv_states.stride(0),
                                query_start_loc.data_ptr<int>(), cache_indices.data_ptr<int>(),
                                has_initial_state.data_ptr<int8_t>(),
                                static_cast<int>(pad_slot_id), 0, 1),
          "causal_conv1d_fn_torch");
}

// ------------------------------------------------------------ extensions

void causal_conv1d(const Tensor &x, const Tensor &weight, const c10::optional<Tensor> &bias,
                   Tensor &out, const c10::optional<Tensor> &conv_states, bool silu) {
    need_cuda({&x, &weight, &out});
    check(tecoopsCausalConv1dEx(handle_for(x), x.size(0), x.size(2), x.size(1), weight.size(1),
                                x.data_ptr(), x.stride(0), x.stride(2), x.stride(1),
                                out.data_ptr(), out.stride(0), out.stride(2), out.stride(1),
                                weight.data_ptr(), weight.stride(0), weight.stride(1),
                                bias.has_value() ? bias->data_ptr() : nullptr,
                                conv_states.has_value() ? conv_states->data_ptr() : nullptr,
                                conv_states.has_value() ? conv_states->stride(0) : 0, nullptr,
                                nullptr, nullptr, -1, 0, silu ? 1 : 0),
          "causal_conv1d");
}

void rotary_embedding(const Tensor &positions, Tensor &query, const c10::optional<Tensor> &key,
                      int64_t head_size, const c10::optional<Tensor> &cos_sin_cache,
                      bool is_neox, double base, int64_t rot_dim) {
    need_cuda({&positions, &query});
    const int64_t T = positions.numel();
    const int H = query.numel() / (T * head_size);
    const int Hkv = key.has_value() ? key->numel() / (T * head_size) : 0;
    const int rd = rot_dim > 0 ? rot_dim
                               : (cos_sin_cache.has_value() ? cos_sin_cache->size(1) : head_size);
    check(tecoopsRotaryEmbedding(handle_for(query), positions.data_ptr<int64_t>(),
                                 query.data_ptr(), key.has_value() ? key->data_ptr() : nullptr,
                                 T, H, Hkv, head_size, rd, query.stride(0),
                                 key.has_value() ? key->stride(0) : 0,
                                 cos_sin_cache.has_value() ? cos_sin_cache->data_ptr<float>()
                                                           : nullptr,
                                 cos_sin_cache.has_value() ? cos_sin_cache->size(0) : 0,
                                 static_cast<float>(base), is_neox ? 1 : 0, dtype_of(query)),
          "rotary_embedding");
}

void rotary_reshape_and_cache(const Tensor &positions, Tensor &query, Tensor &key,
                              const Tensor &value, const Tensor &slot_mapping, Tensor &key_cache,
                              Tensor &value_cache, int64_t head_size,
                              const c10::optional<Tensor> &cos_sin_cache, bool is_neox,
                              double base, int64_t rot_dim, bool write_key) {
    need_cuda({&positions, &query, &key, &value, &slot_mapping, &key_cache, &value_cache});
    const int64_t T = positions.numel();
    const int H = query.numel() / (T * head_size);
    const int Hkv = key.numel() / (T * head_size);
    const int rd = rot_dim > 0 ? rot_dim
                               : (cos_sin_cache.has_value() ? cos_sin_cache->size(1) : head_size);
    check(tecoopsRotaryReshapeAndCache(
              handle_for(query), positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(),
              value.data_ptr(), slot_mapping.data_ptr<int64_t>(), key_cache.data_ptr(),
              value_cache.data_ptr(), T, H, Hkv, head_size, rd, query.stride(0), key.stride(0),
              value.stride(0),
              cos_sin_cache.has_value() ? cos_sin_cache->data_ptr<float>() : nullptr,
              cos_sin_cache.has_value() ? cos_sin_cache->size(0) : 0, static_cast<float>(base),
              is_neox ? 1 : 0, key_cache.size(0), key_cache.size(2), write_key ? 1 : 0,
              dtype_of(query)),
          "rotary_reshape_and_cache");
}

void gemv(const Tensor &weight, const Tensor &x, Tensor &out) {
    need_cuda({&weight, &x, &out});
    need_contiguous({&weight, &x, &out});
    need_dtype(weight, x.scalar_type(), "weight");
    need_dtype(out, x.scalar_type(), "out");
    const int B = x.dim() == 2 ? x.size(0) : 1;
    TORCH_CHECK(weight.dim() == 2 && x.size(-1) == weight.size(1) &&
                    out.numel() == B * weight.size(0),
                "gemv: weight [N, K], x [B, K], out [B, N]");
    check(tecoopsGemv(handle_for(x), weight.data_ptr(), x.data_ptr(), out.data_ptr(), B,
                      weight.size(0), weight.size(1), dtype_of(x)),
          "gemv");
}

void gemv_int8(const Tensor &weight, const Tensor &scales, const Tensor &x, Tensor &out) {
    need_cuda({&weight, &scales, &x, &out});
    need_contiguous({&weight, &scales, &x, &out});
    need_dtype(weight, at::kChar, "weight");
    need_dtype(scales, at::kHalf, "scales");
    need_dtype(x, at::kHalf, "x");
    need_dtype(out, at::kHalf, "out");
    const int B = x.dim() == 2 ? x.size(0) : 1;
    TORCH_CHECK(weight.dim() == 2 && x.size(-1) == weight.size(1) &&
                    out.numel() == B * weight.size(0) && scales.numel() == weight.size(0),
                "gemv_int8: weight [N, K], scales [N], x [B, K], out [B, N]");
    check(tecoopsGemvInt8(handle_for(x), weight.data_ptr<int8_t>(), scales.data_ptr(),
                          x.data_ptr(), out.data_ptr(), B, weight.size(0), weight.size(1)),
          "gemv_int8");
}

// Rows packed, any distance apart: the distance in elements.
int64_t row_stride(const Tensor &t, int64_t rows, int64_t width, const char *name) {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == width &&
                    (width <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= width),
                "tecoops: ", name, " must be [", rows, ", ", width, "] with packed rows");
    return rows > 1 ? t.stride(0) : width;
}

void same_device(const Tensor &x, std::initializer_list<const Tensor *> ts) {
    for (const Tensor *t : ts)
        if (t && t->defined())
            TORCH_CHECK(t->device() == x.device(), "tecoops: tensors must be on one device");
}

const Tensor *given(const c10::optional<Tensor> &t) { return t.has_value() ? &*t : nullptr; }

int fits_int(int64_t v, const char *name) {
    TORCH_CHECK(v >= 0 && v <= 0x7fffffff, "tecoops: ", name, " is too large");
    return static_cast<int>(v);
}

tecoopsActivation_t activation_of(c10::string_view s) {
    if (s == "none") return TECOOPS_ACTIVATION_NONE;
    if (s == "relu") return TECOOPS_ACTIVATION_RELU;
    if (s == "silu") return TECOOPS_ACTIVATION_SILU;
    if (s == "gelu") return TECOOPS_ACTIVATION_GELU;
    if (s == "gelu_tanh") return TECOOPS_ACTIVATION_GELU_TANH;
    TORCH_CHECK(false, "tecoops: activation must be none, relu, silu, gelu or gelu_tanh, got ", s);
}

Tensor workspace_of(size_t bytes, const Tensor &like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

void linear(const Tensor &x, const Tensor &weight, Tensor &out, const c10::optional<Tensor> &bias,
            const c10::optional<Tensor> &residual, c10::string_view activation, bool gated) {
    const Tensor *b = given(bias), *r = given(residual);
    need_cuda({&x, &weight, &out, b, r});
    same_device(x, {&weight, &out, b, r});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const tecoopsDataType_t dt = dtype_of(x);
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 2 && out.dim() == 2,
                "linear: x [M, K], weight [N, K], out [M, N]");
    const int m = fits_int(out.size(0), "M"), n = fits_int(out.size(1), "N"),
              k = fits_int(weight.size(1), "K");
    TORCH_CHECK(weight.size(0) == (gated ? 2LL * n : n), "linear: weight must hold N rows, 2 N gated");
    need_contiguous({&weight, b});
    need_dtype(weight, x.scalar_type(), "weight");
    need_dtype(out, x.scalar_type(), "out");
    if (b) {
        need_dtype(*b, x.scalar_type(), "bias");
        TORCH_CHECK(b->numel() == weight.size(0), "linear: bias must hold an element per row of weight");
    }
    if (r) need_dtype(*r, x.scalar_type(), "residual");
    const int64_t xs = row_stride(x, m, k, "x"), os = row_stride(out, m, n, "out");
    const int64_t rs = r ? row_stride(*r, m, n, "residual") : 0;
    const tecoopsActivation_t act = activation_of(activation);
    if (m == 0) return;
    // of these tensors' plan alone: most products of few rows need none
    const size_t bytes = n > 0 && k > 0 ? tecoops::linear_workspace(m, n, k, gated,
        tecoops::linear_copies(k, xs, x.data_ptr(), weight.data_ptr())) : 0;
    const Tensor ws = workspace_of(bytes, x);
    check(tecoopsLinear(handle_for(x), x.data_ptr(), xs, weight.data_ptr(), b ? b->data_ptr() : nullptr,
                        r ? r->data_ptr() : nullptr, rs, out.data_ptr(), os, m, n, k, act, gated,
                        bytes ? ws.data_ptr() : nullptr, bytes, dt),
          "linear");
}

void moe_layer(const Tensor &x, const Tensor &w_in, const Tensor &w_out, const Tensor &router_logits,
               int64_t top_k, Tensor &out, bool renormalize, c10::string_view activation,
               const c10::optional<Tensor> &topk_ids, const c10::optional<Tensor> &topk_weights) {
    const Tensor *ids = given(topk_ids), *weights = given(topk_weights);
    need_cuda({&x, &w_in, &w_out, &router_logits, &out, ids, weights});
    same_device(x, {&w_in, &w_out, &router_logits, &out, ids, weights});
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    const tecoopsDataType_t dt = dtype_of(x);
    TORCH_CHECK(x.dim() == 2 && w_in.dim() == 3 && w_out.dim() == 3 && router_logits.dim() == 2,
                "moe_layer: x [T, H], w_in [E, 2I, H], w_out [E, H, I], router_logits [T, E]");
    const int t = fits_int(x.size(0), "T"), e = fits_int(w_out.size(0), "E"),
              h = fits_int(w_out.size(1), "H"), i = fits_int(w_out.size(2), "I"),
              k = static_cast<int>(std::min<int64_t>(std::max<int64_t>(top_k, -1), 1 << 20));
    TORCH_CHECK(w_in.size(0) == e && w_in.size(1) == 2LL * i && w_in.size(2) == h &&
                    router_logits.size(0) == t && router_logits.size(1) == e && out.dim() == 2 &&
                    out.size(0) == t && out.size(1) == h,
                "moe_layer: x [T, H], w_in [E, 2I, H], w_out [E, H, I], router_logits [T, E], out [T, H]");
    need_contiguous({&w_in, &w_out, &router_logits, &out, ids, weights});
    need_dtype(w_in, x.scalar_type(), "w_in");
    need_dtype(w_out, x.scalar_type(), "w_out");
    need_dtype(out, x.scalar_type(), "out");
    const bool wide = router_logits.scalar_type() == at::kFloat;
    if (!wide) need_dtype(router_logits, x.scalar_type(), "router_logits");
    for (const Tensor *o : {ids, weights})
        if (o)
            TORCH_CHECK(o->dim() == 2 && o->size(0) == t && o->size(1) == k,
                        "moe_layer: topk_ids and topk_weights must be [T, top_k]");
    if (ids) need_dtype(*ids, at::kInt, "topk_ids");
    if (weights) need_dtype(*weights, at::kFloat, "topk_weights");
    const int64_t xs = row_stride(x, t, h, "x");
    const tecoopsActivation_t act = activation_of(activation);
    if (t == 0) return;
    size_t bytes = 0;
    check(tecoopsGetMoeLayerWorkspaceSize(t, h, i, e, k, &bytes), "moe_layer");
    const Tensor ws = workspace_of(bytes, x);
    check(tecoopsMoeLayer(handle_for(x), x.data_ptr(), xs, w_in.data_ptr(), w_out.data_ptr(),
                          router_logits.data_ptr(), wide ? TECOOPS_DATA_FLOAT : dt, out.data_ptr(),
                          ids ? ids->data_ptr<int>() : nullptr,
                          weights ? weights->data_ptr<float>() : nullptr, t, h, i, e, k, renormalize,
                          act, ws.data_ptr(), bytes, dt),
          "moe_layer");
}

// The arguments of the rotary functions of several axes, checked.
struct AxesArgs {
    std::vector<int> sections;
    tecoopsRotaryLayout_t layout;
    int tokens, heads, kv_heads, rot_dim;
    int64_t position_stride, query_stride, key_stride;
    const float *table;
    int max_position;

    AxesArgs(const Tensor &positions, const Tensor &query, const Tensor *key, int64_t head_size,
             at::IntArrayRef sec, const Tensor *cos_sin_cache, int64_t rot, c10::string_view lay, bool flat = false) {
        need_cuda({&positions, &query, key, cos_sin_cache});
        same_device(query, {&positions, key, cos_sin_cache});
        need_dtype(positions, at::kLong, "positions");
        TORCH_CHECK(head_size > 0, "tecoops: head_size must be positive");
        // (flat: one axis may come as [tokens])
        const bool one = flat && positions.dim() == 1 && sec.size() == 1;
        TORCH_CHECK((one || (positions.dim() == 2 && positions.size(0) == static_cast<int64_t>(sec.size()))) &&
                        (positions.size(-1) <= 1 || positions.stride(-1) == 1),
                    "tecoops: positions must be [axes, tokens] with adjacent tokens, one axis per section");
        tokens = fits_int(positions.size(-1), "tokens");
        position_stride = sec.size() > 1 ? positions.stride(0) : tokens;
        for (int64_t s : sec) sections.push_back(static_cast<int>(std::min<int64_t>(std::max<int64_t>(s, -1), 1 << 20)));
        heads = rows(query, query, head_size, "query", &query_stride);
        kv_heads = 0;
        key_stride = 0;
        if (key) kv_heads = rows(*key, query, head_size, "key", &key_stride);
        table = nullptr;
        max_position = 0;
        rot_dim = fits_int(rot > 0 ? rot : head_size, "rot_dim");
        if (cos_sin_cache) {
            need_dtype(*cos_sin_cache, at::kFloat, "cos_sin_cache");
            need_contiguous({cos_sin_cache});
            TORCH_CHECK(cos_sin_cache->dim() == 2 && (rot <= 0 || rot == cos_sin_cache->size(1)),
                        "tecoops: cos_sin_cache must be [positions, rot_dim]");
            rot_dim = fits_int(cos_sin_cache->size(1), "rot_dim");
            table = cos_sin_cache->data_ptr<float>();
            max_position = fits_int(cos_sin_cache->size(0), "positions of cos_sin_cache");
        }
        if (lay == "contiguous") layout = TECOOPS_ROTARY_CONTIGUOUS;
        else if (lay == "interleaved") layout = TECOOPS_ROTARY_INTERLEAVED;
        else if (lay == "per_axis") layout = TECOOPS_ROTARY_PER_AXIS;
        else TORCH_CHECK(false, "tecoops: layout must be contiguous, interleaved or per_axis, got ", lay);
    }

    int rows(const Tensor &t, const Tensor &query, int64_t head_size, const char *name,
             int64_t *stride) const {
        need_dtype(t, query.scalar_type(), name);
        const int64_t row = t.dim() == 2 ? t.size(1) : t.dim() == 3 ? t.size(1) * t.size(2) : 0;
        TORCH_CHECK(row > 0 && t.size(0) == tokens && row % head_size == 0,
                    "tecoops: ", name, " must be [tokens, heads * head_size] or [tokens, heads, head_size]");
        TORCH_CHECK((t.dim() == 2 || t.size(1) <= 1 || t.stride(1) == t.size(2)) &&
                        (t.size(-1) <= 1 || t.stride(-1) == 1),
                    "tecoops: the heads of a token of ", name, " must be adjacent");
        *stride = tokens > 1 ? t.stride(0) : row;
        return fits_int(row / head_size, "heads");
    }
};

void rotary_embedding_axes(const Tensor &positions, Tensor &query, const c10::optional<Tensor> &key,
                           int64_t head_size, at::IntArrayRef sections,
                           const c10::optional<Tensor> &cos_sin_cache, bool is_neox, double base,
                           int64_t rot_dim, c10::string_view layout) {
    const Tensor *k = given(key);
    const AxesArgs a(positions, query, k, head_size, sections, given(cos_sin_cache), rot_dim, layout);
    if (a.tokens == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
    check(tecoopsRotaryEmbeddingAxes(
              handle_for(query), positions.data_ptr<int64_t>(), a.position_stride,
              static_cast<int>(a.sections.size()), a.sections.data(), a.layout, query.data_ptr(),
              k ? k->data_ptr() : nullptr, a.tokens, a.heads, a.kv_heads, head_size, a.rot_dim,
              a.query_stride, a.key_stride, a.table, a.max_position, static_cast<float>(base),
              is_neox ? 1 : 0, dtype_of(query)),
          "rotary_embedding_axes");
}

void rotary_axes_reshape_and_cache(const Tensor &positions, Tensor &query, Tensor &key,
                                   const Tensor &value, const Tensor &slot_mapping,
                                   Tensor &key_cache, Tensor &value_cache, int64_t head_size,
                                   at::IntArrayRef sections,
                                   const c10::optional<Tensor> &cos_sin_cache, bool is_neox,
                                   double base, int64_t rot_dim, c10::string_view layout,
                                   bool write_key) {
    const AxesArgs a(positions, query, &key, head_size, sections, given(cos_sin_cache), rot_dim, layout);
    need_cuda({&value, &slot_mapping, &key_cache, &value_cache});
    same_device(query, {&value, &slot_mapping, &key_cache, &value_cache});
    need_contiguous({&slot_mapping, &key_cache, &value_cache});
    need_dtype(slot_mapping, at::kLong, "slot_mapping");
    need_dtype(key_cache, query.scalar_type(), "key_cache");
    need_dtype(value_cache, query.scalar_type(), "value_cache");
    TORCH_CHECK(slot_mapping.numel() == a.tokens, "tecoops: slot_mapping must hold a slot per token");
    TORCH_CHECK(key_cache.dim() == 4 && key_cache.size(1) == a.kv_heads && key_cache.size(3) == head_size &&
                    value_cache.sizes() == key_cache.sizes(),
                "tecoops: caches must be [num_blocks, kv heads, block_size, head_size]");
    int64_t value_stride = 0;
    TORCH_CHECK(a.rows(value, query, head_size, "value", &value_stride) == a.kv_heads,
                "tecoops: value must match key");
    if (a.tokens == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
    check(tecoopsRotaryAxesReshapeAndCache(
              handle_for(query), positions.data_ptr<int64_t>(), a.position_stride,
              static_cast<int>(a.sections.size()), a.sections.data(), a.layout, query.data_ptr(),
              key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr<int64_t>(),
              key_cache.data_ptr(), value_cache.data_ptr(), a.tokens, a.heads, a.kv_heads, head_size,
              a.rot_dim, a.query_stride, a.key_stride, value_stride, a.table, a.max_position,
              static_cast<float>(base), is_neox ? 1 : 0, fits_int(key_cache.size(0), "num_blocks"),
              fits_int(key_cache.size(2), "block_size"), write_key ? 1 : 0, dtype_of(query)),
          "rotary_axes_reshape_and_cache");
}

// The positions and sections of a call in one or several axes: [tokens] and no
// sections is one axis that all frequencies turn by.
struct Axes {
    int64_t whole;  // the one section where none are given
    at::IntArrayRef sections;

    Axes(at::IntArrayRef sec, const Tensor *cos_sin_cache, int64_t head_size, int64_t rot) : sections(sec) {
        if (cos_sin_cache && cos_sin_cache->dim() == 2) rot = cos_sin_cache->size(1);
        whole = (rot > 0 ? rot : head_size) / 2;
        if (sections.empty()) sections = at::IntArrayRef(&whole, 1);
    }
    Axes(const Axes &) = delete;
};

void need_weight(const Tensor *w, const Tensor &query, int64_t head_size, const char *name) {
    TORCH_CHECK(w && w->dim() == 1 && w->size(0) == head_size, "tecoops: ", name, " must be [head_size]");
    need_dtype(*w, query.scalar_type(), name);
    need_contiguous({w});
}

void qk_norm_rotary(const Tensor &positions, Tensor &query, const c10::optional<Tensor> &key,
                    const Tensor &query_weight, const c10::optional<Tensor> &key_weight, int64_t head_size,
                    double eps, at::IntArrayRef sections, const c10::optional<Tensor> &cos_sin_cache,
                    bool is_neox, double base, int64_t rot_dim, c10::string_view layout) {
    const Tensor *k = given(key), *table = given(cos_sin_cache), *kw = given(key_weight);
    need_cuda({&positions, &query, k, &query_weight, kw});
    same_device(query, {&query_weight, kw});
    const Axes ax(sections, table, head_size, rot_dim);
    const AxesArgs a(positions, query, k, head_size, ax.sections, table, rot_dim, layout, true);
    need_weight(&query_weight, query, head_size, "query_weight");
    if (k) need_weight(kw, query, head_size, "key_weight");
    if (a.tokens == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
    check(tecoopsQkNormRotary(
              handle_for(query), positions.data_ptr<int64_t>(), a.position_stride,
              static_cast<int>(a.sections.size()), a.sections.data(), a.layout, query.data_ptr(),
              k ? k->data_ptr() : nullptr, query_weight.data_ptr(), k ? kw->data_ptr() : nullptr,
              static_cast<float>(eps), a.tokens, a.heads, a.kv_heads, fits_int(head_size, "head_size"), a.rot_dim,
              a.query_stride, a.key_stride, a.table, a.max_position, static_cast<float>(base), is_neox ? 1 : 0,
              dtype_of(query)),
          "qk_norm_rotary");
}

void qk_norm_rotary_reshape_and_cache(const Tensor &positions, Tensor &query, Tensor &key, const Tensor &value,
                                      const Tensor &query_weight, const Tensor &key_weight,
                                      const Tensor &slot_mapping, Tensor &key_cache, Tensor &value_cache,
                                      int64_t head_size, double eps, at::IntArrayRef sections,
                                      const c10::optional<Tensor> &cos_sin_cache, bool is_neox, double base,
                                      int64_t rot_dim, c10::string_view layout, bool write_key) {
    const Tensor *table = given(cos_sin_cache);
    need_cuda({&positions, &query, &key, &value, &query_weight, &key_weight, &slot_mapping, &key_cache, &value_cache});
    same_device(query, {&query_weight, &key_weight, &value, &slot_mapping, &key_cache, &value_cache});
    const Axes ax(sections, table, head_size, rot_dim);
    const AxesArgs a(positions, query, &key, head_size, ax.sections, table, rot_dim, layout, true);
    need_weight(&query_weight, query, head_size, "query_weight");
    need_weight(&key_weight, query, head_size, "key_weight");
    need_contiguous({&slot_mapping, &key_cache, &value_cache});
    need_dtype(slot_mapping, at::kLong, "slot_mapping");
    need_dtype(key_cache, query.scalar_type(), "key_cache");
    need_dtype(value_cache, query.scalar_type(), "value_cache");
    TORCH_CHECK(slot_mapping.numel() == a.tokens, "tecoops: slot_mapping must hold a slot per token");
    TORCH_CHECK(key_cache.dim() == 4 && key_cache.size(1) == a.kv_heads && key_cache.size(3) == head_size &&
                    value_cache.sizes() == key_cache.sizes(),
                "tecoops: caches must be [num_blocks, kv heads, block_size, head_size]");
    int64_t value_stride = 0;
    TORCH_CHECK(a.rows(value, query, head_size, "value", &value_stride) == a.kv_heads,
                "tecoops: value must match key");
    if (a.tokens == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(query.device());
    check(tecoopsQkNormRotaryReshapeAndCache(
              handle_for(query), positions.data_ptr<int64_t>(), a.position_stride,
              static_cast<int>(a.sections.size()), a.sections.data(), a.layout, query.data_ptr(), key.data_ptr(),
              value.data_ptr(), query_weight.data_ptr(), key_weight.data_ptr(), static_cast<float>(eps),
              slot_mapping.data_ptr<int64_t>(), key_cache.data_ptr(), value_cache.data_ptr(), a.tokens, a.heads,
              a.kv_heads, fits_int(head_size, "head_size"), a.rot_dim, a.query_stride, a.key_stride, value_stride,
              a.table, a.max_position, static_cast<float>(base), is_neox ? 1 : 0,
              fits_int(key_cache.size(0), "num_blocks"), fits_int(key_cache.size(2), "block_size"),
              write_key ? 1 : 0, dtype_of(query)),
          "qk_norm_rotary_reshape_and_cache");
}

// The four tensors of a 4-bit cache of `like`'s type, checked.
void need_cache_int4(const Tensor &key_cache, const Tensor &value_cache, const Tensor &key_scales,
                     const Tensor &value_scales, const Tensor &like, int64_t head_size) {
    need_cuda({&key_cache, &value_cache, &key_scales, &value_scales});
    same_device(like, {&key_cache, &value_cache, &key_scales, &value_scales});
    need_contiguous({&key_cache, &value_cache, &key_scales, &value_scales});
    need_dtype(key_cache, at::kByte, "key_cache");
    need_dtype(value_cache, at::kByte, "value_cache");
    need_dtype(key_scales, like.scalar_type(), "key_scales");
    need_dtype(value_scales, like.scalar_type(), "value_scales");
    TORCH_CHECK(key_cache.dim() == 4 && 2 * key_cache.size(3) == head_size && value_cache.sizes() == key_cache.sizes(),
                "tecoops: caches must be uint8 [num_blocks, kv heads, block_size, head_size / 2]");
    TORCH_CHECK(key_scales.dim() == 4 && key_scales.size(0) == key_cache.size(0) &&
                    key_scales.size(1) == key_cache.size(1) && key_scales.size(2) == key_cache.size(2) &&
                    key_scales.size(3) == 2 && value_scales.sizes() == key_scales.sizes(),
                "tecoops: scales must be [num_blocks, kv heads, block_size, 2]");
}

// [tokens, heads, head_size] with packed heads, tokens any distance apart: the distance.
int64_t token_stride(const Tensor &t, const char *name) {
    const int64_t row = t.size(1) * t.size(2);
    TORCH_CHECK((t.size(2) <= 1 || t.stride(2) == 1) && (t.size(1) <= 1 || t.stride(1) == t.size(2)) &&
                    (t.size(0) <= 1 || t.stride(0) >= row),
                "tecoops: the heads of a token of ", name, " must be adjacent");
    return t.size(0) > 1 ? t.stride(0) : row;
}

void reshape_and_cache_int4(const Tensor &key, const Tensor &value, const Tensor &slot_mapping, Tensor &key_cache,
                            Tensor &value_cache, Tensor &key_scales, Tensor &value_scales) {
    need_cuda({&key, &value, &slot_mapping});
    same_device(key, {&value, &slot_mapping});
    const tecoopsDataType_t dt = dtype_of(key);
    need_dtype(value, key.scalar_type(), "value");
    need_dtype(slot_mapping, at::kLong, "slot_mapping");
    need_contiguous({&slot_mapping});
    TORCH_CHECK(key.dim() == 3 && value.sizes() == key.sizes() && slot_mapping.numel() == key.size(0),
                "reshape_and_cache_int4: key / value [tokens, kv heads, head_size], slot_mapping [tokens]");
    need_cache_int4(key_cache, value_cache, key_scales, value_scales, key, key.size(2));
    TORCH_CHECK(key_cache.size(1) == key.size(1), "reshape_and_cache_int4: the caches' kv heads must be key's");
    const int64_t ks = token_stride(key, "key"), vs = token_stride(value, "value");
    if (key.size(0) == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(key.device());
    check(tecoopsReshapeAndCacheInt4(
              handle_for(key), key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr<int64_t>(), key_cache.data_ptr(),
              value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), fits_int(key.size(0), "tokens"),
              fits_int(key.size(1), "kv heads"), fits_int(key.size(2), "head_size"), ks, vs,
              fits_int(key_cache.size(0), "num_blocks"), fits_int(key_cache.size(2), "block_size"), dt),
          "reshape_and_cache_int4");
}

void flash_attn_varlen_int4(const Tensor &q, const Tensor &key_cache, const Tensor &value_cache,
                            const Tensor &key_scales, const Tensor &value_scales, int64_t max_seqlen_q,
                            const Tensor &cu_seqlens_q, int64_t max_seqlen_k, const Tensor &seqused_k,
                            double softmax_scale, bool causal, const Tensor &block_table, Tensor &out) {
    need_cuda({&q, &cu_seqlens_q, &seqused_k, &block_table, &out});
    same_device(q, {&cu_seqlens_q, &seqused_k, &block_table, &out});
    const tecoopsDataType_t dt = dtype_of(q);
    TORCH_CHECK(q.dim() == 3 && out.sizes() == q.sizes(), "flash_attn_varlen_int4: q and out [rows, heads, head_size]");
    need_dtype(out, q.scalar_type(), "out");
    need_contiguous({&q, &out, &cu_seqlens_q, &seqused_k});
    need_cache_int4(key_cache, value_cache, key_scales, value_scales, q, q.size(2));
    need_dtype(cu_seqlens_q, at::kInt, "cu_seqlens_q");
    need_dtype(seqused_k, at::kInt, "seqused_k");
    need_dtype(block_table, at::kInt, "block_table");
    const int64_t batch = seqused_k.numel();
    TORCH_CHECK(batch > 0 && cu_seqlens_q.numel() == batch + 1 && block_table.dim() == 2 &&
                    block_table.size(0) == batch && (block_table.size(1) <= 1 || block_table.stride(1) == 1),
                "flash_attn_varlen_int4: cu_seqlens_q [batch + 1], seqused_k [batch], block_table [batch, blocks] "
                "with adjacent entries in a row");
    const auto bound = [](int64_t v) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(v, 0), 0x7fffffff)); };
    const int total = fits_int(q.size(0), "rows"), heads = fits_int(q.size(1), "heads"),
              kv_heads = fits_int(key_cache.size(1), "kv heads"), head_size = fits_int(q.size(2), "head_size");
    const int most_q = bound(max_seqlen_q);
    // (keys that the table can name bound those of a sequence)
    const int64_t cap = std::max<int64_t>(1, std::min<int64_t>(block_table.size(1) * key_cache.size(2), 0x7fffffff));
    const int most_k = static_cast<int>(max_seqlen_k > 0 ? std::min(max_seqlen_k, cap) : cap);
    if (total == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q.device());
    size_t bytes = 0;
    check(tecoopsGetFlashAttentionInt4WorkspaceSize(static_cast<int>(batch), total, heads, kv_heads, head_size, most_q,
                                                    most_k, &bytes),
          "flash_attn_varlen_int4");
    const Tensor ws = workspace_of(bytes, q);
    check(tecoopsFlashAttentionInt4(
              handle_for(q), most_q, most_k, cu_seqlens_q.data_ptr<int>(), seqused_k.data_ptr<int>(),
              block_table.data_ptr<int>(), block_table.size(0) > 1 ? block_table.stride(0) : block_table.size(1),
              static_cast<int>(batch), fits_int(block_table.size(1), "blocks"), q.data_ptr(), key_cache.data_ptr(),
              value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), out.data_ptr(), total, heads,
              kv_heads, head_size, fits_int(key_cache.size(0), "num_blocks"), fits_int(key_cache.size(2), "block_size"),
              softmax_scale > 0 ? static_cast<float>(softmax_scale) : -1.0f, causal ? 1 : 0,
              bytes ? ws.data_ptr() : nullptr, bytes, dt),
          "flash_attn_varlen_int4");
}

void gemv_int4(const Tensor &weight, const Tensor &scales, const Tensor &x, Tensor &out,
               const c10::optional<Tensor> &zeros) {
    const Tensor *z = given(zeros);
    need_cuda({&weight, &scales, &x, &out, z});
    same_device(x, {&weight, &scales, &out, z});
    need_contiguous({&weight, &scales, &x, &out, z});
    const tecoopsDataType_t dt = dtype_of(x);
    need_dtype(weight, at::kByte, "weight");
    need_dtype(scales, x.scalar_type(), "scales");
    need_dtype(out, x.scalar_type(), "out");
    TORCH_CHECK((x.dim() == 1 || x.dim() == 2) && weight.dim() == 2 && scales.dim() == 2,
                "gemv_int4: weight [N, K / 2], scales [N, K / group], x [B, K] or [K]");
    const int b = x.dim() == 2 ? fits_int(x.size(0), "B") : 1, n = fits_int(weight.size(0), "N"),
              k = fits_int(2 * weight.size(1), "K");
    TORCH_CHECK(x.size(-1) == k && out.numel() == static_cast<int64_t>(b) * n && scales.size(0) == n &&
                    scales.size(1) > 0 && k > 0 && k % scales.size(1) == 0,
                "gemv_int4: weight [N, K / 2], scales [N, K / group], x [B, K], out [B, N]");
    if (z) {
        need_dtype(*z, x.scalar_type(), "zeros");
        TORCH_CHECK(z->sizes() == scales.sizes(), "gemv_int4: zeros must match scales");
    }
    if (b == 0) return;
    const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(x.device());
    size_t bytes = 0;
    check(tecoopsGetGemvInt4WorkspaceSize(b, n, k, &bytes), "gemv_int4");
    const Tensor ws = workspace_of(bytes, x);
    check(tecoopsGemvInt4(handle_for(x), weight.data_ptr(), scales.data_ptr(), z ? z->data_ptr() : nullptr, x.data_ptr(),
                          out.data_ptr(), b, n, k, static_cast<int>(k / scales.size(1)), bytes ? ws.data_ptr() : nullptr,
                          bytes, dt),
          "gemv_int4");
}

void memset_(Tensor &t, int64_t value) {
    need_cuda({&t});
    check(tecoopsMemset(handle_for(t), t.data_ptr(), static_cast<int>(value),
                        t.numel() * t.element_size()),
          "memset");
}

}  // namespace

TORCH_LIBRARY(tecoops, m) {
    m.def("reshape_and_cache(Tensor key, Tensor value, Tensor slot_mapping, "
          "Tensor(a!) key_cache, Tensor(b!) value_cache) -> ()");
    m.def("rms_norm(Tensor input, Tensor weight, Tensor? residual, Tensor(a!) output, "
          "Tensor(b!)? residual_out, float eps) -> ()");
    m.def("flash_attn_varlen_func(Tensor q, Tensor k, Tensor v, int max_seqlen_q, "
          "Tensor cu_seqlens_q, int max_seqlen_k, Tensor? cu_seqlens_k, Tensor seqused_k, "
          "float softmax_scale, bool causal, Tensor? window_size, Tensor block_table, "
          "bool return_softmax_lse, Tensor(a!) out) -> ()");
    m.def("causal_conv1d_fn_torch(Tensor(a!) out, Tensor(b!) conv_states, Tensor x, "
          "Tensor weight, Tensor query_start_loc, Tensor cache_indices, "
          "Tensor has_initial_state, int pad_slot_id) -> ()");
    m.def("causal_conv1d(Tensor x, Tensor weight, Tensor? bias, Tensor(a!) out, "
          "Tensor(b!)? conv_states, bool silu) -> ()");
    m.def("rotary_embedding(Tensor positions, Tensor(a!) query, Tensor(b!)? key, int head_size, "
          "Tensor? cos_sin_cache, bool is_neox, float base, int rot_dim) -> ()");
    m.def("rotary_reshape_and_cache(Tensor positions, Tensor(a!) query, Tensor(b!) key, "
          "Tensor value, Tensor slot_mapping, Tensor(c!) key_cache, Tensor(d!) value_cache, "
          "int head_size, Tensor? cos_sin_cache, bool is_neox, float base, int rot_dim, "
          "bool write_key) -> ()");
    m.def("gemv(Tensor weight, Tensor x, Tensor(a!) out) -> ()");
    m.def("gemv_int8(Tensor weight, Tensor scales, Tensor x, Tensor(a!) out) -> ()");
    m.def("linear(Tensor x, Tensor weight, Tensor(a!) out, Tensor? bias, Tensor? residual, "
          "str activation, bool gated) -> ()");
    m.def("moe_layer(Tensor x, Tensor w_in, Tensor w_out, Tensor router_logits, int top_k, "
          "Tensor(a!) out, bool renormalize, str activation, Tensor(b!)? topk_ids, "
          "Tensor(c!)? topk_weights) -> ()");
    m.def("rotary_embedding_axes(Tensor positions, Tensor(a!) query, Tensor(b!)? key, "
          "int head_size, int[] sections, Tensor? cos_sin_cache, bool is_neox, float base, "
          "int rot_dim, str layout) -> ()");
    m.def("rotary_axes_reshape_and_cache(Tensor positions, Tensor(a!) query, Tensor(b!) key, "
          "Tensor value, Tensor slot_mapping, Tensor(c!) key_cache, Tensor(d!) value_cache, "
          "int head_size, int[] sections, Tensor? cos_sin_cache, bool is_neox, float base, "
          "int rot_dim, str layout, bool write_key) -> ()");
    m.def("qk_norm_rotary(Tensor positions, Tensor(a!) query, Tensor(b!)? key, Tensor query_weight, "
          "Tensor? key_weight, int head_size, float eps, int[] sections, Tensor? cos_sin_cache, "
          "bool is_neox, float base, int rot_dim, str layout) -> ()");
    m.def("qk_norm_rotary_reshape_and_cache(Tensor positions, Tensor(a!) query, Tensor(b!) key, "
          "Tensor value, Tensor query_weight, Tensor key_weight, Tensor slot_mapping, "
          "Tensor(c!) key_cache, Tensor(d!) value_cache, int head_size, float eps, int[] sections, "
          "Tensor? cos_sin_cache, bool is_neox, float base, int rot_dim, str layout, "
          "bool write_key) -> ()");
    m.def("reshape_and_cache_int4(Tensor key, Tensor value, Tensor slot_mapping, "
          "Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor(c!) key_scales, "
          "Tensor(d!) value_scales) -> ()");
    m.def("flash_attn_varlen_int4(Tensor q, Tensor key_cache, Tensor value_cache, Tensor key_scales, "
          "Tensor value_scales, int max_seqlen_q, Tensor cu_seqlens_q, int max_seqlen_k, "
          "Tensor seqused_k, float softmax_scale, bool causal, Tensor block_table, "
          "Tensor(a!) out) -> ()");
    m.def("gemv_int4(Tensor weight, Tensor scales, Tensor x, Tensor(a!) out, Tensor? zeros) -> ()");
    m.def("memset(Tensor(a!) t, int value) -> ()");
}

TORCH_LIBRARY_IMPL(tecoops, CUDA, m) {
    m.impl("reshape_and_cache", &reshape_and_cache);
    m.impl("rms_norm", &rms_norm);
    m.impl("flash_attn_varlen_func", &flash_attn_varlen_func);
    m.impl("causal_conv1d_fn_torch", &causal_conv1d_fn_torch);
    m.impl("causal_conv1d", &causal_conv1d);
    m.impl("rotary_embedding", &rotary_embedding);
    m.impl("rotary_reshape_and_cache", &rotary_reshape_and_cache);
    m.impl("gemv", &gemv);
    m.impl("gemv_int8", &gemv_int8);
    m.impl("linear", &linear);
    m.impl("moe_layer", &moe_layer);
    m.impl("rotary_embedding_axes", &rotary_embedding_axes);
    m.impl("rotary_axes_reshape_and_cache", &rotary_axes_reshape_and_cache);
    m.impl("qk_norm_rotary", &qk_norm_rotary);
    m.impl("qk_norm_rotary_reshape_and_cache", &qk_norm_rotary_reshape_and_cache);
    m.impl("reshape_and_cache_int4", &reshape_and_cache_int4);
    m.impl("flash_attn_varlen_int4", &flash_attn_varlen_int4);
    m.impl("gemv_int4", &gemv_int4);
    m.impl("memset", &memset_);
}
