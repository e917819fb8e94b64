// PyTorch-ROCm extension `ff_attention`: the Python-visible class FastForwardAttn with the
// constructor, get_cache() and the three positional attention(...) overloads of the
// reference extension (torch_ffa_api.cpp:161-214), implemented on the C ABI of
// include/ffa_c_api.h.  torch is used for device memory and the current stream only.
//
// Differences from the reference, all on the side of refusing bad input:
//   - arguments are checked (device, dtype, element count, t < max_len) and C-ABI status
//     codes become Python exceptions; the reference prints and continues
//     (torch_ffa_api.cpp:101, :129, :154; attention.cu:1444-1451);
//   - kernels run on torch's current HIP stream instead of the legacy default stream
//     (attention.cu:1504);
//   - the launch plan is recomputed from t at every call instead of once from the prompt
//     length (torch_ffa_api.cpp:176).
#include <torch/extension.h>

// PyTorch-ROCm presents HIP devices under the device type "cuda"; these are the guard and
// stream accessors that understand that.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <tuple>
#include <utility>
#include <vector>

#include "ffa_c_api.h"

namespace {

void check_status(int st, const char* what) {
    TORCH_CHECK(st == FFA_OK, "ff_attention: ", what, " failed: ", ffa_status_string(st),
                " (status ", st, ")");
}

int precision_of(const torch::Tensor& x) {
    if (x.scalar_type() == torch::kHalf) return FFA_PRECISION_F16;
    if (x.scalar_type() == torch::kFloat) return FFA_PRECISION_F32;
    if (x.scalar_type() == torch::kBFloat16) return FFA_PRECISION_BF16;
    TORCH_CHECK(false, "ff_attention: unsupported tensor type ", x.scalar_type(),
                " (float16, bfloat16 and float32 are supported)");
}

// The planner knows two element sizes: bf16 plans like fp16.
int plan_precision(int precision) { return precision == FFA_PRECISION_BF16 ? FFA_PRECISION_F16 : precision; }

void* stream_of(const torch::Tensor& x) {
    return static_cast<void*>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream());
}

struct CacheDims {
    int B, H, Lmax, Dh;
};

// Every dimension is recovered from the K cache's 5-D shape, as the reference does
// (torch_ffa_api.cpp:112-115, :137-140).
CacheDims dims_of(const torch::Tensor& k_cache, const torch::Tensor& v_cache) {
    TORCH_CHECK(k_cache.dim() == 5, "ff_attention: k_cache must be [B,H,Dh/x,Lmax,x]");
    TORCH_CHECK(v_cache.dim() == 4, "ff_attention: v_cache must be [B,H,Lmax,Dh]");
    CacheDims d;
    d.B = (int)k_cache.size(0);
    d.H = (int)k_cache.size(1);
    d.Lmax = (int)k_cache.size(3);
    d.Dh = (int)(k_cache.size(2) * k_cache.size(4));
    TORCH_CHECK(k_cache.size(4) * k_cache.element_size() == 16,
                "ff_attention: last k_cache dimension must span 16 bytes");
    TORCH_CHECK(v_cache.size(0) == d.B && v_cache.size(1) == d.H && v_cache.size(2) == d.Lmax &&
                    v_cache.size(3) == d.Dh,
                "ff_attention: k_cache and v_cache shapes disagree");
    TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous(),
                "ff_attention: caches must be contiguous");
    return d;
}

torch::Tensor token_input(const torch::Tensor& x, const torch::Tensor& like, int64_t numel,
                          const char* name) {
    TORCH_CHECK(x.device() == like.device(), "ff_attention: ", name, " is on ", x.device(),
                " but the cache is on ", like.device());
    TORCH_CHECK(x.scalar_type() == like.scalar_type(), "ff_attention: ", name,
                " dtype differs from the cache dtype");
    TORCH_CHECK(x.numel() == numel, "ff_attention: ", name, " must hold B*H*Dh = ", numel,
                " elements, got ", x.numel());
    return x.contiguous();  // storage order [B,H,Dh]; no copy when already contiguous
}

// A contiguous tensor may start anywhere in its storage; the kernels read 16 bytes at a time.
torch::Tensor aligned_input(const torch::Tensor& x) {
    return (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0 ? x : x.clone();
}

// ---------------------------------------------------------------------------------------
// Operators next to the decode step.  None of them has a counterpart in the reference; they work on
// caches of the layouts get_cache() returns and keep nothing between calls: workspaces come from
// torch's allocator, which hands them out in stream order.
using OptTensor = c10::optional<torch::Tensor>;
using CachePair = std::pair<torch::Tensor, torch::Tensor>;
using CacheTriple = std::tuple<torch::Tensor, torch::Tensor, torch::Tensor>;

CacheDims checked_caches(const torch::Tensor& k_cache, const torch::Tensor& v_cache) {
    TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_cache.device() == v_cache.device() &&
                    k_cache.scalar_type() == v_cache.scalar_type(),
                "ff_attention: caches must be GPU tensors of one dtype on one device");
    const CacheDims d = dims_of(k_cache, v_cache);
    TORCH_CHECK(d.B > 0 && d.H > 0 && d.Lmax > 0 && d.Dh > 0, "ff_attention: empty caches");
    return d;
}

// An int32 tensor of `shape` on the caches' device; empty = not given.
torch::Tensor int_input(const OptTensor& x, const torch::Tensor& like, at::IntArrayRef shape, const char* name) {
    if (!x.has_value()) return torch::Tensor();
    TORCH_CHECK(x->device() == like.device() && x->scalar_type() == torch::kInt && x->sizes() == shape,
                "ff_attention: ", name, " must be an int32 tensor of shape ", shape, " on the caches' device");
    return x->contiguous();
}
const int* int_ptr(const torch::Tensor& x) { return x.defined() ? x.data_ptr<int>() : nullptr; }

// [B, heads, n, Dh] in any order of its first three dimensions; copied only if a row is not
// contiguous, not made of aligned 16-byte pieces, or too far from the next.
torch::Tensor group_input(const torch::Tensor& x, const torch::Tensor& like, const char* name) {
    TORCH_CHECK(x.device() == like.device() && x.scalar_type() == like.scalar_type(), "ff_attention: ", name,
                " must have the caches' dtype and device");
    const int64_t unit = 16 / x.element_size();
    bool fits = x.stride(3) == 1 && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0;
    for (int i = 0; i < 3; ++i) fits = fits && x.stride(i) % unit == 0;
    fits = fits && x.stride(2) * x.element_size() < (1 << 26);
    return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}

torch::Tensor scratch(size_t bytes, const torch::Tensor& like) {
    if (bytes == 0) return torch::Tensor();
    return torch::empty({(int64_t)bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(like.device()));
}

// Attention of a group of n new tokens a sample: q [B,Hq,n,Dh], k, v [B,H,n,Dh] -> [B,Hq,n,Dh].
torch::Tensor attention_tree(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                             torch::Tensor v_cache, float softmax_scale, int t, OptTensor parents, OptTensor first_keys,
                             OptTensor lengths, OptTensor counts) {
    const CacheDims d = checked_caches(k_cache, v_cache);
    TORCH_CHECK(q.dim() == 4 && q.size(0) == d.B && q.size(3) == d.Dh && q.size(1) > 0 && q.size(1) % d.H == 0,
                "ff_attention: q must be [B, Hq, n, Dh] with Hq a multiple of the caches' heads, got ", q.sizes());
    const int64_t n = q.size(2);
    TORCH_CHECK(n >= 1 && n <= FFA_MAX_TREE_TOKENS, "ff_attention: a group holds 1 to ", FFA_MAX_TREE_TOKENS,
                " new tokens a sample, got ", n);
    TORCH_CHECK(k.sizes() == at::IntArrayRef({d.B, d.H, n, d.Dh}) && v.sizes() == k.sizes(),
                "ff_attention: k and v must be [B, H, n, Dh] with q's n, got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK(t >= 0 && n <= d.Lmax && t <= d.Lmax - n, "ff_attention: ", n, " tokens at timestep ", t,
                " do not fit the cache [0, ", d.Lmax, ")");
    const int precision = precision_of(k_cache);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    q = group_input(q, k_cache, "q");
    k = group_input(k, k_cache, "k");
    v = group_input(v, k_cache, "v");
    const torch::Tensor par = int_input(parents, k_cache, {d.B, n}, "parents");
    const torch::Tensor fk = int_input(first_keys, k_cache, {d.B}, "first_keys");
    const torch::Tensor len = int_input(lengths, k_cache, {d.B}, "lengths");
    const torch::Tensor cnt = int_input(counts, k_cache, {d.B}, "counts");
    // Token-major in memory, so that [B, n, Hq * Dh] is a view; rows past a sample's count are zero.
    const int64_t Hq = q.size(1);
    torch::Tensor out = at::empty_strided({d.B, Hq, n, d.Dh}, {n * Hq * d.Dh, d.Dh, Hq * d.Dh, 1}, q.options());
    ffa_tree_tokens tt = {};
    tt.tokens = (int)n;
    tt.q_head_num = (int)Hq;
    tt.parents = int_ptr(par);
    tt.first_keys = int_ptr(fk);
    tt.lengths = int_ptr(len);
    tt.counts = int_ptr(cnt);
    tt.zero_rest = 1;
    for (int i = 0; i < 3; ++i) {
        tt.q_stride[i] = q.stride(i);
        tt.k_stride[i] = k.stride(i);
        tt.v_stride[i] = v.stride(i);
        tt.out_stride[i] = out.stride(i);
    }
    const size_t bytes = ffa_tree_workspace_bytes(precision, d.B, d.H, (int)Hq, d.Dh, (int)n, t);
    const torch::Tensor ws = scratch(bytes, k_cache);
    check_status(ffa_attention_tree(precision, d.B, d.H, d.Dh, d.Lmax, softmax_scale, t, &tt, q.data_ptr(), k.data_ptr(),
                                    v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                    bytes ? ws.data_ptr() : nullptr, bytes, stream_of(k_cache)),
                 "attention_tree");
    return out;
}

// The one-token step that adds its softmax weights to key_weights: q [B,Hq,Dh] -> [B,Hq,Dh].
torch::Tensor attention_weights(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                                torch::Tensor v_cache, float softmax_scale, int t, torch::Tensor key_weights,
                                OptTensor first_keys, OptTensor lengths) {
    const CacheDims d = checked_caches(k_cache, v_cache);
    const int64_t per = (int64_t)d.B * d.Dh;
    TORCH_CHECK(q.numel() > 0 && q.numel() % (per * d.H) == 0,
                "ff_attention: q must hold B*Hq*Dh elements with Hq a multiple of the caches' heads, got ", q.sizes());
    const int64_t Hq = q.numel() / per;
    TORCH_CHECK(t >= 0 && t < d.Lmax, "ff_attention: timestep ", t, " outside the cache [0, ", d.Lmax, ")");
    TORCH_CHECK(key_weights.device() == k_cache.device() && key_weights.scalar_type() == torch::kFloat &&
                    key_weights.is_contiguous() && key_weights.sizes() == at::IntArrayRef({d.B, d.H, d.Lmax}),
                "ff_attention: key_weights must be a contiguous float32 tensor [B, H, max_len] on the caches' device");
    const int precision = precision_of(k_cache);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
    q = aligned_input(token_input(q, k_cache, per * Hq, "q"));
    k = aligned_input(token_input(k, k_cache, per * d.H, "k"));
    v = aligned_input(token_input(v, k_cache, per * d.H, "v"));
    const torch::Tensor fk = int_input(first_keys, k_cache, {d.B}, "first_keys");
    const torch::Tensor len = int_input(lengths, k_cache, {d.B}, "lengths");
    torch::Tensor out = torch::empty({d.B, Hq, d.Dh}, q.options());
    const size_t bytes = ffa_weights_workspace_bytes(precision, d.B, d.H, (int)Hq, d.Dh, t);
    const torch::Tensor ws = scratch(bytes, k_cache);
    check_status(ffa_attention_weights(precision, d.B, d.H, (int)Hq, d.Dh, d.Lmax, softmax_scale, t, q.data_ptr(),
                                       k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                                       key_weights.data_ptr<float>(), int_ptr(fk), int_ptr(len),
                                       bytes ? ws.data_ptr() : nullptr, bytes, stream_of(k_cache)),
                 "attention_weights");
    return out;
}

// Caches of one shape, type and device, one a layer.
CacheDims layer_caches(const std::vector<CachePair>& caches) {
    TORCH_CHECK(!caches.empty(), "ff_attention: no caches");
    const CacheDims d = checked_caches(caches[0].first, caches[0].second);
    for (const auto& c : caches) {
        TORCH_CHECK(c.first.sizes() == caches[0].first.sizes() && c.first.scalar_type() == caches[0].first.scalar_type() &&
                        c.first.device() == caches[0].first.device(),
                    "ff_attention: the caches of a call must share shape, dtype and device");
        checked_caches(c.first, c.second);
    }
    return d;
}

// Moves the accepted path of every sample's tree behind its length, in all layers' caches.
void commit_tree(const std::vector<CachePair>& caches, int t, torch::Tensor path, torch::Tensor accepted,
                 OptTensor lengths) {
    const CacheDims d = layer_caches(caches);
    const torch::Tensor& like = caches[0].first;
    TORCH_CHECK(path.dim() == 2 && path.size(1) >= 1 && path.size(1) <= FFA_MAX_TREE_TOKENS,
                "ff_attention: path must be [B, 1 .. ", FFA_MAX_TREE_TOKENS, "], got ", path.sizes());
    const int64_t m = path.size(1);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(like.device());
    path = int_input(path, like, {d.B, m}, "path");
    accepted = int_input(accepted, like, {d.B}, "accepted");
    const torch::Tensor len = int_input(lengths, like, {d.B}, "lengths");
    std::vector<void*> k, v;
    for (const auto& c : caches) {
        k.push_back(c.first.data_ptr());
        v.push_back(c.second.data_ptr());
    }
    check_status(ffa_commit_tree(precision_of(like), (int)caches.size(), k.data(), v.data(), d.B, d.H, d.Dh, d.Lmax, t,
                                 path.data_ptr<int>(), (int)m, accepted.data_ptr<int>(), int_ptr(len), stream_of(like)),
                 "commit_tree");
}

// Keeps the last `recent` and the heaviest of the others, `keep` slots a pair in all; returns the
// old slots kept, int32 [caches, B, H, keep].
torch::Tensor evict(const std::vector<CachePair>& caches, const std::vector<torch::Tensor>& key_weights, int t, int keep,
                    int recent, OptTensor first_keys, OptTensor lengths, c10::optional<std::vector<CacheTriple>> into) {
    const CacheDims d = layer_caches(caches);
    const torch::Tensor& like = caches[0].first;
    TORCH_CHECK(key_weights.size() == caches.size() && (!into.has_value() || into->size() == caches.size()),
                "ff_attention: evict needs one tensor of weights, and one target if any, for each cache");
    std::vector<CachePair> to;
    std::vector<torch::Tensor> w_to;
    if (into.has_value()) {
        for (const auto& x : *into) {
            to.emplace_back(std::get<0>(x), std::get<1>(x));
            w_to.push_back(std::get<2>(x));
        }
    } else {
        to = caches;
        w_to = key_weights;
    }
    const CacheDims e = layer_caches(to);
    TORCH_CHECK(e.B == d.B && e.H == d.H && e.Dh == d.Dh && to[0].first.scalar_type() == like.scalar_type() &&
                    to[0].first.device() == like.device(),
                "ff_attention: a target differs from its cache in more than its length");
    auto check_weights = [&](const torch::Tensor& w, int len) {
        TORCH_CHECK(w.device() == like.device() && w.scalar_type() == torch::kFloat && w.is_contiguous() &&
                        w.sizes() == at::IntArrayRef({d.B, d.H, len}),
                    "ff_attention: weights must be contiguous float32 tensors [B, H, max_len] on the caches' device");
    };
    for (const auto& w : key_weights) check_weights(w, d.Lmax);
    for (const auto& w : w_to) check_weights(w, e.Lmax);
    TORCH_CHECK(t >= 0 && t <= d.Lmax, "ff_attention: ", t, " slots in a cache of ", d.Lmax);
    TORCH_CHECK(keep >= 1 && keep <= e.Lmax && recent >= 0 && recent <= keep, "ff_attention: evict wants 1 <= keep <= ",
                e.Lmax, " (the target's slots) and 0 <= recent <= keep, got keep ", keep, ", recent ", recent);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(like.device());
    const torch::Tensor fk = int_input(first_keys, like, {d.B}, "first_keys");
    const torch::Tensor len = int_input(lengths, like, {d.B}, "lengths");
    std::vector<const void*> k, v;
    std::vector<void*> k2, v2;
    std::vector<const float*> w;
    std::vector<float*> w2;
    for (size_t i = 0; i < caches.size(); ++i) {
        k.push_back(caches[i].first.data_ptr());
        v.push_back(caches[i].second.data_ptr());
        w.push_back(key_weights[i].data_ptr<float>());
        k2.push_back(to[i].first.data_ptr());
        v2.push_back(to[i].second.data_ptr());
        w2.push_back(w_to[i].data_ptr<float>());
    }
    torch::Tensor kept = torch::empty({(int64_t)caches.size(), d.B, d.H, keep}, like.options().dtype(torch::kInt));
    check_status(ffa_evict(precision_of(like), (int)caches.size(), k.data(), v.data(), w.data(), k2.data(), v2.data(),
                           w2.data(), d.B, d.H, d.Dh, d.Lmax, e.Lmax, t, keep, recent, int_ptr(fk), int_ptr(len),
                           kept.data_ptr<int>(), stream_of(like)),
                 "evict");
    return kept;
}

}  // namespace

struct FastForwardAttn {
    FastForwardAttn(torch::Tensor K, torch::Tensor V, int max_timesteps, bool _ft_kernel_launch) {
        TORCH_CHECK(K.is_cuda() && V.is_cuda(), "ff_attention: K and V must be GPU tensors");
        TORCH_CHECK(K.dim() == 4 && V.sizes() == K.sizes(),
                    "ff_attention: K and V must both be [B,H,L,Dh]");
        TORCH_CHECK(K.scalar_type() == V.scalar_type() && K.device() == V.device(),
                    "ff_attention: K and V must share dtype and device");
        const int precision = precision_of(K);
        const int B = (int)K.size(0), H = (int)K.size(1), L = (int)K.size(2), Dh = (int)K.size(3);
        TORCH_CHECK(max_timesteps >= L && max_timesteps > 0,
                    "ff_attention: max_timesteps (", max_timesteps, ") < prompt length (", L, ")");
        const int x = 16 / (int)K.element_size();
        TORCH_CHECK(Dh % x == 0, "ff_attention: head dim must be a multiple of ", x);

        c10::hip::HIPGuardMasqueradingAsCUDA guard(K.device());
        K = K.contiguous();
        V = V.contiguous();
        k_cache = torch::empty({B, H, Dh / x, max_timesteps, x}, K.options());
        v_cache = torch::empty({B, H, max_timesteps, Dh}, K.options());
        void* st = stream_of(K);
        int rc;
        if (precision != FFA_PRECISION_F32)  // fp16 and bf16 alike: cache construction moves 16-byte chunks
            rc = ffa_init_cache_f16((uint16_t*)k_cache.data_ptr(), (uint16_t*)v_cache.data_ptr(),
                                    (const uint16_t*)K.data_ptr(), (const uint16_t*)V.data_ptr(), B, L,
                                    max_timesteps, Dh, H, st);
        else
            rc = ffa_init_cache_f32((float*)k_cache.data_ptr(), (float*)v_cache.data_ptr(),
                                    (const float*)K.data_ptr(), (const float*)V.data_ptr(), B, L,
                                    max_timesteps, Dh, H, st);
        check_status(rc, "cache construction");
        ft_kernel_launch = _ft_kernel_launch;
        ensure_workspace(B, H, Dh, max_timesteps, K.device());
    }

    // attention(q, k, v, k_cache, v_cache, softmax_scale, t, p)      torch_ffa_api.cpp:179-182
    torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                            torch::Tensor v_cache, float softmax_scale, int curr_timestep,
                            float prob_thresh = 0) {
        return run(q, k, v, k_cache, v_cache, softmax_scale, curr_timestep, nullptr, prob_thresh, true,
                   nullptr, nullptr);
    }

    // attention(q, k, v, k_cache, v_cache, softmax_scale, t, seq_lengths, p): left-padded
    // batch, seq_lengths[b] = first real key (torch_ffa_api.cpp:184-187, :122).
    torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                            torch::Tensor v_cache, float softmax_scale, int curr_timestep,
                            torch::Tensor seq_lengths, float prob_thresh = 0) {
        return run(q, k, v, k_cache, v_cache, softmax_scale, curr_timestep, &seq_lengths, prob_thresh,
                   false, nullptr, nullptr);
    }

    // attention(q, k, v, softmax_scale, t, p)                         torch_ffa_api.cpp:189-192
    torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, float softmax_scale,
                            int curr_timestep, float prob_thresh = 0) {
        return run(q, k, v, k_cache, v_cache, softmax_scale, curr_timestep, nullptr, prob_thresh, true,
                   nullptr, nullptr);
    }

    std::pair<torch::Tensor, torch::Tensor> get_cache() { return std::make_pair(k_cache, v_cache); }

    // Not in the reference's Python surface: the step with the FasterTransformer features its host
    // code switches off (attention.cu:1472-1483) -- q/k/v bias [H,Dh] and the rotary embedding of
    // q and k over the first rotary_dim elements (GPT-J's pairing), applied to the new token
    // before it is attended and appended.  seq_lengths = None, or int32 [B] first real keys of
    // a left-padded batch; biases may be None.
    torch::Tensor attention_ex(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor k_cache,
                               torch::Tensor v_cache, float softmax_scale, int curr_timestep,
                               c10::optional<torch::Tensor> seq_lengths, float prob_thresh, int rotary_dim,
                               c10::optional<torch::Tensor> q_bias, c10::optional<torch::Tensor> k_bias,
                               c10::optional<torch::Tensor> v_bias, c10::optional<torch::Tensor> cache_indir,
                               int beam_width) {
        const CacheDims d = dims_of(k_cache, v_cache);
        torch::Tensor bias[3];
        const c10::optional<torch::Tensor>* in[3] = {&q_bias, &k_bias, &v_bias};
        ffa_token_transform tt = {nullptr, nullptr, nullptr, rotary_dim, 0.f};
        const void** slot[3] = {&tt.q_bias, &tt.k_bias, &tt.v_bias};
        for (int i = 0; i < 3; ++i) {
            if (!in[i]->has_value()) continue;
            bias[i] = token_input(in[i]->value(), k_cache, (int64_t)d.H * d.Dh, "bias");
            *slot[i] = bias[i].data_ptr();
        }
        torch::Tensor sl, indir;
        if (seq_lengths.has_value()) sl = seq_lengths.value();
        ffa_beam_indirection beams = {nullptr, beam_width};
        if (cache_indir.has_value()) {
            indir = cache_indir.value();
            TORCH_CHECK(indir.device() == k_cache.device() && indir.scalar_type() == torch::kInt &&
                            indir.is_contiguous() && indir.dim() == 2 && indir.size(0) == d.B &&
                            indir.size(1) == d.Lmax,
                        "ff_attention: cache_indir must be a contiguous int32 tensor [B, max_len] on the cache's device");
            beams.cache_indir = indir.data_ptr<int>();
        }
        return run(q, k, v, k_cache, v_cache, softmax_scale, curr_timestep, seq_lengths.has_value() ? &sl : nullptr,
                   prob_thresh, !seq_lengths.has_value(), nullptr, nullptr, &tt,
                   cache_indir.has_value() ? &beams : nullptr);
    }

    // Not in the reference: the same step plus what pruning dropped.
    // Returns (out [B,H,Dh], kept_count int32 [B,H], skip_mask uint8 [B,H,Lmax]).
    std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attention_diag(
        torch::Tensor q, torch::Tensor k, torch::Tensor v, float softmax_scale, int curr_timestep,
        float prob_thresh) {
        const CacheDims d = dims_of(k_cache, v_cache);
        auto kept = torch::zeros({d.B, d.H}, k_cache.options().dtype(torch::kInt32));
        auto mask = torch::zeros({d.B, d.H, d.Lmax}, k_cache.options().dtype(torch::kUInt8));
        auto out = run(q, k, v, k_cache, v_cache, softmax_scale, curr_timestep, nullptr, prob_thresh,
                       true, &kept, &mask);
        return std::make_tuple(out, kept, mask);
    }

    // Not in the reference: the plan the next call at (t, p) would use, as
    // (kind, waves_per_wg, threads_per_key, keys_per_wave, n_splits, tiles_per_split, combine,
    //  whole_heads).
    std::vector<int> launch_plan(int curr_timestep, float prob_thresh) {
        const CacheDims d = dims_of(k_cache, v_cache);
        ffa_launch_plan plan;
        check_status(ffa_plan_launch(plan_precision(precision_of(k_cache)), d.B, d.H, d.Dh, curr_timestep, prob_thresh,
                                     ft_kernel_launch ? 1 : 0, 0, &plan),
                     "launch planning");
        return {plan.kind, plan.waves_per_wg, plan.threads_per_key, plan.keys_per_wave, plan.n_splits,
                plan.tiles_per_split, plan.combine, plan.whole_heads};
    }

    torch::Tensor k_cache;
    torch::Tensor v_cache;
    torch::Tensor workspace;
    bool ft_kernel_launch;

private:
    void ensure_workspace(int B, int H, int Dh, int Lmax, const torch::Device& dev) {
        const size_t need = ffa_workspace_bytes(B, H, Dh, Lmax);
        if (workspace.defined() && workspace.device() == dev && (size_t)workspace.numel() >= need) return;
        // zeros(): the arrival counters must start at zero; the kernels restore that.
        workspace = torch::zeros({(int64_t)need}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
    }

    torch::Tensor run(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in,
                      torch::Tensor& kc, torch::Tensor& vc, float softmax_scale, int t,
                      const torch::Tensor* seq_lengths, float prob_thresh, bool right_or_no_padding,
                      torch::Tensor* kept, torch::Tensor* mask, const ffa_token_transform* transform = nullptr,
                      const ffa_beam_indirection* beams = nullptr) {
        TORCH_CHECK(kc.is_cuda() && vc.is_cuda() && kc.device() == vc.device() &&
                        kc.scalar_type() == vc.scalar_type(),
                    "ff_attention: caches must be GPU tensors of one dtype on one device");
        const CacheDims d = dims_of(kc, vc);
        const int precision = precision_of(kc);
        TORCH_CHECK(t >= 0 && t < d.Lmax, "ff_attention: timestep ", t, " outside the cache [0, ",
                    d.Lmax, ")");
        const int64_t numel = (int64_t)d.B * d.H * d.Dh;
        c10::hip::HIPGuardMasqueradingAsCUDA guard(kc.device());
        torch::Tensor q = token_input(q_in, kc, numel, "q");
        torch::Tensor k = token_input(k_in, kc, numel, "k");
        torch::Tensor v = token_input(v_in, kc, numel, "v");

        torch::Tensor sl;
        const int* sl_ptr = nullptr;
        if (seq_lengths != nullptr) {
            TORCH_CHECK(seq_lengths->device() == kc.device() && seq_lengths->scalar_type() == torch::kInt &&
                            seq_lengths->numel() == d.B,
                        "ff_attention: seq_lengths must be an int32 tensor of B entries on the cache's device");
            sl = seq_lengths->contiguous();
            sl_ptr = sl.data_ptr<int>();
        }

        ensure_workspace(d.B, d.H, d.Dh, d.Lmax, kc.device());
        torch::Tensor out = torch::empty({d.B, d.H, d.Dh}, q.options());

        ffa_launch_plan plan;
        const bool diag = kept != nullptr || mask != nullptr;
        // The default launch keeps diagnostics at any length; the exact split kernel has none.
        check_status(ffa_plan_launch(plan_precision(precision), d.B, d.H, d.Dh, t, prob_thresh,
                                     (ft_kernel_launch || diag) ? 1 : 0, 0, &plan),
                     "launch planning");
        if (transform != nullptr || beams != nullptr) {
            TORCH_CHECK(!diag, "ff_attention: diagnostics cannot be combined with a token transform or beams");
            check_status(ffa_attention_ex(precision, d.B, d.H, d.Dh, d.Lmax, softmax_scale, t, q.data_ptr(),
                                          k.data_ptr(), v.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr(),
                                          sl_ptr, prob_thresh, &plan, right_or_no_padding ? 1 : 0, transform, beams,
                                          workspace.data_ptr(), (size_t)workspace.numel(), stream_of(kc)),
                         "attention");
            return out;
        }
        const int rc = ffa_attention_diag(
            precision, d.B, d.H, d.Dh, d.Lmax, softmax_scale, t, q.data_ptr(), k.data_ptr(), v.data_ptr(),
            kc.data_ptr(), vc.data_ptr(), out.data_ptr(), sl_ptr, prob_thresh, &plan,
            right_or_no_padding ? 1 : 0, workspace.data_ptr(), (size_t)workspace.numel(),
            kept ? (uint32_t*)kept->data_ptr() : nullptr, mask ? (uint8_t*)mask->data_ptr() : nullptr,
            stream_of(kc));
        check_status(rc, "attention");
        return out;
    }
};

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "MI355X-native FastForwardAttention decode step (drop-in for ff_attention)";
    py::class_<FastForwardAttn>(m, "FastForwardAttn")
        .def(py::init<torch::Tensor, torch::Tensor, int, bool>())
        .def("get_cache", &FastForwardAttn::get_cache, "Get KV_cache")
        .def("attention",
             py::overload_cast<torch::Tensor, torch::Tensor, torch::Tensor, float, int, float>(
                 &FastForwardAttn::attention),
             "Attention forward, fixed timestep, cache held by the object")
        .def("attention",
             py::overload_cast<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor,
                               float, int, float>(&FastForwardAttn::attention),
             "Attention forward, fixed timestep")
        .def("attention",
             py::overload_cast<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor,
                               float, int, torch::Tensor, float>(&FastForwardAttn::attention),
             "Attention forward, left-padded batch")
        .def("attention_ex", &FastForwardAttn::attention_ex,
             "Attention forward with q/k/v bias and rotary embedding of the new token and, optionally, "
             "beam-search cache indirection (cache_indir int32 [B, max_len], beam_width)",
             py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
             py::arg("softmax_scale"), py::arg("curr_timestep"), py::arg("seq_lengths"), py::arg("prob_thresh"),
             py::arg("rotary_dim"), py::arg("q_bias"), py::arg("k_bias"), py::arg("v_bias"),
             py::arg("cache_indir") = py::none(), py::arg("beam_width") = 1)
        .def("attention_diag", &FastForwardAttn::attention_diag,
             "Attention forward plus (kept_count, skip_mask) of the pruning rule")
        .def_static("attention_tree", &attention_tree,
                    "Attention of a group of up to 64 new tokens a sample (a drafted tree, or a chain) over the caches "
                    "and the tokens' own ancestors; appends them.  q [B,Hq,n,Dh], k, v [B,H,n,Dh] -> [B,Hq,n,Dh]",
                    py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
                    py::arg("softmax_scale"), py::arg("curr_timestep"), py::arg("parents") = py::none(),
                    py::arg("first_keys") = py::none(), py::arg("lengths") = py::none(), py::arg("counts") = py::none())
        .def_static("commit_tree", &commit_tree,
                    "Moves the accepted path (path int32 [B,m], accepted int32 [B]) behind each sample's length in "
                    "every (k_cache, v_cache) of the list",
                    py::arg("caches"), py::arg("curr_timestep"), py::arg("path"), py::arg("accepted"),
                    py::arg("lengths") = py::none())
        .def_static("attention_weights", &attention_weights,
                    "Attention forward of one token that adds the softmax weight every key receives to key_weights "
                    "(float32 [B,H,max_len])",
                    py::arg("q"), py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("v_cache"),
                    py::arg("softmax_scale"), py::arg("curr_timestep"), py::arg("key_weights"),
                    py::arg("first_keys") = py::none(), py::arg("lengths") = py::none())
        .def_static("evict", &evict,
                    "Keeps, for every head, the last `recent` slots and the heaviest others, `keep` in all, in slot order "
                    "at the front of the caches (or of `into`, a list of (k_cache, v_cache, key_weights)); returns the "
                    "old slots kept, int32 [caches,B,H,keep]",
                    py::arg("caches"), py::arg("key_weights"), py::arg("curr_timestep"), py::arg("keep"),
                    py::arg("recent"), py::arg("first_keys") = py::none(), py::arg("lengths") = py::none(),
                    py::arg("into") = py::none())
        .def("launch_plan", &FastForwardAttn::launch_plan, "Launch plan for (t, p)");
}
