// torch_serving.cpp -- the serving operators (include/hxq_serving.h) on torch
// tensors: checks, outputs and workspaces from PyTorch's allocator, the
// tensors' device and its current stream.  A Python extension
// (hxq_b200/_serving.so) because a decode step makes these calls hundreds of
// times: the same checks in Python and ctypes cost more host time than the
// kernels take (plan of 64 requests: 14 us a call, here 8.5 with the kernel).  The functions of
// libhxq.so are handed over by address (bind), so that there is one library in
// the process, whichever the binding loaded.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <map>
#include <optional>
#include <string>

#include "hxq_cuda.h"
#include "hxq_serving.h"

namespace py = pybind11;

namespace {

using MaybeTensor = std::optional<at::Tensor>;

struct Api {
    decltype(&hxq_cuda_kv_plan) plan;
    decltype(&hxq_cuda_kv_append) append;
    decltype(&hxq_cuda_kv_read) read;
    decltype(&hxq_cuda_kv_attention_workspace) attention_workspace;
    decltype(&hxq_cuda_kv_attention) attention;
    decltype(&hxq_lora_tiles) lora_tiles;
    decltype(&hxq_cuda_lora_plan) lora_plan;
    decltype(&hxq_cuda_lora_workspace) lora_workspace;
    decltype(&hxq_cuda_lora) lora;
    decltype(&hxq_error_string) error_string;
} api;

template <typename F> void take(F &f, const std::map<std::string, uintptr_t> &at, const char *name)
{
    const auto i = at.find(name);
    if (i == at.end() || i->second == 0) throw std::runtime_error(std::string("libhxq.so has no ") + name);
    f = reinterpret_cast<F>(i->second);
}

void bind(const std::map<std::string, uintptr_t> &at)
{
    take(api.plan, at, "hxq_cuda_kv_plan");
    take(api.append, at, "hxq_cuda_kv_append");
    take(api.read, at, "hxq_cuda_kv_read");
    take(api.attention_workspace, at, "hxq_cuda_kv_attention_workspace");
    take(api.attention, at, "hxq_cuda_kv_attention");
    take(api.lora_tiles, at, "hxq_lora_tiles");
    take(api.lora_plan, at, "hxq_cuda_lora_plan");
    take(api.lora_workspace, at, "hxq_cuda_lora_workspace");
    take(api.lora, at, "hxq_cuda_lora");
    take(api.error_string, at, "hxq_error_string");
}

void check(hxq_error_t err, const char *what)
{
    if (err != HXQ_OK)
        throw std::runtime_error(std::string(what) + ": hxq error " + std::to_string((int)err) + " (" + api.error_string(err) + ")");
}

void need(bool ok, const char *what)
{
    if (!ok) throw py::value_error(what);
}

// None of the operators has a gradient: where one would be expected, the call
// is refused rather than its part of the gradient left out.
void without_grad(std::initializer_list<const at::Tensor *> tensors)
{
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor *t : tensors)
        if (t->requires_grad())
            throw std::runtime_error("the serving operators have no gradient, and a tensor given requires one: call under torch.no_grad()");
}

// A tensor that a call writes: autograd and others who keep it see that it changed.
void changed(const at::Tensor &t)
{
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void changed(const MaybeTensor &t)
{
    if (t) changed(*t);
}

// Sizes go to the library in 32 bits.
void fits(std::initializer_list<int64_t> sizes)
{
    for (const int64_t n : sizes)
        if (n >= (int64_t(1) << 31)) throw py::value_error("a size of 2^31 or more");
}

void on_cuda(const at::Tensor &t, const char *name)
{
    if (!t.is_cuda()) throw py::value_error(std::string(name) + " must be a CUDA tensor");
}

void ints(const at::Tensor &t, const char *name, const at::Device &dev, int64_t dim = 1)
{
    if (t.scalar_type() != at::kInt || t.device() != dev || t.dim() != dim || !t.is_contiguous())
        throw py::value_error(std::string(name) + " must be a contiguous int32 tensor of " + std::to_string(dim) +
                              " dimension(s) on the same CUDA device");
}

const int32_t *i32(const at::Tensor &t) { return static_cast<const int32_t *>(t.data_ptr()); }

uint32_t *word(const MaybeTensor &status, const at::Device &dev)
{
    if (!status) return nullptr;
    need(status->element_size() == 4 && !status->is_floating_point() && status->device() == dev && status->numel() == 1,
         "status must be an int32 tensor of one element on the same CUDA device");
    return static_cast<uint32_t *>(status->data_ptr());
}

int elem_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
    case at::kFloat: return HXQ_ELEM_F32;
    case at::kBFloat16: return HXQ_ELEM_BF16;
    case at::kHalf: return HXQ_ELEM_F16;
    default: return -1;
    }
}

void *stream_of(const at::Device &dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

at::Tensor make(at::IntArrayRef size, at::ScalarType type, const at::Device &dev)
{
    return at::empty(size, at::TensorOptions().dtype(type).device(dev));
}

py::tuple kv_plan(const at::Tensor &fresh, const at::Tensor &cached, const at::Tensor &table, const at::Tensor &free_blocks,
                  int64_t block_tokens, int64_t n_slots, const MaybeTensor &status)
{
    on_cuda(fresh, "new");
    const at::Device dev = fresh.device();
    ints(fresh, "new", dev);
    ints(cached, "cached", dev);
    ints(free_blocks, "free", dev);
    ints(table, "table", dev, 2);
    const int64_t B = fresh.numel();
    fits({B, table.size(1), free_blocks.numel()});
    need(cached.numel() == B && table.size(0) == B, "new, cached and table must have one entry per request");
    need(block_tokens > 0 && block_tokens <= 65536 && n_slots >= 0 && n_slots < (int64_t(1) << 31), "block_tokens or n_slots out of range");
    const c10::cuda::OptionalCUDAGuard guard(dev);
    // one allocation: starts, lens, taken, slots, positions
    const at::Tensor buf = make({2 * B + 2 + 2 * n_slots}, at::kInt, dev);
    int32_t *at0 = static_cast<int32_t *>(buf.data_ptr());
    check(api.plan(i32(fresh), i32(cached), (uint32_t)B, static_cast<int32_t *>(table.data_ptr()), (uint32_t)table.size(1),
                   (uint32_t)block_tokens, i32(free_blocks), (uint32_t)free_blocks.numel(), at0, at0 + B + 1, at0 + 2 * B + 2,
                   at0 + 2 * B + 2 + n_slots, (uint32_t)n_slots, at0 + 2 * B + 1, word(status, dev), stream_of(dev)),
          "hxq_cuda_kv_plan");
    changed(table);
    changed(status);
    const auto part = buf.split_with_sizes({B + 1, B, 1, n_slots, n_slots});
    return py::make_tuple(part[0], part[1], part[3], part[4], part[2]);
}

class Cache {
public:
    Cache(at::Tensor k, at::Tensor v, at::Tensor k_scales, at::Tensor v_scales)
        : k_(std::move(k)), v_(std::move(v)), ks_(std::move(k_scales)), vs_(std::move(v_scales)), dev_(k_.device())
    {
        on_cuda(k_, "k");
        look();
    }

    void append(at::Tensor k, at::Tensor v, const at::Tensor &slots, const MaybeTensor &status)
    {
        look();
        rows(k, "k and v must be [tokens, n_heads, head_dim] in fp32, bf16 or f16 on the cache's device");
        rows(v, "k and v must be [tokens, n_heads, head_dim] in fp32, bf16 or f16 on the cache's device");
        ints(slots, "slots", dev_);
        fits({slots.numel()});
        need(k.scalar_type() == v.scalar_type() && k.size(0) == v.size(0) && k.size(0) == slots.numel(), "k, v and slots must go together");
        without_grad({&k, &v, &ks_, &vs_});
        const c10::cuda::OptionalCUDAGuard guard(dev_);
        check(api.append(&desc_, k.data_ptr(), v.data_ptr(), elem_of(k), k.stride(0), k.stride(1), v.stride(0), v.stride(1), i32(slots),
                         (uint32_t)slots.numel(), word(status, dev_), stream_of(dev_)),
              "hxq_cuda_kv_append");
        for (const at::Tensor *t : {&k_, &v_, &ks_, &vs_}) changed(*t);
        changed(status);
    }

    py::tuple read(const at::Tensor &slots, at::ScalarType dtype, const MaybeTensor &status)
    {
        look();
        ints(slots, "slots", dev_);
        fits({slots.numel()});
        need(dtype == at::kFloat || dtype == at::kBFloat16 || dtype == at::kHalf, "dtype must be fp32, bf16 or f16");
        without_grad({&ks_, &vs_});
        const c10::cuda::OptionalCUDAGuard guard(dev_);
        const at::Tensor out = make({2, slots.numel(), desc_.n_heads, desc_.head_dim}, dtype, dev_);
        at::Tensor k = out.select(0, 0), v = out.select(0, 1);
        check(api.read(&desc_, i32(slots), (uint32_t)slots.numel(), k.data_ptr(), v.data_ptr(), elem_of(out), word(status, dev_),
                       stream_of(dev_)),
              "hxq_cuda_kv_read");
        changed(status);
        return py::make_tuple(k, v);
    }

    at::Tensor attention(at::Tensor q, const at::Tensor &starts, const at::Tensor &lens, const at::Tensor &table, int64_t max_new,
                         std::optional<double> scale, int64_t window, bool causal, const MaybeTensor &out_or, const MaybeTensor &lse,
                         const MaybeTensor &status)
    {
        look();
        need(q.device() == dev_ && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && q.dim() == 3 &&
                 q.size(2) == desc_.head_dim && q.size(1) > 0 && q.size(1) % desc_.n_heads == 0,
             "q must be [rows, a multiple of the cache's heads, head_dim] in bf16 or f16 on the cache's device");
        without_grad({&q, &ks_, &vs_});
        if (out_or) without_grad({&*out_or});
        if (lse) without_grad({&*lse});
        if (q.stride(2) != 1 || ((q.stride(0) | q.stride(1)) & 7) != 0 || ((uintptr_t)q.data_ptr() & 15u) != 0)
            q = q.clone(at::MemoryFormat::Contiguous);
        ints(starts, "starts", dev_);
        ints(lens, "lens", dev_);
        ints(table, "table", dev_, 2);
        const int64_t B = lens.numel(), T = q.size(0);
        fits({B, T, q.size(1), table.size(1)});
        need(starts.numel() == B + 1 && table.size(0) == B, "starts must have one entry more than lens, table as many");
        need(window >= 0 && (causal || window == 0), "a window needs causal attention");
        need(max_new >= 0, "max_new must not be negative");
        need(!lse || (lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->dim() == 2 && lse->size(0) == T &&
                      lse->size(1) == q.size(1) && lse->device() == dev_),
             "lse must be fp32 [rows, heads]");
        const c10::cuda::OptionalCUDAGuard guard(dev_);
        need(!out_or || (out_or->sizes() == q.sizes() && out_or->scalar_type() == q.scalar_type() && out_or->device() == dev_ &&
                         out_or->stride(2) == 1),
             "out must be like q");
        const at::Tensor out = out_or ? *out_or : make(q.sizes(), q.scalar_type(), dev_);
        hxq_kv_attention_t a = {};
        a.d_q = q.data_ptr();
        a.d_out = out.data_ptr();
        a.d_lse = lse ? static_cast<float *>(lse->data_ptr()) : nullptr;
        a.q_stride_t = q.stride(0);
        a.q_stride_h = q.stride(1);
        a.out_stride_t = out.stride(0);
        a.out_stride_h = out.stride(1);
        a.d_starts = i32(starts);
        a.d_lens = i32(lens);
        a.d_table = i32(table);
        a.n_requests = (uint32_t)B;
        a.n_rows = (uint32_t)T;
        a.n_heads = (uint32_t)q.size(1);
        a.table_width = (uint32_t)table.size(1);
        a.max_new = (uint32_t)std::min<int64_t>(max_new, 0x7fffffff);
        a.window = (uint32_t)std::min<int64_t>(window, 0x7fffffff);
        a.scale = scale ? (float)*scale : 1.0f / std::sqrt((float)desc_.head_dim);
        a.elem = elem_of(q);
        a.causal = causal;
        const size_t size = api.attention_workspace(&desc_, &a);
        const at::Tensor ws = make({(int64_t)size}, at::kByte, dev_);
        check(api.attention(&desc_, &a, ws.data_ptr(), size, word(status, dev_), stream_of(dev_)), "hxq_cuda_kv_attention");
        changed(out_or);
        changed(lse);
        changed(status);
        return out;
    }

private:
    // The tensors as they are now: they may have been given other memory since the last call.
    void look()
    {
        const bool i8 = k_.scalar_type() == at::kChar, f8 = k_.scalar_type() == at::kFloat8_e4m3fn;
        need((i8 || f8) && v_.scalar_type() == k_.scalar_type(), "codes must be torch.int8 or torch.float8_e4m3fn");
        need(k_.dim() == 4 && v_.sizes() == k_.sizes(), "codes must be [n_blocks, n_heads, block_tokens, head_dim]");
        const int64_t blocks = k_.size(0), heads = k_.size(1), tokens = k_.size(2), dim = k_.size(3);
        need(dim == 64 || dim == 128 || dim == 256, "head_dim must be 64, 128 or 256");
        need(tokens % 16 == 0 && tokens > 0 && tokens <= 256, "block_tokens must be a multiple of 16, at most 256");
        need(blocks > 0 && heads > 0 && heads < 65536 && blocks * tokens < (int64_t(1) << 31), "cache too large or empty");
        for (const at::Tensor *t : {&ks_, &vs_})
            need(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == blocks && t->size(1) == heads,
                 "scales must be fp32 [n_blocks, n_heads]");
        for (const at::Tensor *t : {&k_, &v_, &ks_, &vs_})
            need(t->device() == dev_ && t->is_contiguous(), "the cache's tensors must be contiguous and on one device");
        need((((uintptr_t)k_.data_ptr() | (uintptr_t)v_.data_ptr()) & 15u) == 0, "codes must be 16-byte aligned");
        need(desc_.k == nullptr || (desc_.n_blocks == blocks && desc_.n_heads == heads && desc_.block_tokens == tokens &&
                                    desc_.head_dim == dim && desc_.format == (i8 ? HXQ_KV_INT8 : HXQ_KV_E4M3)),
             "the cache's tensors have another shape or type than it was made with");
        desc_ = {k_.data_ptr(), v_.data_ptr(), static_cast<float *>(ks_.data_ptr()), static_cast<float *>(vs_.data_ptr()),
                 (uint32_t)blocks, (uint32_t)heads, (uint32_t)tokens, (uint32_t)dim, (uint32_t)(i8 ? HXQ_KV_INT8 : HXQ_KV_E4M3)};
    }

    void rows(at::Tensor &t, const char *what) const
    {
        need(t.device() == dev_ && elem_of(t) >= 0 && t.dim() == 3 && t.size(1) == desc_.n_heads && t.size(2) == desc_.head_dim, what);
        if (t.stride(2) != 1) t = t.contiguous();
    }

    at::Tensor k_, v_, ks_, vs_;
    at::Device dev_;
    hxq_kv_cache_t desc_{};
};

std::pair<at::Tensor, int64_t> lora_plan(const at::Tensor &starts, const at::Tensor &adapters, int64_t n_adapters, int64_t n_tokens,
                                         const MaybeTensor &status)
{
    on_cuda(starts, "starts");
    const at::Device dev = starts.device();
    ints(starts, "starts", dev);
    ints(adapters, "adapters", dev);
    const int64_t B = adapters.numel();
    need(starts.numel() == B + 1, "starts must have one entry more than adapters");
    need(n_adapters > 0 && n_adapters <= HXQ_LORA_MAX_ADAPTERS && n_tokens >= 0 && n_tokens < (int64_t(1) << 31),
         "n_adapters or n_tokens out of range");
    need(B <= HXQ_LORA_MAX_REQUESTS, "too many requests");
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const int64_t tiles = api.lora_tiles((uint32_t)B, (uint32_t)n_adapters, (uint32_t)n_tokens);
    const at::Tensor buf = make({4 * tiles + n_tokens}, at::kInt, dev);
    int32_t *at0 = static_cast<int32_t *>(buf.data_ptr());
    check(api.lora_plan(i32(starts), i32(adapters), (uint32_t)B, (uint32_t)n_adapters, (uint32_t)n_tokens, at0 + 4 * tiles,
                        reinterpret_cast<hxq_lora_tile_t *>(at0), word(status, dev), stream_of(dev)),
          "hxq_cuda_lora_plan");
    changed(status);
    return {buf, tiles};
}

class Adapters {
public:
    Adapters(at::Tensor a, at::Tensor b, at::Tensor scales)
        : a_(std::move(a)), b_(std::move(b)), s_(std::move(scales)), dev_(a_.device())
    {
        on_cuda(a_, "a");
        look();
    }

    at::Tensor add(at::Tensor y, at::Tensor x, const at::Tensor &plan, int64_t n_tiles, int64_t n_tokens, int64_t n_requests,
                   int64_t n_adapters, const MaybeTensor &out_or)
    {
        look();
        need(x.device() == dev_ && x.scalar_type() == at::kBFloat16 && x.dim() == 2 && x.size(1) == desc_.in_features,
             "x must be bf16 [tokens, in_features] on the adapters' device");
        const int64_t T = x.size(0);
        fits({T, n_requests});
        need(y.device() == dev_ && y.scalar_type() == at::kFloat && y.dim() == 2 && y.size(0) == T && y.size(1) == desc_.out_features,
             "y must be fp32 [tokens, out_features] on the adapters' device");
        need(n_adapters == desc_.n_adapters && n_tokens == T && plan.device() == dev_ && plan.scalar_type() == at::kInt &&
                 plan.is_contiguous() && plan.numel() == 4 * n_tiles + n_tokens &&
                 n_tiles == api.lora_tiles((uint32_t)n_requests, desc_.n_adapters, (uint32_t)T),
             "the plan was made for other adapters or tokens");
        without_grad({&x, &y, &a_, &b_, &s_});
        if (out_or) without_grad({&*out_or});
        if (x.stride(1) != 1 || (x.stride(0) & 7) != 0 || ((uintptr_t)x.data_ptr() & 15u) != 0) x = x.clone(at::MemoryFormat::Contiguous);
        const c10::cuda::OptionalCUDAGuard guard(dev_);
        need(!out_or || (out_or->device() == dev_ && out_or->scalar_type() == at::kFloat && out_or->sizes() == y.sizes() &&
                         out_or->stride(1) == 1),
             "out must be like y, with consecutive elements");
        if (y.stride(1) != 1) y = y.contiguous();
        const at::Tensor out = out_or ? *out_or : make({T, (int64_t)desc_.out_features}, at::kFloat, dev_);
        const size_t size = api.lora_workspace(&desc_, (uint32_t)n_requests, (uint32_t)T);
        const at::Tensor ws = make({(int64_t)size}, at::kByte, dev_);
        const int32_t *at0 = i32(plan);
        check(api.lora(&desc_, static_cast<const uint16_t *>(x.data_ptr()), x.stride(0), static_cast<const float *>(y.data_ptr()),
                       y.stride(0), static_cast<float *>(out.data_ptr()), out.stride(0), (uint32_t)n_requests, (uint32_t)T,
                       at0 + 4 * n_tiles, reinterpret_cast<const hxq_lora_tile_t *>(at0), ws.data_ptr(), size, stream_of(dev_)),
              "hxq_cuda_lora");
        changed(out_or);
        return out;
    }

private:
    // The tensors as they are now: they may have been given other memory since the last call.
    void look()
    {
        need(a_.scalar_type() == at::kBFloat16 && b_.scalar_type() == at::kBFloat16 && a_.dim() == 3 && b_.dim() == 3,
             "a and b must be bf16 with three dimensions");
        const int64_t n = a_.size(0), r = a_.size(1), in = a_.size(2), out = b_.size(1);
        need(b_.size(0) == n && b_.size(2) == r, "b must be [n_adapters, out_features, rank]");
        need(r % 8 == 0 && r > 0 && r <= 128, "rank must be a multiple of 8, at most 128");
        need(in % 8 == 0 && in > 0 && out > 0 && in < 0x7fffff00 && out < 0x7fffff00, "in_features must be a multiple of 8");
        need(n > 0 && n <= HXQ_LORA_MAX_ADAPTERS, "between 1 and 4096 adapters");
        need(s_.scalar_type() == at::kFloat && s_.dim() == 1 && s_.size(0) == n, "scales must be fp32 [n_adapters]");
        for (const at::Tensor *t : {&a_, &b_, &s_})
            need(t->device() == dev_ && t->is_contiguous(), "the adapters' tensors must be contiguous and on one device");
        need((((uintptr_t)a_.data_ptr() | (uintptr_t)b_.data_ptr()) & 15u) == 0, "a and b must be 16-byte aligned");
        need(desc_.d_a == nullptr || (desc_.n_adapters == n && desc_.rank == r && desc_.in_features == in && desc_.out_features == out),
             "the adapters' tensors have another shape than they were made with");
        desc_ = {static_cast<const uint16_t *>(a_.data_ptr()), static_cast<const uint16_t *>(b_.data_ptr()),
                 static_cast<const float *>(s_.data_ptr()), (uint32_t)n, (uint32_t)r, (uint32_t)in, (uint32_t)out};
    }

    at::Tensor a_, b_, s_;
    at::Device dev_;
    hxq_lora_t desc_{};
};

}  // namespace

PYBIND11_MODULE(_serving, m)
{
    m.def("bind", &bind);
    m.def("kv_plan", &kv_plan);
    m.def("lora_plan", &lora_plan);
    py::class_<Cache>(m, "Cache")
        .def(py::init<at::Tensor, at::Tensor, at::Tensor, at::Tensor>())
        .def("append", &Cache::append)
        .def("read", &Cache::read)
        .def("attention", &Cache::attention);
    py::class_<Adapters>(m, "Adapters").def(py::init<at::Tensor, at::Tensor, at::Tensor>()).def("add", &Adapters::add);
}
