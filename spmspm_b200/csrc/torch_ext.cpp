// Python calls of the 4-bit operators, straight from tensors to the C entry points.
//
// A decode step makes these calls with kernels of a few microseconds, so that checking the arguments and marshalling them
// in Python took longer than the work (attention 17 us of host time, 7 from here; an append 3.3).  The checks are the wrappers' own:
// kind, type, shape, layout and device of every tensor; sizes and alignment are checked again behind the C boundary.  The
// library is the one spmspm_b200._lib has loaded.
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>

#include <cmath>
#include <cstdint>
#include <optional>
#include <string>

#include "../../include/spmm_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

PyObject* g_error = nullptr;
decltype(&spb_last_error) p_last_error;
decltype(&spb_kv_cache_bytes) p_kv_cache_bytes;
decltype(&spb_kv_append) p_kv_append;
decltype(&spb_kv_read) p_kv_read;
decltype(&spb_kv_attention) p_kv_attention;
decltype(&spb_kv_attention_workspace_bytes) p_kv_attention_workspace_bytes;
decltype(&spb_linear_int4) p_linear_int4;
decltype(&spb_int4_workspace_bytes) p_int4_workspace_bytes;
decltype(&spb_int4_bytes) p_int4_bytes;

[[noreturn]] void fail(const std::string& what)
{
    PyErr_SetString(g_error, what.c_str());
    throw py::error_already_set();
}
void check(int code, const char* name)
{
    if (code) fail(std::string(name) + " failed: cudaError " + std::to_string(code) + ": " + p_last_error());
}
std::string shape_text(at::IntArrayRef s)
{
    std::string t = "[";
    for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
    return t + "]";
}

// A size as the C entry points take it: what does not fit is refused, not cut.
int as_int(int64_t x, const char* name)
{
    if (x < INT32_MIN || x > INT32_MAX) fail(std::string(name) + " is out of range: " + std::to_string(x));
    return (int)x;
}

void init(const std::string& path, py::object error)
{
    void* lib = dlopen(path.c_str(), RTLD_NOW);
    if (!lib) throw std::runtime_error(dlerror());
    auto get = [&](auto& f, const char* name) {
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(lib, name));
        if (!f) throw std::runtime_error(std::string(name) + " is missing in " + path);
    };
    get(p_last_error, "spb_last_error");
    get(p_kv_cache_bytes, "spb_kv_cache_bytes");
    get(p_kv_append, "spb_kv_append");
    get(p_kv_read, "spb_kv_read");
    get(p_kv_attention, "spb_kv_attention");
    get(p_kv_attention_workspace_bytes, "spb_kv_attention_workspace_bytes");
    get(p_linear_int4, "spb_linear_int4");
    get(p_int4_workspace_bytes, "spb_int4_workspace_bytes");
    get(p_int4_bytes, "spb_int4_bytes");
    g_error = error.release().ptr();
}

// at::empty without the dispatcher's detour (0.6 us instead of 1.1; a call with one launch takes 3).
Tensor make(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) { return Tensor(at::detail::empty_cuda(shape, type, dev, std::nullopt)); }

// Device and stream of a call: the tensors' device is made current, and with it the stream, the given one or torch's current one there.
// Outputs and workspaces are then of that stream's pool: memory of another one may still be in use there, and goes back to it while this
// stream is at work.
struct Place {
    c10::cuda::CUDAGuard guard;
    c10::cuda::CUDAStream caller, stream;
    std::optional<c10::cuda::CUDAStreamGuard> given;
    Place(int dev, std::optional<int64_t> s)
        : guard((c10::DeviceIndex)dev),
          caller(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev)),
          stream(s ? c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(*s), (c10::DeviceIndex)dev) : caller)
    {
        // beside a capture of the caller's stream nothing can be allocated outside the graph's pool
        if (s && (!captured(caller) || captured(stream))) given.emplace(stream.unwrap());
    }
    static bool captured(c10::cuda::CUDAStream s)
    {
        cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
        C10_CUDA_CHECK(cudaStreamIsCapturing(s.stream(), &status));
        return status != cudaStreamCaptureStatusNone;
    }
    void* ptr() const { return stream.stream(); }
    Tensor output(at::IntArrayRef shape, c10::Device dev) const
    {
        Tensor t = make(shape, at::kHalf, dev);
        if (given && t.numel()) t.record_stream(caller.unwrap());   // not used anew before the caller's stream, too, is done with it
        return t;
    }
};
// Workspace of the caller, or a new one.
Tensor pick_workspace(const OptTensor& given, size_t need, const Tensor& like, const char* where, size_t& have)
{
    if (!given) {
        have = need;
        return need ? make({(int64_t)need}, at::kByte, like.device()) : Tensor();
    }
    have = given->nbytes();
    if (!given->is_cuda() || given->device() != like.device() || !given->is_contiguous() || have < need)
        fail("the workspace must be a contiguous CUDA tensor of at least " + std::to_string(need) + " bytes on the " + where + "'s device");
    return *given;
}
void dense_half(const Tensor& t, const char* name, at::IntArrayRef shape, c10::Device dev, const char* where)
{
    if (t.device() != dev || t.scalar_type() != at::kHalf || !t.is_contiguous() || t.sizes() != shape)
        fail(std::string(name) + " must be a contiguous CUDA float16 " + shape_text(shape) + " tensor on the " + where + "'s device");
}

// ---------------------------------------------------------------------------------------------------- 4-bit cache

struct Cache {
    Tensor pool;
    int num_pages, page_size, kv_heads, head_dim;
};
// The pool as the kernels take it.  A saved cache may be loaded without a device, but is used on one.
void check_pool(const Cache& c)
{
    if (!c.pool.is_cuda()) fail("the cache lives on a CUDA device, its pool is on " + c.pool.device().str());
    if (c.pool.scalar_type() != at::kByte || !c.pool.is_contiguous() ||
        c.pool.nbytes() < p_kv_cache_bytes(c.num_pages, c.page_size, c.kv_heads, c.head_dim))
        fail("the cache's pool must be a contiguous uint8 tensor of spb_kv_cache_bytes bytes");
}
struct Batch {
    const int *table, *lens, *cu;
    int width, batch;
};
Batch check_batch(const Cache& c, const Tensor& table, const Tensor& lens, const OptTensor& cu)
{
    check_pool(c);
    const auto dev = c.pool.device();
    if (table.device() != dev || table.scalar_type() != at::kInt || table.dim() != 2 || !table.is_contiguous() || !table.numel())
        fail("page_table must be a contiguous CUDA int32 [batch, pages] tensor on the cache's device");
    const int64_t n = table.size(0);
    if (n > 65535) fail("page_table has " + std::to_string(n) + " sequences, at most 65535 are taken");
    const int width = as_int(table.size(1), "the width of page_table");
    if (lens.device() != dev || lens.scalar_type() != at::kInt || lens.dim() != 1 || lens.size(0) != n || !lens.is_contiguous())
        fail("kv_lens must be a contiguous CUDA int32 [" + std::to_string(n) + "] tensor on the cache's device");
    if (cu && (cu->device() != dev || cu->scalar_type() != at::kInt || cu->dim() != 1 || cu->size(0) != n + 1 || !cu->is_contiguous()))
        fail("cu_q must be a contiguous CUDA int32 [" + std::to_string(n + 1) + "] tensor on the cache's device");
    return {table.const_data_ptr<int>(), lens.const_data_ptr<int>(), cu ? cu->const_data_ptr<int>() : nullptr, width, (int)n};
}
// [tokens, heads, head_dim] with contiguous channels and strides that hold four channels together
const uint16_t* check_vectors(const Cache& c, const Tensor& t, const char* name, int64_t tokens, int64_t heads)
{
    if (t.device() != c.pool.device() || t.scalar_type() != at::kHalf || t.dim() != 3 || t.size(2) != c.head_dim || (heads >= 0 && t.size(1) != heads) ||
        (tokens >= 0 && t.size(0) != tokens))
        fail(std::string(name) + " must be a CUDA float16 [" + (tokens >= 0 ? std::to_string(tokens) : "tokens") + ", " +
             (heads >= 0 ? std::to_string(heads) : "heads") + ", " + std::to_string(c.head_dim) + "] tensor on the cache's device");
    const auto* p = static_cast<const uint16_t*>(t.const_data_ptr());
    if (t.numel() && (t.stride(2) != 1 || t.stride(0) & 3 || t.stride(1) & 3 || reinterpret_cast<uintptr_t>(p) & 7))
        fail(std::string(name) + " must have contiguous channels, strides that are multiples of 4 and an 8-byte aligned start");
    return p;
}
void check_rows(int64_t n, const Batch& b)
{
    if (!b.cu && n % b.batch) fail("without cu_q the tokens must divide evenly among the sequences");
}

OptTensor kv_append(const Cache& c, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lens, const OptTensor& cu, const OptTensor& q,
                    const OptTensor& cos, const OptTensor& sin, bool interleaved, const OptTensor& q_out, std::optional<int64_t> stream)
{
    const Batch b = check_batch(c, table, lens, cu);
    const uint16_t* kp = check_vectors(c, k, "k", -1, c.kv_heads);
    const int64_t n = k.size(0);
    const uint16_t* vp = check_vectors(c, v, "v", n, c.kv_heads);
    check_rows(n, b);
    if (cos.has_value() != sin.has_value()) fail("cos and sin are given together");
    int64_t rot = 0, max_pos = 0;
    if (cos) {
        for (const auto* t : {&*cos, &*sin})
            if (t->device() != c.pool.device() || t->scalar_type() != at::kFloat || t->dim() != 2 || !t->is_contiguous() || t->sizes() != cos->sizes() || !t->size(0))
                fail(std::string(t == &*cos ? "cos" : "sin") + " must be a contiguous CUDA float32 [positions, rot/2] tensor on the cache's device");
        max_pos = as_int(cos->size(0), "the number of positions"), rot = 2 * cos->size(1);
        if (rot == 0 || rot % 8 || rot > c.head_dim) fail("the rotated channels must be a multiple of 8 up to head_dim");
    }
    const uint16_t* qp = nullptr;
    if (!q && q_out) fail("q_out without q");
    if (q) {
        if (!cos) fail("q is only taken to be rotated: cos and sin are missing");
        qp = check_vectors(c, *q, "q", n, -1);
        if (!as_int(q->size(1), "the number of heads")) fail("q has no heads");
        if (q_out) dense_half(*q_out, "q_out", q->sizes(), c.pool.device(), "cache");
    }
    const Place at_(c.pool.get_device(), stream);
    OptTensor out = q_out;
    if (q && !q_out) out = at_.output(q->sizes(), q->device());
    if (n)
        check(p_kv_append(at_.ptr(), c.pool.data_ptr(), c.num_pages, c.page_size, c.kv_heads, c.head_dim, b.table, b.width, b.lens, b.cu, b.batch, n, kp,
                          k.stride(0), k.stride(1), vp, v.stride(0), v.stride(1), qp, q ? q->stride(0) : 0, q ? q->stride(1) : 0, q ? (int)q->size(1) : 0,
                          out ? static_cast<uint16_t*>(out->data_ptr()) : nullptr, cos ? cos->const_data_ptr<float>() : nullptr,
                          sin ? sin->const_data_ptr<float>() : nullptr, (int)max_pos, (int)rot, interleaved),
              "spb_kv_append");
    return out;
}

std::pair<Tensor, Tensor> kv_read(const Cache& c, const Tensor& table, const Tensor& lens, const OptTensor& cu, std::optional<int64_t> n_tokens,
                                  const OptTensor& k_out, const OptTensor& v_out, std::optional<int64_t> stream)
{
    const Batch b = check_batch(c, table, lens, cu);
    if (!n_tokens && !k_out) fail("n_tokens or k_out is needed");
    const int64_t n = n_tokens ? *n_tokens : k_out->dim() ? k_out->size(0) : 0;
    if (n < 0) fail("n_tokens must not be negative");
    check_rows(n, b);
    const int64_t shape[3] = {n, c.kv_heads, c.head_dim};
    if (k_out) dense_half(*k_out, "k_out", shape, c.pool.device(), "cache");
    if (v_out) dense_half(*v_out, "v_out", shape, c.pool.device(), "cache");
    const Place at_(c.pool.get_device(), stream);
    Tensor k = k_out ? *k_out : at_.output(shape, c.pool.device()), v = v_out ? *v_out : at_.output(shape, c.pool.device());
    if (n)
        check(p_kv_read(at_.ptr(), c.pool.data_ptr(), c.num_pages, c.page_size, c.kv_heads, c.head_dim, b.table, b.width, b.lens, b.cu, b.batch, n,
                        static_cast<uint16_t*>(k.data_ptr()), static_cast<uint16_t*>(v.data_ptr())),
              "spb_kv_read");
    return {k, v};
}

size_t kv_attention_workspace(const Cache& c, int64_t q_heads, int64_t batch, int64_t max_q)
{
    check_pool(c);
    for (const auto& [x, name] : {std::pair{q_heads, "q_heads"}, {batch, "batch"}, {max_q, "max_q"}}) as_int(x, name);
    const c10::cuda::CUDAGuard guard(c.pool.device());
    const size_t bytes = p_kv_attention_workspace_bytes(c.head_dim, (int)batch, (int)q_heads, c.kv_heads, (int)max_q);
    if (!bytes) fail("batch must be positive, q_heads a positive multiple of the cache's heads and max_q not negative");
    return bytes;
}

Tensor kv_attention(const Tensor& q, const Cache& c, const Tensor& table, const Tensor& lens, const OptTensor& cu, std::optional<int64_t> max_q,
                    std::optional<double> scale, const OptTensor& out_given, const OptTensor& ws_given, std::optional<int64_t> stream)
{
    const Batch b = check_batch(c, table, lens, cu);
    const uint16_t* qp = check_vectors(c, q, "q", -1, -1);
    const int64_t n = q.size(0);
    const int heads = as_int(q.size(1), "the number of heads");
    if (!heads || heads % c.kv_heads) fail("the heads of q must be a positive multiple of the cache's");
    check_rows(n, b);
    const int64_t bound = max_q ? *max_q : b.cu ? n : n / b.batch;
    if (bound < 0 || bound > n) fail("max_q must be in 0..tokens");
    const int most = as_int(bound, "max_q");
    if (out_given) dense_half(*out_given, "out", q.sizes(), c.pool.device(), "cache");
    const Place at_(c.pool.get_device(), stream);
    Tensor out = out_given ? *out_given : at_.output(q.sizes(), q.device());
    if (!n) return out;
    size_t have;
    const Tensor ws = pick_workspace(ws_given, p_kv_attention_workspace_bytes(c.head_dim, b.batch, heads, c.kv_heads, most), q, "cache", have);
    check(p_kv_attention(at_.ptr(), c.pool.data_ptr(), c.num_pages, c.page_size, c.kv_heads, c.head_dim, b.table, b.width, b.lens, b.cu, b.batch, n, qp,
                         q.stride(0), q.stride(1), heads, most, (float)(scale ? *scale : 1 / std::sqrt((double)c.head_dim)),
                         static_cast<uint16_t*>(out.data_ptr()), ws.data_ptr(), have),
          "spb_kv_attention");
    return out;
}

// -------------------------------------------------------------------------------------------------- 4-bit weights

Tensor linear_int4(const Tensor& data, int64_t rows, int64_t columns, int64_t group, const Tensor& x, const OptTensor& bias, const OptTensor& residual,
                   int64_t activation, const OptTensor& out_given, const OptTensor& ws_given, std::optional<int64_t> stream)
{
    const auto dev = data.device();
    const int M = as_int(rows, "M"), K = as_int(columns, "K");
    const size_t bytes = p_int4_bytes(M, K, as_int(group, "the group"));
    if (!bytes) fail("M and K must be positive multiples of 64 and the group 32, 64 or 128 and divide K");
    if (!data.is_cuda() || data.scalar_type() != at::kByte || !data.is_contiguous() || data.dim() != 1 || (size_t)data.size(0) != bytes)
        fail("W.data must be the contiguous CUDA uint8 tensor that pack_int4 made");
    if (x.device() != dev || x.scalar_type() != at::kHalf || x.dim() != 2 || x.size(1) != K || !x.size(0) || !x.is_contiguous())
        fail("B must be a contiguous CUDA float16 [N,K] tensor on the weight's device");
    const int N = as_int(x.size(0), "N");
    const int64_t shape[2] = {N, M};
    if (activation != 0 && activation != 1) fail("activation must be ACT_NONE or ACT_RELU");
    if (bias && (bias->device() != dev || bias->scalar_type() != at::kHalf || !bias->is_contiguous() || bias->dim() != 1 || bias->size(0) != M))
        fail("bias must be a contiguous CUDA float16 [M] tensor");
    if (residual) dense_half(*residual, "residual", shape, dev, "weight");
    if (out_given) dense_half(*out_given, "out", shape, dev, "weight");
    const Place at_(data.get_device(), stream);
    Tensor out = out_given ? *out_given : at_.output(shape, dev);
    size_t have;
    const Tensor ws = pick_workspace(ws_given, p_int4_workspace_bytes(M, N, K), x, "weight", have);
    auto half = [](const OptTensor& t) { return t ? static_cast<const uint16_t*>(t->const_data_ptr()) : nullptr; };
    check(p_linear_int4(at_.ptr(), data.const_data_ptr(), M, K, (int)group, static_cast<const uint16_t*>(x.const_data_ptr()),
                        static_cast<uint16_t*>(out.data_ptr()), N, half(bias), half(residual), (int)activation, ws.defined() ? ws.data_ptr() : nullptr, have),
          "spb_linear_int4");
    return out;
}

}  // namespace

PYBIND11_MODULE(_torch_ext, m)
{
    m.def("init", &init);
    py::class_<Cache>(m, "Cache").def(py::init([](Tensor pool, int pages, int page_size, int heads, int dim) { return Cache{pool, pages, page_size, heads, dim}; }));
    m.def("kv_append", &kv_append);
    m.def("kv_read", &kv_read);
    m.def("kv_attention", &kv_attention);
    m.def("kv_attention_workspace", &kv_attention_workspace);
    m.def("linear_int4", &linear_int4);
}
