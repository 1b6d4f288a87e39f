// Python calls of the paged-serving operators: argument checks, outputs, scratch and the C-ABI call in one native function
// each. Their kernels take 3 to 12 us for a decoded token, less than checking the same arguments and converting them in
// Python does (15 to 20 us a call); this takes 2 to 3.
//
// Torch tensors in, the C ABI (include/exl3_b200.h) out; nothing here computes. Checks raise TypeError for types and
// ValueError for the rest, as the ctypes binding does.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <map>
#include <tuple>

#include "exl3_b200.h"

namespace {

using at::Tensor;

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)
#define NEED_TYPE(cond, ...) TORCH_CHECK_TYPE(cond, __VA_ARGS__)

const Tensor& tensor(PyObject* o, const char* name)
{
    NEED_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}

long long integer(PyObject* o, const char* name)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, name, " must be an integer");
    }
    return v;
}

double number(PyObject* o, const char* name)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        TORCH_CHECK_TYPE(false, name, " must be a number");
    }
    return v;
}

void raise_status(int status, const char* what)
{
    if (status == EXL3_OK) return;
    const std::string msg = std::string(what) + ": " + exl3_strerror(status) + " (status " + std::to_string(status) + ")";
    if (status == EXL3_E_DTYPE) TORCH_CHECK_TYPE(false, msg);
    TORCH_CHECK(status != EXL3_E_CUDA && status != EXL3_E_DEVICE, msg);
    TORCH_CHECK_VALUE(false, msg);
}

bool capturing() { return at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None; }

// The paged kernels' status word of a device. All of this file's state is touched with the interpreter lock held, and never
// destroyed: the CUDA context may be gone by then.
std::map<int, Tensor>& status_words()
{
    static auto* words = new std::map<int, Tensor>;
    return *words;
}

uint32_t* status_word(const Tensor& like)
{
    auto& words = status_words();
    const auto it = words.find(like.get_device());
    if (it != words.end()) return reinterpret_cast<uint32_t*>(it->second.data_ptr());
    TORCH_CHECK(!capturing(), "call a paged kernel once on this device before capturing it in a graph");
    const c10::InferenceMode plain(false);            // whoever makes the first call
    Tensor word = at::zeros({4}, like.options().dtype(at::kInt));
    at::cuda::getCurrentCUDAStream().synchronize();   // zero before a call on any other stream may set a bit
    words[like.get_device()] = word;
    return reinterpret_cast<uint32_t*>(word.data_ptr());
}

// Scratch of one operator on this device and stream: calls on different streams may overlap, calls on one stream run one
// after another. A captured call gets scratch of its own from the graph's pool, so replays may run beside eager calls.
Tensor workspace(int kind, const Tensor& like, cudaStream_t stream, size_t bytes)
{
    const auto options = like.options().dtype(at::kByte);
    if (capturing()) return at::empty({(int64_t)bytes}, options);
    static auto* spaces = new std::map<std::tuple<int, int, cudaStream_t>, Tensor>;
    Tensor& ws = (*spaces)[{kind, like.get_device(), stream}];
    if (!ws.defined() || (size_t)ws.numel() < bytes) ws = at::empty({(int64_t)bytes}, options);
    return ws;
}

bool half_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }

int dtype_code(at::ScalarType t) { return t == at::kHalf ? EXL3_F16 : t == at::kBFloat16 ? EXL3_BF16 : EXL3_F32; }

// Checked descriptor of a batch: what can be checked without reading device memory.
exl3_paged_desc descriptor(const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& cu, const Tensor& lens, int64_t rows)
{
    NEED_TYPE(half_type(kp.scalar_type()) && vp.scalar_type() == kp.scalar_type(), "k_pages and v_pages must both be fp16 or both bf16");
    NEED_TYPE(table.scalar_type() == at::kInt && cu.scalar_type() == at::kInt && lens.scalar_type() == at::kInt,
              "page_table, cu_rows and lens must be int32");
    NEED(kp.is_cuda(), "EXL3 kernels take CUDA tensors");
    const auto dev = kp.device();
    NEED(vp.device() == dev && table.device() == dev && cu.device() == dev && lens.device() == dev,
         "the pages and the batch's tables must be on one device");
    NEED(kp.dim() == 4 && vp.sizes() == kp.sizes(), "pages must be (num_pages, hkv, page_size, head_dim), K and V alike");
    NEED(table.dim() == 2 && cu.dim() == 1 && lens.dim() == 1, "page_table is 2-d, cu_rows and lens 1-d");
    const int64_t seqs = table.size(0);
    NEED(seqs >= 1 && cu.size(0) == seqs + 1 && lens.size(0) == seqs, "page_table (seqs, cols), cu_rows (seqs + 1) and lens (seqs) must agree");
    NEED(kp.is_contiguous() && vp.is_contiguous(), "pages must be contiguous");
    NEED(table.is_contiguous() && cu.is_contiguous() && lens.is_contiguous(), "page_table, cu_rows and lens must be contiguous");
    constexpr int64_t most = 0x7fffffff;
    NEED(rows <= most && seqs <= most && table.size(1) <= most && kp.size(0) <= most && kp.size(1) <= most && kp.size(2) <= most,
         "sizes must fit 32 bits");
    exl3_paged_desc b{};
    b.k_pages = kp.data_ptr();
    b.v_pages = vp.data_ptr();
    b.page_table = table.data_ptr<int>();
    b.cu_rows = cu.data_ptr<int>();
    b.lens = lens.data_ptr<int>();
    b.seqs = (int32_t)seqs;
    b.rows = (int32_t)rows;
    b.table_cols = (int32_t)table.size(1);
    b.num_pages = (int32_t)kp.size(0);
    b.hkv = (int32_t)kp.size(1);
    b.page_size = (int32_t)kp.size(2);
    b.head_dim = (int32_t)kp.size(3);
    b.dtype = dtype_code(kp.scalar_type());
    return b;
}

// Row stride in elements of a (rows, width) view with contiguous rows.
int64_t row_stride(const Tensor& x, int64_t rows, int64_t width, const char* name)
{
    NEED(x.dim() == 2 && x.size(0) == rows && x.size(1) == width, name, " must be (", rows, ", ", width, ")");
    const int64_t s0 = x.stride(0), s1 = x.stride(1);
    if (s1 == 1 && s0 >= width) return s0;
    NEED(rows <= 1 && (s1 == 1 || width <= 1), name, " needs contiguous, non-overlapping rows");
    return width;
}

const void* norm_weight(PyObject* o, const Tensor& q, int64_t hd)
{
    if (o == Py_None) return nullptr;
    const Tensor& w = tensor(o, "a norm weight");
    NEED_TYPE(w.scalar_type() == q.scalar_type(), "norm weights must have q's dtype");
    NEED(w.numel() == hd && w.is_contiguous() && w.device() == q.device(), "norm weights must be contiguous (head_dim) on the pages' device");
    return w.data_ptr();
}

Tensor output(PyObject* o, at::IntArrayRef sizes, const at::TensorOptions& options, const char* what)
{
    if (o == Py_None) return at::empty(sizes, options);
    const Tensor& t = tensor(o, what);
    NEED(t.sizes() == sizes && t.scalar_type() == options.dtype() && t.is_contiguous() && t.device() == options.device(), what,
         " must be contiguous (rows, hq, head_dim) in the cache's dtype, on its device");
    return t;
}

// paged_qkv_post(q, k, v, q_norm_w, k_norm_w, eps, cos, sin, k_pages, v_pages, page_table, cu_rows, lens, q_out)
PyObject* paged_qkv_post(PyObject*, PyObject* const* arg, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    NEED_TYPE(n == 14, "paged_qkv_post takes 14 arguments");
    const Tensor &q = tensor(arg[0], "q"), &k = tensor(arg[1], "k"), &v = tensor(arg[2], "v"), &cos = tensor(arg[6], "cos"),
                 &sin = tensor(arg[7], "sin"), &kp = tensor(arg[8], "k_pages");
    const double eps = number(arg[5], "eps");
    NEED(q.dim() == 2, "q must be (rows, hq * head_dim)");
    const int64_t rows = q.size(0), width = q.size(1);
    const exl3_paged_desc b = descriptor(kp, tensor(arg[9], "v_pages"), tensor(arg[10], "page_table"), tensor(arg[11], "cu_rows"),
                                         tensor(arg[12], "lens"), rows);
    NEED_TYPE(half_type(q.scalar_type()) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must all be fp16 or all bf16");
    const int64_t hd = b.head_dim, nk = b.hkv * hd;
    NEED(width > 0 && nk > 0 && width % nk == 0, "q's width must be a multiple of hkv * head_dim");
    const int64_t sq = row_stride(q, rows, width, "q"), sk = row_stride(k, rows, nk, "k"), sv = row_stride(v, rows, nk, "v");
    NEED_TYPE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin must be fp32");
    NEED(cos.dim() == 2 && sin.sizes() == cos.sizes() && cos.is_contiguous() && sin.is_contiguous(),
         "cos and sin must be contiguous (positions, rotated / 2)");
    const auto dev = kp.device();
    NEED(q.device() == dev && k.device() == dev && v.device() == dev && cos.device() == dev && sin.device() == dev,
         "all tensors must be on one device");
    const void *wq = norm_weight(arg[3], q, hd), *wk = norm_weight(arg[4], q, hd);
    const int64_t hq = width / hd;
    NEED(hq <= 0x7fffffff && cos.size(0) <= 0x7fffffff && cos.size(1) <= 0x7fffffff, "sizes must fit 32 bits");
    const c10::cuda::CUDAGuard guard(dev);
    Tensor out = output(arg[13], {rows, hq, hd}, kp.options(), "q_out");
    raise_status(exl3_paged_qkv_post(&b, q.data_ptr(), k.data_ptr(), v.data_ptr(), sq, sk, sv, dtype_code(q.scalar_type()), (int)hq, wq, wk,
                                     (float)eps, cos.data_ptr<float>(), sin.data_ptr<float>(), (int)cos.size(0), (int)cos.size(1),
                                     out.data_ptr(), status_word(kp), at::cuda::getCurrentCUDAStream().stream()),
                 "exl3_paged_qkv_post");
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// paged_attn(q, k_pages, v_pages, page_table, cu_rows, lens, scale, out, max_rows)
PyObject* paged_attn(PyObject*, PyObject* const* arg, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    NEED_TYPE(n == 9, "paged_attn takes 9 arguments");
    Tensor q = tensor(arg[0], "q");
    const Tensor& kp = tensor(arg[1], "k_pages");
    NEED(q.dim() == 3, "q must be (rows, hq, head_dim)");
    const int64_t rows = q.size(0), hq = q.size(1), hd = q.size(2);
    const exl3_paged_desc b = descriptor(kp, tensor(arg[2], "v_pages"), tensor(arg[3], "page_table"), tensor(arg[4], "cu_rows"),
                                         tensor(arg[5], "lens"), rows);
    NEED_TYPE(q.scalar_type() == kp.scalar_type(), "q must have the cache's dtype");
    NEED(hd == b.head_dim && q.device() == kp.device(), "q must be (rows, hq, head_dim) on the pages' device");
    NEED(hq >= 1 && b.hkv > 0 && hq % b.hkv == 0 && hq / b.hkv <= 128, "hq must be a multiple of hkv, at most 128 heads per kv head");
    const double scale = arg[6] == Py_None ? 1.0 / std::sqrt((double)hd) : number(arg[6], "scale");
    NEED(scale > 0 && std::isfinite(scale), "scale must be positive");
    const long long max_rows = integer(arg[8], "max_rows");
    NEED(max_rows >= 0 && max_rows <= 0x7fffffff, "max_rows must be zero or more");
    const c10::cuda::CUDAGuard guard(kp.device());
    if (q.stride(2) != 1 || q.stride(1) != hd || q.stride(0) % 8 || q.stride(0) < hq * hd || reinterpret_cast<uintptr_t>(q.data_ptr()) % 16)
        q = q.clone(at::MemoryFormat::Contiguous);
    Tensor out = output(arg[7], {rows, hq, hd}, kp.options(), "out");
    if (rows > 0) {
        static auto* sizes = new std::map<std::pair<int, int64_t>, size_t>;      // by device and head size alone
        size_t& need = (*sizes)[{kp.get_device(), hd}];
        if (!need) raise_status(exl3_paged_attn_workspace(&b, (int)hq, &need), "exl3_paged_attn_workspace");
        const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
        Tensor ws = workspace(0, kp, stream, need);
        raise_status(exl3_paged_attn(&b, q.data_ptr(), q.stride(0), (int)hq, (float)scale, (int)max_rows, out.data_ptr(), ws.data_ptr(),
                                     need, status_word(kp), stream),
                     "exl3_paged_attn");
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

// verify_drafts(target_logits, draft_tokens, cu_rows, u, noise, max_drafts, draft_logits, temperature) -> (tokens, count, accept_prob)
PyObject* verify_drafts(PyObject*, PyObject* const* arg, Py_ssize_t n_arg)
{
    HANDLE_TH_ERRORS
    NEED_TYPE(n_arg == 8, "verify_drafts takes 8 arguments");
    const Tensor &target = tensor(arg[0], "target_logits"), &drafted = tensor(arg[1], "draft_tokens"), &cu = tensor(arg[2], "cu_rows"),
                 &u = tensor(arg[3], "u"), &noise = tensor(arg[4], "noise");
    const auto type = target.scalar_type();
    NEED_TYPE(half_type(type) || type == at::kFloat, "unsupported dtype of target_logits");
    NEED(target.is_cuda(), "EXL3 kernels take CUDA tensors");
    const long long max_drafts = integer(arg[5], "max_drafts");
    NEED(target.dim() == 2 && cu.dim() == 1 && cu.size(0) >= 2, "need target_logits (rows, n) and cu_rows (seqs + 1)");
    const int64_t rows = target.size(0), n = target.size(1), seqs = cu.size(0) - 1, drafts = rows - seqs;
    NEED(n >= 1 && drafts >= 0 && max_drafts >= 0, "each sequence needs at least one target row");
    NEED(rows <= 0x7fffffff && n <= 0x7fffffff && max_drafts < 0x7fffffff, "sizes must fit 32 bits");
    NEED_TYPE(cu.scalar_type() == at::kInt && drafted.scalar_type() == at::kLong, "cu_rows must be int32 and draft_tokens int64");
    NEED_TYPE(u.scalar_type() == at::kFloat && noise.scalar_type() == at::kFloat, "u, noise and temperature must be fp32");
    NEED(drafted.dim() == 1 && drafted.size(0) == drafts && u.dim() == 1 && u.size(0) == drafts, "draft_tokens and u must be (rows - seqs)");
    NEED(cu.is_contiguous() && drafted.is_contiguous() && u.is_contiguous(), "cu_rows, draft_tokens and u must be contiguous");
    const auto dev = target.device();
    NEED(drafted.device() == dev && cu.device() == dev && u.device() == dev && noise.device() == dev, "all tensors must be on one device");
    const int64_t ld = row_stride(target, rows, n, "target_logits"), noise_ld = row_stride(noise, seqs, n, "noise");
    const void* draft = nullptr;
    int64_t draft_ld = n;
    if (arg[6] != Py_None) {
        const Tensor& d = tensor(arg[6], "draft_logits");
        NEED_TYPE(d.scalar_type() == type, "draft_logits must have target_logits' dtype");
        NEED(d.device() == dev, "all tensors must be on one device");
        draft_ld = row_stride(d, drafts, n, "draft_logits");
        if (drafts) draft = d.data_ptr();
    }
    const float* temperature = nullptr;
    if (arg[7] != Py_None) {
        const Tensor& t = tensor(arg[7], "temperature");
        NEED_TYPE(t.scalar_type() == at::kFloat, "u, noise and temperature must be fp32");
        NEED(t.dim() == 1 && t.size(0) == seqs && t.is_contiguous() && t.device() == dev, "temperature must be contiguous (seqs)");
        temperature = t.data_ptr<float>();
    }
    const c10::cuda::CUDAGuard guard(dev);
    Tensor tokens = at::empty({seqs, max_drafts + 1}, drafted.options()), count = at::empty({seqs}, cu.options()),
           prob = at::empty({drafts}, u.options());
    size_t need = 0;
    raise_status(exl3_verify_workspace((int)rows, (int)seqs, (int)n, &need), "exl3_verify_workspace");
    const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
    Tensor ws = workspace(1, target, stream, need);
    raise_status(exl3_verify_drafts(target.data_ptr(), ld, draft, draft_ld, dtype_code(type), (int)rows, (int)seqs, (int)n,
                                    drafts ? reinterpret_cast<const long long*>(drafted.data_ptr<int64_t>()) : nullptr, cu.data_ptr<int>(),
                                    temperature, drafts ? u.data_ptr<float>() : nullptr, noise.data_ptr<float>(), noise_ld, (int)max_drafts,
                                    reinterpret_cast<long long*>(tokens.data_ptr<int64_t>()), count.data_ptr<int>(),
                                    drafts ? prob.data_ptr<float>() : nullptr, ws.data_ptr(), need, stream),
                 "exl3_verify_drafts");
    PyObject* out = PyTuple_New(3);
    if (!out) throw python_error();
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(tokens));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(count));
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(prob));
    return out;
    END_HANDLE_TH_ERRORS
}

// take_status(device index) -> the device's status word as a tensor of its own, the word cleared; None where no paged kernel has run
PyObject* take_status(PyObject*, PyObject* const* arg, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    NEED_TYPE(n == 1, "take_status takes one argument");
    auto& words = status_words();
    const auto it = words.find((int)integer(arg[0], "device"));
    if (it == words.end()) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard guard(it->second.device());
    Tensor taken = at::empty({1}, it->second.options());
    raise_status(exl3_paged_status_take(reinterpret_cast<uint32_t*>(it->second.data_ptr()), reinterpret_cast<uint32_t*>(taken.data_ptr()),
                                        at::cuda::getCurrentCUDAStream().stream()),
                 "exl3_paged_status_take");
    return THPVariable_Wrap(taken);
    END_HANDLE_TH_ERRORS
}

// status(device index) -> the device's status word as a tensor, or None where no paged kernel has run
PyObject* status(PyObject*, PyObject* const* arg, Py_ssize_t n)
{
    HANDLE_TH_ERRORS
    NEED_TYPE(n == 1, "status takes one argument");
    auto& words = status_words();
    const auto it = words.find((int)integer(arg[0], "device"));
    if (it == words.end()) Py_RETURN_NONE;
    return THPVariable_Wrap(it->second);
    END_HANDLE_TH_ERRORS
}

#define CALL(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {CALL(paged_qkv_post), CALL(paged_attn), CALL(verify_drafts), CALL(status), CALL(take_status),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_exl3_torch", EXL3_BUILT_FOR, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__exl3_torch() { return PyModule_Create(&module); }
