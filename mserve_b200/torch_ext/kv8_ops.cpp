// kv8_ops: the torch binding of the 8-bit paged cache's entry points (mskv_kv8_*, include/mserve_kv.h).
//
// A thin binding: argument checks on ATen tensors, allocation of outputs and workspaces through torch's
// caching allocator, and one call into the C ABI on the current CUDA stream of the tensors' device, with
// that device current.  mserve_b200.ops wraps these functions (its decode-step calls take a few
// microseconds of host time here, against 15 to 20 when a ctypes description is filled in Python).  Checks
// raise ValueError or TypeError; a C ABI error code is returned for the caller to raise.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "mserve_kv.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }

std::string shape_text(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MSKV_DT_F32;
    case at::kHalf: return MSKV_DT_F16;
    case at::kBFloat16: return MSKV_DT_BF16;
    case at::kFloat8_e4m3fn: return MSKV_DT_FP8_E4M3;
    case at::kFloat8_e5m2: return MSKV_DT_FP8_E5M2;
    default: return -1;
  }
}

bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// Shapes, types and layouts of the cache's tensors; fills their addressing.
void fill_pages(mskv_kv8_pages& p, const at::Tensor& k, const at::Tensor& v, const at::Tensor& exps, const OptTensor& bounds,
                const at::Tensor& table, int64_t batch) {
  if (k.dim() != 4 || v.dim() != 4 || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type() ||
      (k.scalar_type() != at::kFloat8_e4m3fn && k.scalar_type() != at::kFloat8_e5m2))
    bad_value("k and v must be fp8 [P, Hkv, page, D] of one shape and type");
  const int64_t P = k.size(0), H = k.size(1), page = k.size(2), D = k.size(3);
  if (k.stride(3) != 1 || k.stride(2) != D || v.strides() != k.strides())
    bad_value("k and v must have contiguous [page, D] pages and the same strides");
  if (exps.scalar_type() != at::kChar || exps.dim() != 3 || exps.size(0) != P || exps.size(1) != H || exps.size(2) != 2 ||
      !exps.is_contiguous())
    bad_value("exps must be a contiguous int8 [P, Hkv, 2] tensor");
  if (bounds && (bounds->scalar_type() != k.scalar_type() || bounds->dim() != 4 || bounds->size(0) != P || bounds->size(1) != H ||
                 bounds->size(2) != 2 || bounds->size(3) != D || !bounds->is_contiguous()))
    bad_value("bounds must be a contiguous [P, Hkv, 2, D] tensor of the cache's type");
  if (table.dim() != 2 || table.scalar_type() != at::kInt || table.size(0) != batch || (table.size(1) > 1 && table.stride(1) != 1))
    bad_value("page_table must be int32 [B=" + std::to_string(batch) + ", max_pages] with unit inner stride");
  if (table.size(1) > INT32_MAX || page > INT32_MAX || H > INT32_MAX || D > INT32_MAX || batch > INT32_MAX)
    bad_value("a size of the cache exceeds 32 bits");
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.exps = exps.data_ptr();
  p.bounds = bounds ? bounds->data_ptr() : nullptr;
  p.page_table = table.data_ptr<int32_t>();
  p.stride_page = k.stride(0);
  p.stride_h = k.stride(1);
  p.pt_stride_b = table.stride(0);
  p.num_pages = P;
  p.max_pages = (int32_t)table.size(1);
  p.page_size = (int32_t)page;
  p.kv_heads = (int32_t)H;
  p.head_dim = (int32_t)D;
  p.dtype = dtype_code(k.scalar_type());
  p.batch = (int32_t)batch;
}

const int32_t* int32_list(const at::Tensor& t, int64_t numel, const char* name) {
  if (t.scalar_type() != at::kInt || t.numel() != numel || !t.is_contiguous())
    bad_value(std::string(name) + " must be a contiguous int32 tensor of " + std::to_string(numel) + " entries");
  return t.data_ptr<int32_t>();
}

// All tensors of a call live on the device of the first.
template <typename... T>
c10::Device one_device(const char* name, const at::Tensor& first, const T&... others) {
  if (!first.is_cuda()) bad_value(std::string(name) + " must be a CUDA tensor");
  const c10::Device d = first.device();
  const auto check = [&](const at::Tensor& t) {
    if (t.device() != d) bad_value("all tensors of the call must live on " + d.str());
  };
  (check(others), ...);
  return d;
}
void same_device(const c10::Device& d, const OptTensor& t) {
  if (t && t->device() != d) bad_value("all tensors of the call must live on " + d.str());
}

// Outputs whose rows lie on each other (expanded ones) would be written by several blocks at once.
void no_overlap(const at::Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) bad_value(std::string(name) + " must not be expanded: its elements share memory");
}

uint32_t* status_ptr(const OptTensor& t) { return t ? reinterpret_cast<uint32_t*>(t->data_ptr()) : nullptr; }

int append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& exps, const OptTensor& bounds, const at::Tensor& table,
           const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& tok0, const OptTensor& counts,
           const OptTensor& status) {
  if (k_new.dim() != 4 || v_new.sizes() != k_new.sizes() || v_new.scalar_type() != k_new.scalar_type())
    bad_value("k_new and v_new must be [B, Hkv, n, D] of one shape and type");
  const int code = dtype_code(k_new.scalar_type());
  if (code != MSKV_DT_F32 && code != MSKV_DT_F16 && code != MSKV_DT_BF16)
    throw py::type_error(std::string("new rows must be float32/float16/bfloat16, got ") + c10::toString(k_new.scalar_type()));
  const int64_t B = k_new.size(0), H = k_new.size(1), n = k_new.size(2), D = k_new.size(3);
  mskv_kv8_append_desc d{};
  fill_pages(d.pages, k, v, exps, bounds, table, B);
  if (H != k.size(1) || D != k.size(3)) bad_value("rows " + shape_text(k_new) + " do not match a cache of " + shape_text(k));
  if (n && (k_new.stride(3) != 1 || v_new.stride(3) != 1)) bad_value("the head_dim axis of the rows must be contiguous");
  if (n > INT32_MAX) bad_value("too many rows for one call");
  for (const at::Tensor* pool : {&k, &v}) no_overlap(*pool, "a cache that is appended to");
  d.tok0 = int32_list(tok0, B, "tok0");
  if (counts) d.counts = int32_list(*counts, B, "counts");
  const c10::Device dev = one_device("k_new", k_new, v_new, k, v, exps, table, tok0);
  same_device(dev, bounds);
  same_device(dev, counts);
  if (B == 0 || n == 0) return MSKV_OK;
  const int64_t es = (int64_t)k_new.element_size();
  d.k_new = k_new.data_ptr();
  d.v_new = v_new.data_ptr();
  d.k_stride_b = k_new.stride(0) * es;
  d.k_stride_h = k_new.stride(1) * es;
  d.k_stride_t = k_new.stride(2) * es;
  d.v_stride_b = v_new.stride(0) * es;
  d.v_stride_h = v_new.stride(1) * es;
  d.v_stride_t = v_new.stride(2) * es;
  d.status = status_ptr(status);
  d.dtype = code;
  d.num_tokens = (int32_t)n;
  const c10::cuda::CUDAGuard guard(dev);
  return mskv_kv8_append(&d, at::cuda::getCurrentCUDAStream(dev.index()).stream());
}

int block_score(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& exps, const OptTensor& bounds,
                const at::Tensor& table, const at::Tensor& lens, int64_t max_blocks, const at::Tensor& out, const OptTensor& status) {
  if (q_in.dim() != 3 && !(q_in.dim() == 4 && q_in.size(2) > 0)) bad_value("q must be [B, Hq, D] or [B, Hq, Q, D]");
  const int last = (int)q_in.dim() - 1;
  if (q_in.stride(last) != 1) bad_value("q must have a contiguous head_dim");
  if (!half_type(q_in)) throw py::type_error(std::string("q must be float16 or bfloat16, got ") + c10::toString(q_in.scalar_type()));
  const int64_t B = q_in.size(0), Hq = q_in.size(1), D = q_in.size(last);
  mskv_kv8_score_desc d{};
  fill_pages(d.pages, k, v, exps, bounds, table, B);
  const int64_t H = k.size(1);
  if (!bounds) bad_value("block scores need pages with bounds");
  if (D != k.size(3) || Hq == 0 || H == 0 || Hq % H) bad_value("q " + shape_text(q_in) + " does not match a cache of " + shape_text(k));
  if (out.scalar_type() != at::kFloat || out.dim() != 3 || out.size(0) != B || out.size(1) != H || out.size(2) < max_blocks ||
      (out.size(2) > 1 && out.stride(2) != 1) || (B > 1 && H > 1 && out.stride(0) != H * out.stride(1)))
    bad_value("out must be fp32 [B, Hkv, >= max_blocks] with rows at a common stride");
  no_overlap(out, "out");
  if (max_blocks < 0 || max_blocks > table.size(1)) bad_value("max_blocks must lie in [0, " + std::to_string(table.size(1)) + "]");
  d.lens = int32_list(lens, B, "lens");
  const c10::Device dev = one_device("q", q_in, k, v, exps, *bounds, table, lens, out);
  if (B == 0 || max_blocks == 0) return MSKV_OK;
  const int64_t es = (int64_t)q_in.element_size();
  d.q = static_cast<const char*>(q_in.data_ptr()) + (last == 3 ? (q_in.size(2) - 1) * q_in.stride(2) * es : 0);
  d.q_stride_b = q_in.stride(0) * es;
  d.q_stride_h = q_in.stride(1) * es;
  d.scores = out.data_ptr<float>();
  // the common stride of the rows (b, h); of a single row, its length
  d.scores_stride = H > 1 ? out.stride(1) : B > 1 ? out.stride(0) : out.size(2);
  d.status = status_ptr(status);
  d.dtype = dtype_code(q_in.scalar_type());
  d.q_heads = (int32_t)Hq;
  d.max_blocks = (int32_t)max_blocks;
  const c10::cuda::CUDAGuard guard(dev);
  return mskv_kv8_block_score(&d, at::cuda::getCurrentCUDAStream(dev.index()).stream());
}

std::tuple<int, at::Tensor> attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& exps,
                                      const OptTensor& bounds, const at::Tensor& table, const at::Tensor& lens,
                                      std::optional<int64_t> max_tokens, const OptTensor& blocks, const OptTensor& counts,
                                      std::optional<double> scale, const OptTensor& out_in, const OptTensor& status) {
  if (q.dim() != 4) bad_value("q must be [B, Hq, Q, D]");
  if (!half_type(q)) throw py::type_error(std::string("q must be float16 or bfloat16, got ") + c10::toString(q.scalar_type()));
  const int64_t B = q.size(0), Hq = q.size(1), Q = q.size(2), D = q.size(3);
  if (q.stride(3) != 1) bad_value("q must have a contiguous head_dim");
  mskv_kv8_attn_desc d{};
  fill_pages(d.pages, k, v, exps, bounds, table, B);
  const int64_t H = k.size(1), most = table.size(1) * k.size(2);
  if (D != k.size(3) || Hq == 0 || H == 0 || Hq % H) bad_value("q " + shape_text(q) + " does not match a cache of " + shape_text(k));
  if (Q < 1 || Q > MSKV_KV8_MAX_QLEN)
    bad_value("q must hold 1 to " + std::to_string(MSKV_KV8_MAX_QLEN) + " positions, got " + std::to_string(Q));
  if (max_tokens && (*max_tokens < 0 || *max_tokens > most)) bad_value("max_tokens must lie in [0, " + std::to_string(most) + "]");
  if (most > INT32_MAX) bad_value("a page table of 2^31 tokens or more");
  if (scale && !std::isfinite(*scale)) bad_value("scale must be finite");
  d.lens = int32_list(lens, B, "lens");
  if (blocks) {
    if (blocks->scalar_type() != at::kInt || blocks->dim() != 3 || blocks->size(0) != B || blocks->size(1) != H ||
        (blocks->size(2) > 1 && blocks->stride(2) != 1) || blocks->size(2) > INT32_MAX)
      bad_value("blocks must be int32 [B=" + std::to_string(B) + ", Hkv=" + std::to_string(H) + ", S] with unit inner stride");
    if (counts) d.counts = int32_list(*counts, B * H, "counts");
    // an empty list has no address, and NULL means the whole cache; nothing of it is read
    d.blocks = blocks->numel() ? blocks->data_ptr<int32_t>() : d.lens;
    d.blk_stride_b = blocks->stride(0);
    d.blk_stride_h = blocks->stride(1);
    d.num_blocks = (int32_t)blocks->size(2);
  } else if (counts) {
    bad_value("counts go with blocks");
  }
  if (out_in && (out_in->sizes() != q.sizes() || out_in->scalar_type() != q.scalar_type() || out_in->stride(3) != 1))
    bad_value("out must have q's shape and dtype and a contiguous head_dim");
  if (out_in) no_overlap(*out_in, "out");
  const c10::Device dev = one_device("q", q, k, v, exps, table, lens);
  same_device(dev, bounds);
  same_device(dev, blocks);
  same_device(dev, counts);
  same_device(dev, out_in);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor out = out_in ? *out_in : at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (B == 0) return {MSKV_OK, out};
  const int64_t es = (int64_t)q.element_size();
  d.q = q.data_ptr();
  d.q_stride_b = q.stride(0) * es;
  d.q_stride_h = q.stride(1) * es;
  d.q_stride_q = q.stride(2) * es;
  d.out = out.data_ptr();
  d.out_stride_b = out.stride(0) * es;
  d.out_stride_h = out.stride(1) * es;
  d.out_stride_q = out.stride(2) * es;
  d.status = status_ptr(status);
  d.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)D));
  d.dtype = dtype_code(q.scalar_type());
  d.q_heads = (int32_t)Hq;
  d.q_len = (int32_t)Q;
  d.max_tokens = (int32_t)(max_tokens ? *max_tokens : most);
  // The workspace is a tensor of the call: the allocator keeps its memory from calls on other streams and
  // from other graphs for as long as this launch can use it.
  at::Tensor ws;
  if (const uint64_t need = mskv_kv8_attention_workspace_bytes(&d)) {
    ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous));
    d.workspace = ws.data_ptr();
    d.workspace_bytes = need;
  }
  return {mskv_kv8_attention(&d, at::cuda::getCurrentCUDAStream(dev.index()).stream()), out};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("append", &append);
  m.def("block_score", &block_score);
  m.def("attention", &attention);
}
