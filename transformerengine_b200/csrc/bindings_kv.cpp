// Bindings of the 8-bit key/value cache (csrc/attn/kv_cache.cu, fp8_attend.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <teb200/api.h>
#include <teb200/kv_cache.h>
#include <teb200/nvtx.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <string>
#include <vector>

namespace py = pybind11;

int* device_status(int device);   // bindings.cpp

namespace {

// numbers go into messages as strings (formatting one through a stream inside a check is not safe with every C++ runtime)
std::string str(int64_t n) { return std::to_string(n); }

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int value_type(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return teb200::kFloat32;
    case at::kHalf: return teb200::kFloat16;
    case at::kBFloat16: return teb200::kBFloat16;
    default: TORCH_CHECK(false, what, " must be fp32, fp16 or bf16");
  }
}

const int* int_vec(const at::Tensor& t, int64_t n, const at::Device& dev, const char* what) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 && t.numel() == n, what,
              " must be a contiguous int32 tensor of ", str(n), " entries on the cache's device");
  return t.data_ptr<int>();
}

teb200::Fp8CacheView cache_view(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                                const at::Tensor& table, const at::Tensor& kv_lens) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() &&
                  v.device() == k.device(),
              "the cache must be contiguous [pages, heads, page_size, d] codes, k and v alike");
  TORCH_CHECK(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn,
              "the cache's codes must be float8_e4m3fn");
  // (a contiguous view into a pool may start anywhere; the kernels copy 16 bytes at a time)
  TORCH_CHECK((reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) % 16 == 0,
              "the cache's codes must start on a multiple of 16 bytes");
  const int64_t page = k.size(2), d = k.size(3);
  TORCH_CHECK(d == 64 || d == 128 || d == 256, "the 8-bit cache kernels take head dims 64, 128 and 256, got ", str(d));
  TORCH_CHECK(page >= teb200::kKvBlock && page % teb200::kKvBlock == 0, "the page size must be a multiple of ",
              str(teb200::kKvBlock), ", got ", str(page));
  for (const at::Tensor* s : {&ks, &vs})
    TORCH_CHECK(s->device() == k.device() && s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 3 &&
                    s->size(0) == k.size(0) && s->size(1) == k.size(1) && s->size(2) == page / teb200::kKvBlock,
                "scales must be contiguous fp32 [pages, heads, page_size / 16]");
  TORCH_CHECK(k.size(0) > 0 && k.size(1) > 0, "the cache is empty");
  TORCH_CHECK(k.size(0) * k.size(1) * (page / teb200::kKvBlock) <= INT_MAX, "the cache has too many 16-token blocks");
  TORCH_CHECK(table.device() == k.device() && table.scalar_type() == at::kInt && table.dim() == 2 && table.is_contiguous() &&
                  table.size(1) > 0,
              "page_table must be contiguous int32 [sequences, width] on the cache's device");
  TORCH_CHECK(table.size(0) < 65535, "at most 65534 sequences at once");
  teb200::Fp8CacheView c;
  c.k = static_cast<uint8_t*>(k.data_ptr());
  c.v = static_cast<uint8_t*>(v.data_ptr());
  c.k_scale = ks.data_ptr<float>();
  c.v_scale = vs.data_ptr<float>();
  c.pages = static_cast<int>(k.size(0));
  c.heads = static_cast<int>(k.size(1));
  c.page_size = static_cast<int>(page);
  c.d = static_cast<int>(d);
  c.table = table.data_ptr<int>();
  c.width = static_cast<int>(table.size(1));
  c.n = static_cast<int>(table.size(0));
  c.kv_lens = int_vec(kv_lens, table.size(0), k.device(), "kv_lens");
  c.status = device_status(k.get_device());
  return c;
}

// [t, h, d] with d contiguous and 16-byte rows, else a contiguous copy
at::Tensor rows16(const at::Tensor& t) {
  const int64_t e = 16 / t.element_size();
  const bool ok = t.stride(2) == 1 && t.stride(0) % e == 0 && t.stride(1) % e == 0 && t.stride(0) >= 0 && t.stride(1) >= 0 &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (ok) return t;
  at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();   // a contiguous view at an odd offset
}

void fp8_cache_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                      const at::Tensor& new_k, const at::Tensor& new_v, const at::Tensor& table, const at::Tensor& cu_new,
                      const at::Tensor& kv_lens, int64_t max_new) {
  c10::cuda::CUDAGuard guard(k.device());
  teb200::Fp8AppendArgs a;
  a.c = cache_view(k, v, ks, vs, table, kv_lens);
  TORCH_CHECK(new_k.dim() == 3 && new_v.sizes() == new_k.sizes() && new_k.size(1) == a.c.heads && new_k.size(2) == a.c.d,
              "new keys and values must be [tokens, ", str(a.c.heads), ", ", str(a.c.d), "]");
  TORCH_CHECK(new_k.device() == k.device() && new_v.device() == k.device() && new_v.scalar_type() == new_k.scalar_type(),
              "new keys and values must have one type and sit on the cache's device");
  a.dtype = value_type(new_k, "new keys and values");
  TORCH_CHECK(new_k.size(0) <= INT_MAX, "too many new tokens");
  const at::Tensor nk = rows16(new_k), nv = rows16(new_v);
  a.new_k = nk.data_ptr();
  a.new_v = nv.data_ptr();
  a.k_st = nk.stride(0); a.k_sh = nk.stride(1);
  a.v_st = nv.stride(0); a.v_sh = nv.stride(1);
  a.cu_new = int_vec(cu_new, a.c.n + 1, k.device(), "cu_new");
  a.t = static_cast<int>(nk.size(0));
  a.max_new = static_cast<int>(max_new < 0 ? 0 : (max_new > a.t ? a.t : max_new));
  const cudaError_t e = teb200::fp8_cache_append(a, cur_stream());
  TORCH_CHECK(e == cudaSuccess, "fp8_cache_append failed: ", cudaGetErrorString(e));
}

void fp8_cache_gather(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                      const at::Tensor& table, const at::Tensor& kv_lens, const at::Tensor& off, const at::Tensor& out_k,
                      const at::Tensor& out_v, int64_t max_kv) {
  c10::cuda::CUDAGuard guard(k.device());
  teb200::Fp8GatherArgs a;
  a.c = cache_view(k, v, ks, vs, table, kv_lens);
  TORCH_CHECK(out_k.dim() == 3 && out_k.sizes() == out_v.sizes() && out_k.is_contiguous() && out_v.is_contiguous() &&
                  out_k.size(1) == a.c.heads && out_k.size(2) == a.c.d && out_k.scalar_type() == out_v.scalar_type() &&
                  out_k.device() == k.device() && out_v.device() == k.device() && out_k.size(0) <= INT_MAX,
              "gathered keys and values must be contiguous [rows, heads, d]");
  a.dtype = value_type(out_k, "gathered keys and values");
  a.out_k = out_k.data_ptr();
  a.out_v = out_v.data_ptr();
  TORCH_CHECK(off.numel() >= a.c.n, "offsets: one per sequence");
  a.off = int_vec(off, off.numel(), k.device(), "offsets");
  a.rows = static_cast<int>(out_k.size(0));
  a.max_kv = static_cast<int>(std::max<int64_t>(std::min<int64_t>(max_kv, a.rows), 0));   // no sequence has more rows
  const cudaError_t e = teb200::fp8_cache_gather(a, cur_stream());
  TORCH_CHECK(e == cudaSuccess, "fp8_cache_gather failed: ", cudaGetErrorString(e));
}

// Keys and values expanded for the packed attention kernel, pitch rows apart: {k, v, cumulative lengths and first rows of the
// keys, those of the queries}; rows of out that no query claims are zeroed (those behind the last query if `last`).
std::vector<at::Tensor> fp8_cache_expand(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks,
                                         const at::Tensor& vs, const at::Tensor& table, const at::Tensor& cu_q,
                                         const at::Tensor& kv_lens, const at::Tensor& out, int64_t max_q, int64_t max_kv,
                                         int64_t window_left, int64_t sinks, bool last) {
  c10::cuda::CUDAGuard guard(k.device());
  teb200::Fp8GatherArgs a;
  a.c = cache_view(k, v, ks, vs, table, kv_lens);
  TORCH_CHECK(q.device() == k.device() && q.dim() == 3 && q.size(0) <= INT_MAX && sinks >= 0 && max_kv > 0 && max_kv <= INT_MAX - 128 && max_q >= 0,
              "attend: a size is out of range, or the queries are on another device than the cache");
  TORCH_CHECK(q.size(2) == a.c.d && q.size(1) % a.c.heads == 0 && q.size(1) > 0, "queries must be [tokens, heads, ", str(a.c.d),
              "] with a multiple of the cache's ", str(a.c.heads), " heads");
  const int64_t pitch = (max_kv + 127) / 128 * 128;
  TORCH_CHECK(pitch * a.c.n <= INT_MAX, "attend: sequences times max_kv is out of range");
  const at::Tensor ek = at::empty({pitch * a.c.n, a.c.heads, a.c.d}, q.options());
  const at::Tensor ev = at::empty_like(ek);
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous() && out.scalar_type() == q.scalar_type() && out.device() == q.device(),
              "the output must be contiguous and like the queries");
  const at::Tensor meta = at::empty({4, a.c.n + 1}, cu_q.options());
  a.dtype = value_type(q, "queries");
  a.out_k = ek.data_ptr();
  a.out_v = ev.data_ptr();
  a.rows = static_cast<int>(pitch * a.c.n);
  a.pitch = static_cast<int>(pitch);
  a.max_kv = static_cast<int>(max_kv);
  a.cu_q = int_vec(cu_q, a.c.n + 1, k.device(), "cu_q");
  a.window_left = static_cast<int>(window_left < 0 ? -1 : std::min(window_left, max_kv));   // no key lies further back
  a.sinks = static_cast<int>(std::min(sinks, max_kv));
  a.cu_k = meta.data_ptr<int>();
  a.first_row = a.cu_k + a.c.n + 1;
  a.cut_q = a.first_row + a.c.n + 1;
  a.first_q = a.cut_q + a.c.n + 1;
  a.max_q = static_cast<int>(std::min(max_q, q.size(0)));
  a.out = out.data_ptr();
  a.tq = static_cast<int>(q.size(0));
  a.last = last;
  a.row_bytes = q.size(1) * q.size(2) * q.element_size();
  const cudaError_t e = teb200::fp8_cache_gather(a, cur_stream());
  TORCH_CHECK(e == cudaSuccess, "fp8_cache_expand failed: ", cudaGetErrorString(e));
  return {ek, ev, meta.select(0, 0), meta.select(0, 1), meta.select(0, 2), meta.select(0, 3)};
}

at::Tensor fp8_cache_attend(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks,
                            const at::Tensor& vs, const at::Tensor& table, const at::Tensor& cu_q, const at::Tensor& kv_lens,
                            int64_t max_q, int64_t max_kv, double scale, bool causal, int64_t window_left, int64_t sinks) {
  c10::cuda::CUDAGuard guard(k.device());
  teb200::Fp8AttendArgs a;
  a.c = cache_view(k, v, ks, vs, table, kv_lens);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == a.c.d && q.size(1) % a.c.heads == 0 && q.size(1) > 0,
              "queries must be [tokens, heads, ", str(a.c.d), "] with a multiple of the cache's ", str(a.c.heads), " heads");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "queries must be fp16 or bf16");
  TORCH_CHECK(q.device() == k.device() && q.size(0) <= INT_MAX && max_kv <= INT_MAX && max_q >= 0 && max_kv >= 0 && sinks >= 0,
              "attend: a size is out of range, or the queries are on another device than the cache");
  const at::Tensor qr = rows16(q);
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  a.q = qr.data_ptr();
  a.q_st = qr.stride(0); a.q_sh = qr.stride(1);
  a.out = out.data_ptr();
  a.cu_q = int_vec(cu_q, a.c.n + 1, k.device(), "cu_q");
  a.tq = static_cast<int>(q.size(0));
  a.hq = static_cast<int>(q.size(1));
  a.is_bf16 = q.scalar_type() == at::kBFloat16;
  a.max_q = static_cast<int>(std::min(max_q, q.size(0)));   // it sizes the launch: no sequence has more
  a.max_kv = static_cast<int>(max_kv);
  a.causal = causal;
  a.window_left = static_cast<int>(window_left < 0 ? -1 : std::min(window_left, max_kv));   // no key lies further back
  a.sinks = static_cast<int>(std::min(sinks, max_kv));
  a.scale = static_cast<float>(scale);
  const long long need = teb200::fp8_attend_workspace(a);
  at::Tensor part;
  if (need > 0) {
    part = at::empty({need}, q.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  const cudaError_t e = teb200::fp8_attend(a, cur_stream());
  TORCH_CHECK(e == cudaSuccess, "fp8_cache_attend failed: ", cudaGetErrorString(e));
  return out;
}

// pages[dst[i]] = pages[src[i]] in every tensor of the list; src / dst are int64 CPU tensors
void copy_pages(const std::vector<at::Tensor>& tensors, const at::Tensor& src, const at::Tensor& dst) {
  if (tensors.empty()) return;
  TORCH_CHECK(src.device().is_cpu() && dst.device().is_cpu() && src.scalar_type() == at::kLong && dst.scalar_type() == at::kLong &&
                  src.is_contiguous() && dst.is_contiguous() && src.dim() == 1 && dst.sizes() == src.sizes(),
              "page ids must be two int64 CPU tensors of one length");
  const at::Device dev = tensors[0].device();
  TORCH_CHECK(dev.is_cuda(), "copy_pages needs CUDA tensors");
  std::vector<teb200::PageCopyTensor> list(tensors.size());
  int64_t pages = INT_MAX;
  for (size_t i = 0; i < tensors.size(); ++i) {
    const at::Tensor& t = tensors[i];
    TORCH_CHECK(t.device() == dev && t.is_contiguous() && t.dim() >= 1, "copy_pages takes contiguous tensors of one device");
    pages = t.size(0) < pages ? t.size(0) : pages;
    list[i].base = t.data_ptr();
    list[i].page_bytes = t.size(0) > 0 ? static_cast<long long>(t.numel() / t.size(0) * t.element_size()) : 0;
  }
  const int64_t* s = src.data_ptr<int64_t>();
  const int64_t* d = dst.data_ptr<int64_t>();
  const int64_t n = src.numel();
  std::vector<int> ids(2 * static_cast<size_t>(n));
  std::vector<uint8_t> seen(static_cast<size_t>(n > 0 ? pages : 0), 0);
  for (int64_t i = 0; i < n; ++i) {
    TORCH_CHECK_VALUE(s[i] >= 0 && s[i] < pages && d[i] >= 0 && d[i] < pages, "copy_pages: page id out of range at pair ", str(i),
                      " (", str(s[i]), " -> ", str(d[i]), " of ", str(pages), " pages)");
    TORCH_CHECK_VALUE(!seen[d[i]], "copy_pages: page ", str(d[i]), " is written twice");
    seen[d[i]] = 1;
    ids[i] = static_cast<int>(s[i]);
    ids[n + i] = static_cast<int>(d[i]);
  }
  for (int64_t i = 0; i < n; ++i) TORCH_CHECK_VALUE(!seen[s[i]], "copy_pages: page ", str(s[i]), " is read and written");
  c10::cuda::CUDAGuard guard(dev);
  const cudaError_t e = teb200::copy_pages(list.data(), static_cast<int>(list.size()), ids.data(), ids.data() + n,
                                           static_cast<int>(n), cur_stream());
  TORCH_CHECK(e == cudaSuccess, "copy_pages failed: ", cudaGetErrorString(e));
}

}  // namespace

void register_kv(py::module_& m) {
  m.def("fp8_cache_append", teb200::traced("teb200.fp8_cache_append", &fp8_cache_append));
  m.def("fp8_cache_gather", teb200::traced("teb200.fp8_cache_gather", &fp8_cache_gather));
  m.def("fp8_cache_expand", teb200::traced("teb200.fp8_cache_expand", &fp8_cache_expand));
  m.def("fp8_cache_attend", teb200::traced("teb200.fp8_cache_attend", &fp8_cache_attend));
  m.def("copy_pages", teb200::traced("teb200.copy_pages", &copy_pages));
}
