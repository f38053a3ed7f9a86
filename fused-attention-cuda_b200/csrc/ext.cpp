// fused_attn._C -- PyTorch operator surface over the C ABI in include/fa_sm100.h.
//
// Reference counterpart: python/fused_attn/ext.cpp.  Same library name (fused_attn), same
// validation messages (make_params, ext.cpp:82-126), same bare PyInit__C module (ext.cpp:240-253)
// so `from . import _C` runs the TORCH_LIBRARY initialisers.  One deliberate change:
//   fused_attn::forward(Tensor q, Tensor k, Tensor v, bool is_causal, float scale)
//       -> (Tensor, Tensor)                           (O, LSE) -- the reference returns O only
// because the B200 build's contract is "forward -> (O, LSE)".  forward_stage keeps its
// (Tensor, Tensor) schema; its LSE is empty for the stages that do not write one (1, 2).
//
// Host C++ only: every launch happens behind fa_forward() in libfa_sm100.so.
#include <Python.h>  // first, per the CPython docs
// (blank comment line keeps include sorters from moving Python.h)

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/library.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "fa_sm100.h"

namespace {

// The reference's stage numbering (fa::Impl): 1..5, with an LSE from stage 3 up.  Constructing a
// Stage is the range check.
struct Stage {
  static constexpr int kLowest = 1;
  static constexpr int kHighest = 5;
  static constexpr int kFirstWithLse = 3;
  int value;
  explicit Stage(int64_t s) : value(static_cast<int>(s)) {
    TORCH_CHECK(s >= kLowest && s <= kHighest, "fused_attn: stage must be in 1..5, got ", s);
  }
  bool writes_lse() const { return value >= kFirstWithLse; }
};

int to_fa_dtype(at::ScalarType t) {
  if (t == at::kFloat) return FA_DTYPE_F32;
  if (t == at::kHalf) return FA_DTYPE_F16;
  TORCH_CHECK(t == at::kBFloat16, "fused_attn: unsupported dtype ", t,
              " (supported: float32, float16, bfloat16)");
  return FA_DTYPE_BF16;
}

int dtype_from_name(const std::string& name) {
  if (name == "fp32") return FA_DTYPE_F32;
  if (name == "fp16") return FA_DTYPE_F16;
  TORCH_CHECK(name == "bf16", "fused_attn: unknown dtype name '", name,
              "' (expected fp32, fp16 or bf16)");
  return FA_DTYPE_BF16;
}

// fa_impl_supports' `sm` (major * 10 + minor) for a CUDA device index (-1: the current one).
int sm_number(int device_index = -1) {
  const cudaDeviceProp* prop = device_index < 0 ? at::cuda::getCurrentDeviceProperties()
                                                : at::cuda::getDeviceProperties(device_index);
  return 10 * prop->major + prop->minor;
}

// A size or knob narrowed to the C ABI's `int` fields, rejected when it does not fit.
int abi_int(int64_t v, const char* what) {
  const bool fits = v >= 0 && v <= static_cast<int64_t>(std::numeric_limits<int>::max());
  TORCH_CHECK(fits, "fused_attn: ", what, "=", v, " does not fit fa_params_t (int)");
  return static_cast<int>(v);
}

// Input contract (reference ext.cpp:82-126): every violation is a RuntimeError, never a fault.
// With `strided`, q/k/v may be any [B, H, N, D] views whose head dim is contiguous and whose other
// strides are positive multiples of 16 bytes (no counterpart in the reference, which requires
// contiguous inputs).
fa_params_t make_params(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                        bool is_causal, double scale, bool strided = false) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(),
              "fused_attn: q, k, v must be CUDA tensors");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device(),
              "fused_attn: q, k, v must live on the same device");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
              "fused_attn: q, k, v must be [B, H, N, D]; got ", q.dim(), "-D, ", k.dim(), "-D, ",
              v.dim(), "-D");
  if (!strided) {
    TORCH_CHECK(q.is_contiguous() && k.is_contiguous() && v.is_contiguous(),
                "fused_attn: q, k, v must be contiguous [B, H, N, D] (call .contiguous())");
  } else {
    for (const at::Tensor* t : {&q, &k, &v}) {
      TORCH_CHECK(t->dim() == 4 && t->stride(3) == 1,
                  "fused_attn: strided views need a contiguous head dim (stride(3) == 1)");
      for (int d = 0; d < 3; ++d) {
        TORCH_CHECK(t->stride(d) > 0 && (t->stride(d) * t->element_size()) % 16 == 0,
                    "fused_attn: strided views need positive strides that are multiples of 16 "
                    "bytes; got stride(", d, ") = ", t->stride(d));
      }
    }
  }
  for (const at::Tensor* t : {&q, &k, &v}) {
    TORCH_CHECK(reinterpret_cast<std::uintptr_t>(t->data_ptr()) % 16 == 0,
                "fused_attn: q/k/v must be 16-byte aligned (use a fresh contiguous tensor)");
  }
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "fused_attn: q, k, v must share one dtype; got ", q.scalar_type(), ", ",
              k.scalar_type(), ", ", v.scalar_type());
  (void)to_fa_dtype(q.scalar_type());

  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  const int64_t Hkv = k.size(1);
  TORCH_CHECK(k.size(0) == B && v.size(0) == B, "fused_attn: batch mismatch between q, k, v");
  TORCH_CHECK(v.size(1) == Hkv, "fused_attn: k and v must have the same number of heads");
  TORCH_CHECK(k.size(2) == N && v.size(2) == N,
              "fused_attn: Nq == Nkv is required in-window (got Nq=", N, ", Nkv=", k.size(2), ")");
  TORCH_CHECK(k.size(3) == D && v.size(3) == D, "fused_attn: head-dim mismatch between q, k, v");
  TORCH_CHECK(D == 64 || D == 128, "fused_attn: D must be 64 or 128, got ", D);
  TORCH_CHECK(N % 32 == 0, "fused_attn: N must be a multiple of 32, got ", N,
              " (ragged sequence lengths are a stated in-window limitation)");
  TORCH_CHECK(Hkv >= 1 && H % Hkv == 0, "fused_attn: H=", H, " must be a multiple of Hkv=", Hkv);
  TORCH_CHECK(scale > 0.0 && std::isfinite(scale), "fused_attn: scale must be finite and > 0, got ",
              scale);

  fa_params_t p;
  p.B = abi_int(B, "B");
  p.H = abi_int(H, "H");
  p.Hkv = abi_int(Hkv, "Hkv");
  p.N = abi_int(N, "N");
  p.D = abi_int(D, "D");
  p.scale = static_cast<float>(scale);
  p.causal = is_causal ? 1 : 0;
  return p;
}

// The stage's outputs and scratch on q's device.  O takes q's layout (empty_like keeps the strides
// of a dense view, e.g. the [B, H, N, D] transpose of a [B, N, H, D] buffer), so a head merge after
// the op is a free view too.  The LSE is [B, H, N] fp32, or empty for a stage that writes none.
struct StageBuffers {
  at::Tensor o, lse, workspace;
  StageBuffers(const at::Tensor& q, const fa_params_t& p, Stage stage, int dtype) {
    const auto f32 = q.options().dtype(at::kFloat);
    o = at::empty_like(q);
    lse = stage.writes_lse() ? at::empty({p.B, p.H, p.N}, f32) : at::empty({0}, f32);
    const std::size_t scratch = fa_workspace_bytes(stage.value, dtype, &p);
    if (scratch > 0) {
      workspace = at::empty({static_cast<int64_t>(scratch)}, q.options().dtype(at::kByte));
    }
  }
  float* lse_ptr() { return lse.numel() > 0 ? lse.data_ptr<float>() : nullptr; }
  void* workspace_ptr() { return workspace.defined() ? workspace.data_ptr() : nullptr; }
};

std::tuple<at::Tensor, at::Tensor> run_stage(const at::Tensor& q, const at::Tensor& k,
                                             const at::Tensor& v, bool is_causal, double scale,
                                             Stage stage, bool strided = false) {
  const fa_params_t p = make_params(q, k, v, is_causal, scale, strided);
  const c10::cuda::CUDAGuard guard(q.device());
  const int impl = stage.value;
  const int dtype = to_fa_dtype(q.scalar_type());
  const int sm = sm_number(q.device().index());
  TORCH_CHECK(fa_impl_supports(impl, dtype, p.D, sm), "fused_attn: stage ", impl, " (",
              fa_impl_name(impl), ") is not implemented for ", fa_dtype_name(dtype), " D=", p.D,
              " on sm_", sm);
  StageBuffers out(q, p, stage, dtype);
  at::Tensor& o = out.o;
  const bool has_lse = stage.writes_lse();
  void* ws_ptr = out.workspace_ptr();
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(q.device().index()).stream();
  int err;
  if (strided) {
    TORCH_CHECK(o.stride(3) == 1, "fused_attn: output layout has a non-contiguous head dim");
    fa_strides_t st;
    const at::Tensor* ts[4] = {&q, &k, &v, &o};
    long long* dst[4] = {st.q, st.k, st.v, st.o};
    for (int t = 0; t < 4; ++t) {
      for (int d = 0; d < 3; ++d) dst[t][d] = static_cast<long long>(ts[t]->stride(d));
    }
    err = fa_forward_strided(impl, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                             has_lse ? out.lse_ptr() : nullptr, ws_ptr, &p, &st, stream);
  } else {
    err = fa_forward(impl, dtype, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                     has_lse ? out.lse_ptr() : nullptr, ws_ptr, &p, stream);
  }
  TORCH_CHECK(err == 0, "fused_attn: stage ", impl, " (", fa_impl_name(impl),
              ") failed: ", cudaGetErrorString(static_cast<cudaError_t>(err)));
  return std::make_tuple(std::move(out.o), std::move(out.lse));
}

// The stage `forward` runs: the highest one with an LSE that this device supports for the dtype
// and head dim (the reference's forward picks its best stage the same way, ext.cpp:174-188).
Stage best_stage(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool is_causal,
                 double scale, bool strided) {
  const fa_params_t p = make_params(q, k, v, is_causal, scale, strided);
  const int dtype = to_fa_dtype(q.scalar_type());
  const int sm = sm_number(q.device().index());
  int chosen = 0;
  for (int s = Stage::kHighest; s >= Stage::kFirstWithLse && chosen == 0; --s) {
    if (fa_impl_supports(s, dtype, p.D, sm)) chosen = s;
  }
  TORCH_CHECK(chosen != 0, "fused_attn: no stage is implemented for ", fa_dtype_name(dtype),
              " D=", p.D, " on sm_", sm);
  return Stage(chosen);
}

std::tuple<at::Tensor, at::Tensor> forward_cuda(const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& v, bool is_causal,
                                                double scale) {
  return run_stage(q, k, v, is_causal, scale, best_stage(q, k, v, is_causal, scale, false));
}

// forward over strided [B, H, N, D] views (no counterpart in the reference): same stage choice.
std::tuple<at::Tensor, at::Tensor> forward_strided_cuda(const at::Tensor& q, const at::Tensor& k,
                                                        const at::Tensor& v, bool is_causal,
                                                        double scale) {
  return run_stage(q, k, v, is_causal, scale, best_stage(q, k, v, is_causal, scale, true), true);
}

std::tuple<at::Tensor, at::Tensor> forward_stage_cuda(const at::Tensor& q, const at::Tensor& k,
                                                      const at::Tensor& v, bool is_causal,
                                                      double scale, int64_t stage) {
  return run_stage(q, k, v, is_causal, scale, Stage(stage));
}

// LSE-weighted merge of partials over disjoint key sets (no counterpart in the reference).
std::tuple<at::Tensor, at::Tensor> combine_cuda(at::TensorList o_parts, at::TensorList lse_parts) {
  TORCH_CHECK(!o_parts.empty() && o_parts.size() == lse_parts.size(),
              "fused_attn: combine needs as many LSE tensors as O partials (at least one)");
  TORCH_CHECK(o_parts.size() <= FA_COMBINE_MAX_SPLITS, "fused_attn: combine takes at most ",
              FA_COMBINE_MAX_SPLITS, " partials, got ", o_parts.size());
  const at::Tensor& o0 = o_parts[0];
  TORCH_CHECK(o0.is_cuda() && o0.dim() == 4, "fused_attn: partials must be CUDA [B, H, N, D]");
  const int64_t B = o0.size(0), H = o0.size(1), N = o0.size(2), D = o0.size(3);
  TORCH_CHECK(D == 64 || D == 128, "fused_attn: D must be 64 or 128, got ", D);
  std::vector<const void*> op;
  std::vector<const float*> lp;
  for (size_t i = 0; i < o_parts.size(); ++i) {
    const at::Tensor& o = o_parts[i];
    const at::Tensor& l = lse_parts[i];
    TORCH_CHECK(o.device() == o0.device() && l.device() == o0.device(),
                "fused_attn: combine inputs must live on one device");
    TORCH_CHECK(o.sizes() == o0.sizes() && o.scalar_type() == o0.scalar_type() &&
                    o.is_contiguous(),
                "fused_attn: O partials must be contiguous with one shape and dtype");
    TORCH_CHECK(l.scalar_type() == at::kFloat && l.is_contiguous() && l.dim() == 3 &&
                    l.size(0) == B && l.size(1) == H && l.size(2) == N,
                "fused_attn: LSE partials must be contiguous fp32 [B, H, N]");
    TORCH_CHECK(reinterpret_cast<std::uintptr_t>(o.data_ptr()) % 16 == 0,
                "fused_attn: O partials must be 16-byte aligned");
    op.push_back(o.data_ptr());
    lp.push_back(l.data_ptr<float>());
  }
  const c10::cuda::CUDAGuard guard(o0.device());
  at::Tensor out = at::empty_like(o0, at::MemoryFormat::Contiguous);
  at::Tensor lse = at::empty({B, H, N}, o0.options().dtype(at::kFloat));
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(o0.device().index()).stream();
  const int err = fa_combine(to_fa_dtype(o0.scalar_type()), static_cast<int>(op.size()), op.data(),
                             lp.data(), out.data_ptr(), lse.data_ptr<float>(),
                             abi_int(B, "B"), abi_int(H, "H"), abi_int(N, "N"),
                             abi_int(D, "D"), stream);
  TORCH_CHECK(err == 0, "fused_attn: combine failed: ",
              cudaGetErrorString(static_cast<cudaError_t>(err)));
  return std::make_tuple(std::move(out), std::move(lse));
}

// ---- paged 8-bit cache (no counterpart in the reference) ----

// A stride of a view, or `any` where the dimension has one element and its stride says nothing.
long long stride_of(const at::Tensor& t, int d, long long any) {
  return t.size(d) <= 1 ? any : static_cast<long long>(t.stride(d));
}

void check_i32(const at::Tensor& t, const char* what, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, "fused_attn: ", what,
              " must live on the cache's device");
  TORCH_CHECK(t.scalar_type() == at::kInt, "fused_attn: ", what, " must be int32, got ",
              t.scalar_type());
}

// New rows [T, heads, D]: fp16 / bf16 views with a contiguous head dim.
void check_rows(const at::Tensor& t, const char* what, const at::Device& dev, int64_t D,
                long long (&st)[2]) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, "fused_attn: ", what,
              " must live on the cache's device");
  TORCH_CHECK(t.dim() == 3 && t.size(2) == D, "fused_attn: ", what, " must be [T, heads, ", D,
              "], got ", t.sizes());
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, "fused_attn: ",
              what, " must be float16 or bfloat16, got ", t.scalar_type());
  TORCH_CHECK(t.numel() == 0 || t.stride(2) == 1, "fused_attn: ", what,
              " needs a contiguous head dim (stride(2) == 1)");
  st[0] = stride_of(t, 0, D);
  st[1] = stride_of(t, 1, D);
  for (int d = 0; d < 2; ++d) {
    TORCH_CHECK(t.numel() == 0 || (st[d] > 0 && st[d] % 8 == 0), "fused_attn: ", what,
                " needs positive strides that are multiples of 16 bytes; got stride(", d,
                ") = ", st[d]);
  }
  TORCH_CHECK(reinterpret_cast<std::uintptr_t>(t.data_ptr()) % 16 == 0, "fused_attn: ", what,
              " must be 16-byte aligned");
}

// The cache and the batch; T is the number of packed rows.
fa_cache_t make_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                      const at::Tensor& v_scale, const at::Tensor& block_table,
                      const at::Tensor& seq_lens, const std::optional<at::Tensor>& cu_seqlens,
                      int64_t T) {
  fa_cache_t c;
  const at::Device dev = k.device();
  TORCH_CHECK(k.is_cuda(), "fused_attn: k_cache must be a CUDA tensor");
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(),
              "fused_attn: k_cache and v_cache must be [pages, Hkv, page_size, D], got ", k.sizes(),
              " and ", v.sizes());
  const at::Tensor* caches[2] = {&k, &v};
  long long* strides[2] = {c.k_strides, c.v_strides};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *caches[i];
    const char* what = i == 0 ? "k_cache" : "v_cache";
    TORCH_CHECK(t.device() == dev, "fused_attn: the cache must live on one device");
    TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn, "fused_attn: ", what,
                " must be float8_e4m3fn, got ", t.scalar_type());
    TORCH_CHECK(t.numel() > 0, "fused_attn: ", what, " is empty");
    TORCH_CHECK(t.stride(3) == 1, "fused_attn: ", what,
                " needs a contiguous head dim (stride(3) == 1)");
    for (int d = 0; d < 3; ++d) {
      strides[i][d] = stride_of(t, d, t.size(3));
      TORCH_CHECK(strides[i][d] > 0 && strides[i][d] % 16 == 0, "fused_attn: ", what,
                  " needs positive strides that are multiples of 16 bytes; got stride(", d,
                  ") = ", strides[i][d]);
    }
    TORCH_CHECK(reinterpret_cast<std::uintptr_t>(t.data_ptr()) % 16 == 0, "fused_attn: ", what,
                " must be 16-byte aligned");
  }
  const int64_t P = k.size(0), Hkv = k.size(1), page = k.size(2), D = k.size(3);
  TORCH_CHECK(D == 64 || D == 128, "fused_attn: D must be 64 or 128, got ", D);
  TORCH_CHECK(page == 16 || page == 32 || page == 64 || page == 128,
              "fused_attn: page_size must be 16, 32, 64 or 128, got ", page);
  for (const at::Tensor* t : {&k_scale, &v_scale}) {
    TORCH_CHECK(t->is_cuda() && t->device() == dev && t->scalar_type() == at::kFloat &&
                    t->dim() == 2 && t->size(0) == P && t->size(1) == Hkv && t->is_contiguous(),
                "fused_attn: k_scale and v_scale must be contiguous float32 [", P, ", ", Hkv,
                "] on the cache's device");
  }
  check_i32(block_table, "block_table", dev);
  check_i32(seq_lens, "seq_lens", dev);
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.is_contiguous(),
              "fused_attn: seq_lens must be a contiguous [sequences]");
  const int64_t S = seq_lens.size(0);
  TORCH_CHECK(block_table.dim() == 2 && block_table.size(0) == S && block_table.size(1) >= 1 &&
                  (block_table.size(1) == 1 || block_table.stride(1) == 1),
              "fused_attn: block_table must be [", S, ", max_pages] with contiguous rows, got ",
              block_table.sizes());
  c.table_stride = stride_of(block_table, 0, block_table.size(1));
  TORCH_CHECK(c.table_stride >= block_table.size(1),
              "fused_attn: block_table rows must not overlap");
  if (cu_seqlens.has_value()) {
    check_i32(*cu_seqlens, "cu_seqlens", dev);
    TORCH_CHECK(cu_seqlens->dim() == 1 && cu_seqlens->size(0) == S + 1 &&
                    cu_seqlens->is_contiguous(),
                "fused_attn: cu_seqlens must be a contiguous [", S + 1, "]");
  } else {
    TORCH_CHECK(S == 0 ? T == 0 : T % S == 0, "fused_attn: without cu_seqlens, T=", T,
                " must be a multiple of the ", S, " sequences");
  }
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_scale = k_scale.data_ptr<float>();
  c.v_scale = v_scale.data_ptr<float>();
  c.num_pages = P;
  c.page_size = abi_int(page, "page_size");
  c.Hkv = abi_int(Hkv, "Hkv");
  c.D = abi_int(D, "D");
  c.block_table = block_table.data_ptr<int>();
  c.max_pages = abi_int(block_table.size(1), "max_pages");
  TORCH_CHECK(block_table.size(1) * page <= std::numeric_limits<int>::max() - 128,
              "fused_attn: block_table has room for more keys than fit an int");
  c.seq_lens = seq_lens.data_ptr<int>();
  c.cu_seqlens = cu_seqlens.has_value() ? cu_seqlens->data_ptr<int>() : nullptr;
  c.n_seqs = abi_int(S, "sequences");
  return c;
}

// [T, H, D] rotated q, or an empty tensor without q.
at::Tensor cache_append_cuda(const std::optional<at::Tensor>& q, const at::Tensor& k,
                             const at::Tensor& v, const at::Tensor& k_cache,
                             const at::Tensor& v_cache, const at::Tensor& k_scale,
                             const at::Tensor& v_scale, const at::Tensor& block_table,
                             const at::Tensor& seq_lens,
                             const std::optional<at::Tensor>& cu_seqlens,
                             const std::optional<at::Tensor>& cos,
                             const std::optional<at::Tensor>& sin, bool interleaved) {
  TORCH_CHECK(k.dim() == 3, "fused_attn: k must be [T, heads, D], got ", k.sizes());
  const int64_t T = k.size(0);
  const fa_cache_t c = make_cache(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                                  cu_seqlens, T);
  const at::Device dev = k_cache.device();
  TORCH_CHECK(c.k != c.v && c.k_scale != c.v_scale,
              "fused_attn: k_cache and v_cache, k_scale and v_scale must be different tensors");
  fa_append_t p = {};
  check_rows(k, "k", dev, c.D, p.k_strides);
  check_rows(v, "v", dev, c.D, p.v_strides);
  TORCH_CHECK(k.scalar_type() == v.scalar_type() && v.size(0) == T && k.size(1) == c.Hkv &&
                  v.size(1) == c.Hkv,
              "fused_attn: k and v must be [T, ", c.Hkv, ", D] of one dtype, got ", k.sizes(),
              " and ", v.sizes());
  TORCH_CHECK(cos.has_value() == sin.has_value(), "fused_attn: cos and sin come together");
  if (cos.has_value()) {
    for (const at::Tensor* t : {&*cos, &*sin}) {
      TORCH_CHECK(t->is_cuda() && t->device() == dev && t->scalar_type() == at::kFloat &&
                      t->dim() == 2 && t->sizes() == cos->sizes() && t->is_contiguous() &&
                      t->size(0) >= 1 &&
                      reinterpret_cast<std::uintptr_t>(t->data_ptr()) % 16 == 0,
                  "fused_attn: cos and sin must be contiguous, 16-byte aligned float32 "
                  "[positions, rot_dim / 2] on the cache's device");
    }
    const int64_t rot = 2 * cos->size(1);
    TORCH_CHECK(rot >= 16 && rot % 16 == 0 && rot <= c.D,
                "fused_attn: rot_dim must be a multiple of 16 in 16..", c.D, ", got ", rot);
    p.cos = cos->data_ptr<float>();
    p.sin = sin->data_ptr<float>();
    p.table_rows = cos->size(0);
    p.rot_dim = abi_int(rot, "rot_dim");
    p.interleaved = interleaved ? 1 : 0;
  }
  at::Tensor out = at::empty({0}, k.options());
  const c10::cuda::CUDAGuard guard(dev);
  if (q.has_value()) {
    TORCH_CHECK(cos.has_value(), "fused_attn: q is rotated and needs cos and sin");
    check_rows(*q, "q", dev, c.D, p.q_strides);
    TORCH_CHECK(q->scalar_type() == k.scalar_type() && q->size(0) == T && q->size(1) >= 1,
                "fused_attn: q must be [T, H, D] of k's dtype, got ", q->sizes());
    p.H = abi_int(q->size(1), "H");
    out = c.n_seqs == 0 ? at::zeros(q->sizes(), q->options())
                        : at::empty(q->sizes(), q->options(), at::MemoryFormat::Contiguous);
    p.q = q->data_ptr();
    p.q_out = out.data_ptr();
  }
  if (T == 0 || c.n_seqs == 0) return out;
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int err = fa_cache_append(to_fa_dtype(k.scalar_type()), &c, &p, abi_int(T, "T"), stream);
  TORCH_CHECK(err == 0, "fused_attn: cache_append failed: ",
              cudaGetErrorString(static_cast<cudaError_t>(err)));
  return out;
}

std::tuple<at::Tensor, at::Tensor> cache_attention_cuda(
    const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
    const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
    const at::Tensor& seq_lens, const std::optional<at::Tensor>& cu_seqlens, bool is_causal,
    double scale) {
  TORCH_CHECK(q.dim() == 3, "fused_attn: q must be [T, heads, D], got ", q.sizes());
  const int64_t T = q.size(0), H = q.size(1);
  const fa_cache_t c = make_cache(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                                  cu_seqlens, T);
  const at::Device dev = k_cache.device();
  long long q_strides[2];
  check_rows(q, "q", dev, c.D, q_strides);
  TORCH_CHECK(H >= 1 && H % c.Hkv == 0, "fused_attn: H=", H, " must be a multiple of Hkv=", c.Hkv);
  TORCH_CHECK(scale > 0.0 && std::isfinite(scale), "fused_attn: scale must be finite and > 0, got ",
              scale);
  const c10::cuda::CUDAGuard guard(dev);
  const auto f32 = q.options().dtype(at::kFloat);
  if (T == 0 || c.n_seqs == 0) {
    return std::make_tuple(at::zeros(q.sizes(), q.options()), at::zeros({T, H}, f32));
  }
  at::Tensor o = at::empty(q.sizes(), q.options(), at::MemoryFormat::Contiguous);
  at::Tensor lse = at::empty({T, H}, f32);
  const std::size_t bytes =
      fa_cache_attention_workspace_bytes(&c, abi_int(H, "H"), abi_int(T, "T"));
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int err = fa_cache_attention(to_fa_dtype(q.scalar_type()), &c, q.data_ptr(), q_strides,
                                     o.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(),
                                     abi_int(T, "T"), abi_int(H, "H"), static_cast<float>(scale),
                                     is_causal ? 1 : 0, stream);
  TORCH_CHECK(err == 0, "fused_attn: cache_attention failed: ",
              cudaGetErrorString(static_cast<cudaError_t>(err)));
  return std::make_tuple(std::move(o), std::move(lse));
}

void set_debug_overrides_op(int64_t block_m, int64_t block_n) {
  fa_set_debug_overrides(abi_int(block_m, "block_m"), abi_int(block_n, "block_n"));
}

bool impl_supports_op(int64_t stage, std::string dtype, int64_t D) {
  const Stage st(stage);
  if (c10::cuda::device_count() == 0) return false;
  return fa_impl_supports(st.value, dtype_from_name(dtype), abi_int(D, "D"), sm_number()) != 0;
}

std::string impl_name_op(int64_t stage) { return fa_impl_name(Stage(stage).value); }

}  // namespace

TORCH_LIBRARY(fused_attn, m) {
  m.def("forward(Tensor q, Tensor k, Tensor v, bool is_causal, float scale) -> (Tensor, Tensor)");
  m.def(
      "forward_strided(Tensor q, Tensor k, Tensor v, bool is_causal, float scale)"
      " -> (Tensor, Tensor)");
  m.def(
      "forward_stage(Tensor q, Tensor k, Tensor v, bool is_causal, float scale, int stage)"
      " -> (Tensor, Tensor)");
  m.def("combine(Tensor[] o_parts, Tensor[] lse_parts) -> (Tensor, Tensor)");
  m.def(
      "cache_append(Tensor? q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache,"
      " Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor block_table, Tensor seq_lens,"
      " Tensor? cu_seqlens, Tensor? cos, Tensor? sin, bool interleaved) -> Tensor");
  m.def(
      "cache_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale,"
      " Tensor block_table, Tensor seq_lens, Tensor? cu_seqlens, bool is_causal, float scale)"
      " -> (Tensor, Tensor)");
  m.def("set_debug_overrides(int block_m, int block_n) -> ()", &set_debug_overrides_op);
  m.def("impl_supports(int stage, str dtype, int D) -> bool", &impl_supports_op);
  m.def("impl_name(int stage) -> str", &impl_name_op);
}

TORCH_LIBRARY_IMPL(fused_attn, CUDA, m) {
  m.impl("forward", &forward_cuda);
  m.impl("forward_strided", &forward_strided_cuda);
  m.impl("combine", &combine_cuda);
  m.impl("forward_stage", &forward_stage_cuda);
  m.impl("cache_append", &cache_append_cuda);
  m.impl("cache_attention", &cache_attention_cuda);
}

// A module with no functions of its own: importing it runs the TORCH_LIBRARY registrations above,
// and the ops are reached as torch.ops.fused_attn.*.
static PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_C",
                               "B200 SDPA forward; ops under torch.ops.fused_attn", -1};

extern "C" PyObject* PyInit__C(void) { return PyModule_Create(&g_module); }
