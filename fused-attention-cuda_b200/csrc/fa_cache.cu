// fa_cache.cu -- C ABI of the paged 8-bit key/value cache (include/fa_sm100.h): argument checks and
// the step from the public structs to the kernels' view.  No counterpart in the reference.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "fa_cache.h"

namespace fa_sm100 {
namespace {

bool aligned(const void* p, std::uintptr_t n) {
  return (reinterpret_cast<std::uintptr_t>(p) & (n - 1)) == 0;
}

int fail(const char* fn, const char* why) {
  if (std::getenv("FA_VERBOSE") != nullptr) std::fprintf(stderr, "%s: %s\n", fn, why);
  return cudaErrorInvalidValue;
}

// Positive strides that are multiples of 16 bytes and leave room for 2^63-byte offsets.
bool strides_ok(const long long* st, int n, size_t eb) {
  for (int i = 0; i < n; ++i) {
    if (st[i] <= 0 || st[i] >= (1ll << 40) || (st[i] * static_cast<long long>(eb)) % 16 != 0)
      return false;
  }
  return true;
}

const char* check_cache(const fa_cache_t* c, int T) {
  if (c == nullptr) return "cache must be non-null";
  if (c->D != 64 && c->D != 128) return "D must be 64 or 128";
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return "page_size must be 16, 32, 64 or 128";
  if (c->Hkv <= 0 || c->num_pages <= 0 || c->num_pages > 0x7fffffffll)
    return "Hkv and num_pages must be > 0";
  if (c->n_seqs <= 0 || c->max_pages <= 0 || c->table_stride < c->max_pages)
    return "n_seqs and max_pages must be > 0, table_stride >= max_pages";
  if (static_cast<long long>(c->max_pages) * c->page_size > 0x7fffffffll - 128)
    return "max_pages * page_size does not fit an int";
  if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr ||
      c->block_table == nullptr || c->seq_lens == nullptr)
    return "cache pointers must be non-null";
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return "pages must be 16-byte aligned";
  if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->block_table, 4) ||
      !aligned(c->seq_lens, 4) || !aligned(c->cu_seqlens, 4))
    return "scales, table, lengths and offsets must be 4-byte aligned";
  if (!strides_ok(c->k_strides, 3, 1) || !strides_ok(c->v_strides, 3, 1))
    return "page strides must be positive multiples of 16 bytes";
  if (T < 0) return "T must be >= 0";
  if (c->cu_seqlens == nullptr && T % c->n_seqs != 0)
    return "without cu_seqlens, T must be a multiple of n_seqs";
  return nullptr;
}

CacheView view_of(const fa_cache_t* c, int T, unsigned* status) {
  CacheView v;
  v.k = static_cast<unsigned char*>(c->k);
  v.v = static_cast<unsigned char*>(c->v);
  v.k_scale = c->k_scale;
  v.v_scale = c->v_scale;
  for (int i = 0; i < 3; ++i) {
    v.ks[i] = c->k_strides[i];
    v.vs[i] = c->v_strides[i];
  }
  v.num_pages = c->num_pages;
  v.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  v.Hkv = c->Hkv;
  v.block_table = c->block_table;
  v.table_stride = c->table_stride;
  v.max_pages = c->max_pages;
  v.seq_lens = c->seq_lens;
  v.cu_seqlens = c->cu_seqlens;
  v.n_seqs = c->n_seqs;
  v.T = T;
  v.status = status;
  return v;
}

// cudaSuccess on compute capability 10.0, where these kernels run.
cudaError_t check_device() {
  int dev = 0, major = 0, minor = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess)
    e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess)
    e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (e != cudaSuccess) return e;
  return major == 10 && minor == 0 ? cudaSuccess : cudaErrorNotSupported;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      return nullptr;
    }
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

cudaError_t page_map(CUtensorMap* m, int* pos, void* base, const long long st[3],
                     const CacheView& c, int D, int rows) {
  const EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return cudaErrorNotSupported;
  const long long stride[3] = {st[2], st[1], st[0]};  // token, head, page
  const long long size[3] = {1ll << c.page_shift, c.Hkv, c.num_pages};
  int order[3] = {0, 1, 2};
  for (int i = 1; i < 3; ++i) {
    for (int j = i; j > 0 && stride[order[j]] < stride[order[j - 1]]; --j) {
      const int t = order[j];
      order[j] = order[j - 1];
      order[j - 1] = t;
    }
  }
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), 0, 0, 0};
  cuuint64_t strides[3];
  cuuint32_t box[4] = {static_cast<cuuint32_t>(D), 1u, 1u, 1u};
  *pos = 0;
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(size[order[i]]);
    strides[i] = static_cast<cuuint64_t>(stride[order[i]]);
    if (order[i] == 0) box[i + 1] = static_cast<cuuint32_t>(rows);
    *pos |= i << (2 * order[i]);
  }
  const cuuint32_t estride[4] = {1u, 1u, 1u, 1u};
  const CUresult r =
      enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, estride,
          CU_TENSOR_MAP_INTERLEAVE_NONE,
          D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace

cudaError_t make_page_maps(PageMaps* m, const CacheView& c, int D, int rows) {
  const cudaError_t e = page_map(&m->k, &m->k_pos, c.k, c.ks, c, D, rows);
  return e != cudaSuccess ? e : page_map(&m->v, &m->v_pos, c.v, c.vs, c, D, rows);
}

int multiprocessors() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

}  // namespace fa_sm100

using namespace fa_sm100;

extern "C" int fa_cache_append(int dtype, const fa_cache_t* c, const fa_append_t* p, int T,
                               cudaStream_t stream) {
  const char* fn = "fa_cache_append";
  if (const char* why = check_cache(c, T)) return fail(fn, why);
  if (p == nullptr) return fail(fn, "append parameters must be non-null");
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return fail(fn, "dtype must be fp16 or bf16");
  if (p->k == nullptr || p->v == nullptr || !aligned(p->k, 16) || !aligned(p->v, 16))
    return fail(fn, "k and v must be non-null and 16-byte aligned");
  if (!strides_ok(p->k_strides, 2, 2) || !strides_ok(p->v_strides, 2, 2))
    return fail(fn, "k and v strides must be positive multiples of 16 bytes");
  const bool rotates = p->cos != nullptr || p->sin != nullptr;
  if (rotates) {
    if (p->cos == nullptr || p->sin == nullptr || !aligned(p->cos, 16) || !aligned(p->sin, 16))
      return fail(fn, "cos and sin must both be given, 16-byte aligned");
    if (p->rot_dim <= 0 || p->rot_dim % 16 != 0 || p->rot_dim > c->D)
      return fail(fn, "rot_dim must be a positive multiple of 16, at most D");
    if (p->table_rows <= 0) return fail(fn, "cos and sin must have rows");
  }
  if (p->q != nullptr) {
    if (!rotates) return fail(fn, "q needs cos and sin");
    if (p->H <= 0 || p->q_out == nullptr || !aligned(p->q, 16) || !aligned(p->q_out, 16) ||
        !strides_ok(p->q_strides, 2, 2))
      return fail(fn, "q and q_out must be 16-byte aligned, H > 0, strides multiples of 16 bytes");
  }
  if (const cudaError_t e = check_device()) return e;
  if (c->k == c->v || c->k_scale == c->v_scale)
    return fail(fn, "keys and values need pages and scales of their own");
  if (p->q != nullptr && p->q == p->q_out) return fail(fn, "q_out must not overlap q");
  if (T == 0) return cudaSuccess;
  cudaError_t e = cudaSuccess;
  unsigned* status = status_word(&e);
  if (e != cudaSuccess) return e;
  AppendArgs a;
  a.c = view_of(c, T, status);
  a.dtype = dtype;
  a.H = p->q != nullptr ? p->H : 0;
  a.D = c->D;
  a.k = p->k;
  a.v = p->v;
  a.q = p->q;
  a.q_out = p->q_out;
  for (int i = 0; i < 2; ++i) {
    a.sk[i] = p->k_strides[i];
    a.sv[i] = p->v_strides[i];
    a.sq[i] = p->q_strides[i];
  }
  a.cos = p->cos;
  a.sin = p->sin;
  a.table_rows = p->table_rows;
  a.rot_dim = rotates ? p->rot_dim : 0;
  a.interleaved = p->interleaved != 0;
  return launch_cache_append(a, stream);
}

extern "C" size_t fa_cache_attention_workspace_bytes(const fa_cache_t* c, int H, int T) {
  if (check_cache(c, T) != nullptr || H <= 0 || H % c->Hkv != 0) return 0;
  return cache_attention_workspace(H, c->Hkv, c->D, T, c->n_seqs, multiprocessors());
}

extern "C" int fa_cache_attention(int dtype, const fa_cache_t* c, const void* q,
                                  const long long* q_strides, void* o, float* lse, void* workspace,
                                  int T, int H, float scale, int causal, cudaStream_t stream) {
  const char* fn = "fa_cache_attention";
  if (const char* why = check_cache(c, T)) return fail(fn, why);
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16) return fail(fn, "dtype must be fp16 or bf16");
  if (H <= 0 || H % c->Hkv != 0) return fail(fn, "H must be a positive multiple of Hkv");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(fn, "scale must be finite and > 0");
  if (static_cast<long long>(T) * (H / c->Hkv) > 0x7fffffffll - 128)
    return fail(fn, "T * (H / Hkv) does not fit an int");
  if (T > 0 && (q == nullptr || o == nullptr || lse == nullptr || q_strides == nullptr ||
                !aligned(q, 16) || !aligned(o, 16) || !aligned(lse, 4)))
    return fail(fn, "q and o must be non-null and 16-byte aligned, lse non-null");
  if (T > 0 && !strides_ok(q_strides, 2, 2))
    return fail(fn, "q strides must be positive multiples of 16 bytes");
  if (const cudaError_t e = check_device()) return e;
  if (T == 0) return cudaSuccess;
  if (o == q) return fail(fn, "o must not overlap q");
  if (workspace == nullptr || !aligned(workspace, 16))
    return fail(fn, "workspace must be non-null and 16-byte aligned");
  cudaError_t e = cudaSuccess;
  unsigned* status = status_word(&e);
  if (e != cudaSuccess) return e;
  CacheAttnArgs a;
  a.c = view_of(c, T, status);
  a.dtype = dtype;
  a.H = H;
  a.D = c->D;
  a.q = q;
  a.sq[0] = q_strides[0];
  a.sq[1] = q_strides[1];
  a.o = o;
  a.lse = lse;
  a.scale = scale;
  a.causal = causal != 0;
  a.workspace = workspace;
  a.timeout_ns = wait_timeout_ns();
  return launch_cache_attention(a, stream);
}
