// decode_abi.cpp -- extern "C" entry points of the decode step: the paged key-value cache
// (kvcache.hpp) and the 4-bit group-scaled Dense layer (gdense.hpp).
#include "abi_handles.hpp"

#include "dense.hpp"
#include "gdense.hpp"
#include "kvcache.hpp"

#include <cmath>
#include <cstring>
#include <exception>
#include <new>
#include <string>

struct welvet_b200_gdense {
  wb::GroupDense* g;
};

namespace {

welvet_status to_c(const wb::Status& st) {
  welvet_status out;
  out.code = static_cast<int32_t>(st.code);
  out.message[0] = '\0';
  if (!st.message.empty()) {
    std::strncpy(out.message, st.message.c_str(), sizeof(out.message) - 1);
    out.message[sizeof(out.message) - 1] = '\0';
  }
  return out;
}

template <typename F>
welvet_status guarded(F&& f) {
  try {
    return to_c(f());
  } catch (const std::bad_alloc&) {
    return to_c(wb::Status::Internal("host allocation failed"));
  } catch (const std::exception& e) {
    return to_c(wb::Status::Internal(e.what()));
  } catch (...) {
    return to_c(wb::Status::Internal("unknown exception"));
  }
}

wb::Status init_device(int* dev) {
  WB_TRY(wb::library_device(dev));
  WB_CUDA(cudaSetDevice(*dev));
  return wb::Status::Ok();
}

constexpr int kMaxHeadDim = 256;

wb::Status pool_of(const char* name, const void* pages, const int64_t* strides, const welvet_b200_kv_desc& d, int size,
                   wb::KvPool* out) {
  if (!pages) return wb::Status::Invalid(std::string("kv: nil ") + name);
  if (reinterpret_cast<uintptr_t>(pages) % size != 0)
    return wb::Status::Invalid(std::string("kv: ") + name + " not aligned to its type");
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0) return wb::Status::Invalid(std::string("kv: negative stride of ") + name);
  // rows of head_dim elements must not run into one another
  if ((d.page_size > 1 && strides[1] < d.head_dim) || (d.num_kv_heads > 1 && strides[2] < d.head_dim) ||
      (d.num_pages > 1 && strides[0] < d.head_dim))
    return wb::Status::Invalid(std::string("kv: rows of ") + name + " overlap");
  out->base = static_cast<uint8_t*>(const_cast<void*>(pages));
  out->page = strides[0];
  out->slot = strides[1];
  out->head = strides[2];
  return wb::Status::Ok();
}

} // namespace

extern "C" {

welvet_status welvet_b200_kv_create(const welvet_b200_kv_desc* desc, welvet_b200_kv** out) {
  return guarded([&] {
    if (!desc || !out) return wb::Status::Invalid("kv: invalid argument");
    const welvet_b200_kv_desc& d = *desc;
    if (d.dtype < 1 || d.dtype > 4)
      return wb::Status::Unsupported("kv: page dtype id " + std::to_string(d.dtype) + " (Float32, Float16, BFloat16 or FP8E4M3)");
    if (d.num_heads <= 0 || d.num_kv_heads <= 0 || d.num_heads % d.num_kv_heads != 0)
      return wb::Status::Invalid("kv: need num_heads > 0, a multiple of num_kv_heads > 0");
    if (d.head_dim <= 0) return wb::Status::Invalid("kv: need head_dim > 0");
    if (d.head_dim > kMaxHeadDim) return wb::Status::Unsupported("kv: head_dim > 256");
    if (d.page_size <= 0 || d.num_pages <= 0 || d.num_seqs <= 0 || d.pages_per_seq <= 0)
      return wb::Status::Invalid("kv: need page_size, num_pages, num_seqs and pages_per_seq > 0");
    if (static_cast<int64_t>(d.page_size) * d.pages_per_seq > (1ll << 30))
      return wb::Status::Unsupported("kv: more than 2^30 slots per sequence");
    if (d.num_seqs > 65535 || d.num_kv_heads > 65535 || d.num_heads > 65535)
      return wb::Status::Unsupported("kv: more than 65535 sequences or heads");
    if (d.table_stride < d.pages_per_seq && d.num_seqs > 1) return wb::Status::Invalid("kv: table_stride < pages_per_seq");
    if (!d.page_table || !d.lens) return wb::Status::Invalid("kv: nil page_table or lens");
    if (d.positions && !d.seen) return wb::Status::Invalid("kv: positions without seen");
    if (d.positions && d.seen == d.lens) return wb::Status::Invalid("kv: with positions seen must be an array of its own");
    if (!(d.k_scale > 0.0f) || !(d.v_scale > 0.0f) || !std::isnormal(d.k_scale) || !std::isnormal(d.v_scale))
      return wb::Status::Invalid("kv: k_scale and v_scale must be positive, finite and normal");
    wb::KvView v;
    const auto type = static_cast<wb::KvType>(d.dtype);
    WB_TRY(pool_of("k_pages", d.k_pages, d.k_strides, d, wb::kv_size(type), &v.k));
    WB_TRY(pool_of("v_pages", d.v_pages, d.v_strides, d, wb::kv_size(type), &v.v));
    v.k_scale = d.k_scale;
    v.v_scale = d.v_scale;
    v.num_heads = d.num_heads;
    v.num_kv = d.num_kv_heads;
    v.head_dim = d.head_dim;
    v.page_size = d.page_size;
    v.num_pages = d.num_pages;
    v.num_seqs = d.num_seqs;
    v.pages_per_seq = d.pages_per_seq;
    v.table_stride = d.table_stride;
    v.table = d.page_table;
    v.lens = d.lens;
    v.seen = d.seen ? d.seen : d.lens;
    v.weights = d.weights;
    v.positions = d.positions;
    v.max_slots = d.page_size * d.pages_per_seq;
    int dev = 0;
    WB_TRY(init_device(&dev));
    wb::KvCache* c = nullptr;
    WB_TRY(wb::kv_create(dev, type, v, &c));
    *out = new welvet_b200_kv{c};
    return wb::Status::Ok();
  });
}

welvet_status welvet_b200_kv_append(welvet_b200_kv* kv, int32_t rows, const float* k, int64_t k_ld, const float* v,
                                    int64_t v_ld, const float* q, int64_t q_ld, float* q_out, int64_t q_out_ld,
                                    const int32_t* cu_tokens, double theta, const int32_t* start, const int32_t* start_seen,
                                    void* stream) {
  return guarded([&] {
    if (!kv || !kv->c) return wb::Status::Invalid("kv: nil handle");
    const wb::KvView& w = kv->c->view;
    const int64_t kd = static_cast<int64_t>(w.num_kv) * w.head_dim, qd = static_cast<int64_t>(w.num_heads) * w.head_dim;
    if (rows < 0 || (rows > 0 && (!k || !v))) return wb::Status::Invalid("kv append: nil k or v, or rows < 0");
    if (!cu_tokens && rows != w.num_seqs) return wb::Status::Invalid("kv append: without cu_tokens rows must equal num_seqs");
    if ((q == nullptr) != (q_out == nullptr)) return wb::Status::Invalid("kv append: q and q_out go together");
    if (rows > 1 && (k_ld < kd || v_ld < kd || (q && (q_ld < qd || q_out_ld < qd))))
      return wb::Status::Invalid("kv append: a row stride is shorter than a row");
    if (!std::isfinite(theta)) return wb::Status::Invalid("kv append: theta is not finite");
    if (start_seen && w.seen == w.lens)
      return wb::Status::Invalid("kv append: start_seen without a seen array in the cache");
    wb::KvAppendArgs a;
    a.rows = rows;
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.k_ld = k_ld;
    a.v_ld = v_ld;
    a.q_ld = q_ld;
    a.q_out_ld = q_out_ld;
    a.cu = cu_tokens;
    a.theta = theta;
    a.start = start;
    a.start_seen = start_seen;
    return wb::kv_append(kv->c, a, static_cast<cudaStream_t>(stream));
  });
}

welvet_status welvet_b200_kv_attend(welvet_b200_kv* kv, const float* q, int64_t q_ld, float* out, int64_t out_ld, float scale,
                                    int32_t window, int32_t alibi, int32_t accumulate, const float* weights_in, void* stream) {
  return guarded([&] {
    if (!kv || !kv->c) return wb::Status::Invalid("kv: nil handle");
    const wb::KvView& w = kv->c->view;
    const int64_t qd = static_cast<int64_t>(w.num_heads) * w.head_dim;
    if (!q || !out) return wb::Status::Invalid("kv attend: nil q or out");
    if (w.num_seqs > 1 && (q_ld < qd || out_ld < qd)) return wb::Status::Invalid("kv attend: a row stride is shorter than a row");
    if (!std::isfinite(scale)) return wb::Status::Invalid("kv attend: scale is not finite");
    if (window < 0) return wb::Status::Invalid("kv attend: window < 0");
    if ((accumulate || weights_in) && !w.weights) return wb::Status::Invalid("kv attend: the cache has no weights to accumulate");
    wb::KvAttendArgs a;
    a.q = q;
    a.out = out;
    a.q_ld = q_ld;
    a.out_ld = out_ld;
    a.scale = scale;
    a.window = window;
    a.alibi = alibi != 0;
    a.accumulate = accumulate != 0;
    a.weights_in = weights_in;
    return wb::kv_attend(kv->c, a, static_cast<cudaStream_t>(stream));
  });
}

welvet_status welvet_b200_kv_evict(welvet_b200_kv* kv, int32_t keep, int32_t budget, int32_t sinks, int32_t recent,
                                   const int32_t* lens_in, const float* weights_in, const int32_t* positions_in,
                                   void* stream) {
  return guarded([&] {
    if (!kv || !kv->c) return wb::Status::Invalid("kv: nil handle");
    const wb::KvView& w = kv->c->view;
    if (!w.weights || !w.positions) return wb::Status::Invalid("kv evict: the cache has no weights and positions");
    if (keep <= 0 || sinks < 0 || recent < 0) return wb::Status::Invalid("kv evict: need keep > 0, sinks >= 0, recent >= 0");
    if (static_cast<int64_t>(sinks) + recent > keep) return wb::Status::Invalid("kv evict: sinks + recent > keep");
    if (budget < keep) return wb::Status::Invalid("kv evict: budget < keep");
    wb::KvEvictArgs a;
    a.keep = keep;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.lens_in = lens_in;
    a.weights_in = weights_in;
    a.positions_in = positions_in;
    return wb::kv_evict(kv->c, a, static_cast<cudaStream_t>(stream));
  });
}

welvet_status welvet_b200_kv_check_error(welvet_b200_kv* kv, void* stream) {
  return guarded([&] {
    if (!kv || !kv->c) return wb::Status::Invalid("kv: nil handle");
    return wb::kv_check_error(kv->c, static_cast<cudaStream_t>(stream));
  });
}

void welvet_b200_kv_release(welvet_b200_kv* kv) {
  if (!kv) return;
  delete kv->c;
  delete kv;
}

// ------------------------------------------------------------------------- group dense

static wb::Status group_shape(int32_t in, int32_t out, int32_t group, int32_t code, int32_t scale_dtype) {
  if (in <= 0 || out <= 0) return wb::Status::Invalid("group dense: need in > 0 and out > 0");
  if (in > (1 << 30) || out > (1 << 30)) return wb::Status::Unsupported("group dense: more than 2^30 inputs or outputs");
  if (code != wb::kCodeInt4 && code != wb::kCodeUint4 && code != wb::kCodeFp4)
    return wb::Status::Unsupported("group dense: code dtype id " + std::to_string(code) + " (Int4, Uint4 or FP4)");
  if (scale_dtype != wb::kScaleF16 && scale_dtype != wb::kScaleBF16)
    return wb::Status::Unsupported("group dense: scale dtype id " + std::to_string(scale_dtype) + " (Float16 or BFloat16)");
  if (group != 32 && (group <= 0 || group % 64 != 0))
    return wb::Status::Unsupported("group dense: group must be 32 or a multiple of 64");
  if (group > (1 << 20)) return wb::Status::Unsupported("group dense: group > 2^20");
  return wb::Status::Ok();
}

welvet_status welvet_b200_group_quantize(int32_t in, int32_t out, int32_t group, int32_t code, int32_t scale_dtype,
                                         const float* W_dev, uint8_t* codes_dev, void* scales_dev, uint8_t* zeros_dev,
                                         void* stream) {
  return guarded([&] {
    WB_TRY(group_shape(in, out, group, code, scale_dtype));
    if (!W_dev || !codes_dev || !scales_dev || (code == wb::kCodeUint4 && !zeros_dev))
      return wb::Status::Invalid("group quantize: nil argument");
    int dev = 0;
    WB_TRY(init_device(&dev));
    return wb::group_quantize(out, in, group, code, scale_dtype, W_dev, codes_dev, scales_dev, zeros_dev,
                              static_cast<cudaStream_t>(stream));
  });
}

welvet_status welvet_b200_gdense_mount(int32_t in, int32_t out, int32_t group, int32_t code, int32_t scale_dtype, int32_t act,
                                       const uint8_t* codes, const void* scales, const uint8_t* zeros,
                                       int32_t weights_on_device, const double* bias, size_t bias_len,
                                       welvet_b200_gdense** g_out) {
  return guarded([&] {
    if (!g_out || !codes || !scales) return wb::Status::Invalid("group dense: nil argument");
    WB_TRY(group_shape(in, out, group, code, scale_dtype));
    if (code == wb::kCodeUint4 && !zeros) return wb::Status::Invalid("group dense: Uint4 codes need zero points");
    if (code != wb::kCodeUint4 && zeros) return wb::Status::Invalid("group dense: zero points go with Uint4 codes only");
    if (!wb::activation_valid(act)) return wb::Status::Invalid("group dense: unknown activation");
    if (bias_len > 0 && !bias) return wb::Status::Invalid("group dense: nil bias");
    int dev = 0;
    WB_TRY(init_device(&dev));
    wb::GroupDenseSrc src;
    src.codes = codes;
    src.scales = scales;
    src.zeros = zeros;
    src.on_device = weights_on_device != 0;
    src.bias = bias;
    src.bias_len = bias_len;
    wb::GroupDense* g = nullptr;
    WB_TRY(wb::gdense_mount(dev, out, in, group, code, scale_dtype, act, src, &g));
    *g_out = new welvet_b200_gdense{g};
    return wb::Status::Ok();
  });
}

welvet_status welvet_b200_gdense_execute_device(welvet_b200_gdense* g, int32_t rows, const float* x_dev, int64_t x_ld,
                                                float* pre_dev, float* post_dev, void* stream) {
  return guarded([&] {
    if (!g || !g->g) return wb::Status::Invalid("group dense: nil handle");
    if (rows < 0) return wb::Status::Invalid("group dense: rows < 0");
    if (rows == 0) return wb::Status::Ok();
    if (!x_dev || !post_dev) return wb::Status::Invalid("group dense: nil x or post");
    if (rows > 1 && x_ld < g->g->cols) return wb::Status::Invalid("group dense: x_ld is shorter than a row");
    return wb::gdense_forward(g->g, rows, x_dev, x_ld, pre_dev, post_dev, static_cast<cudaStream_t>(stream));
  });
}

int32_t welvet_b200_gdense_plan(int32_t in, int32_t out, int32_t group, int32_t code, int32_t sms, int32_t rows,
                                int64_t* values, int32_t n) {
  int32_t count = -1;
  const welvet_status st = guarded([&] {
    WB_TRY(group_shape(in, out, group, code, wb::kScaleF16));
    if (sms <= 0 || rows < 1 || rows > 8 || (n > 0 && !values)) return wb::Status::Invalid("group dense: plan");
    count = wb::gdense_plan_values(out, in, group, code, sms, rows, values, n < 0 ? 0 : n);
    return wb::Status::Ok();
  });
  return st.code == 0 ? count : -1;
}

void welvet_b200_gdense_release(welvet_b200_gdense* g) {
  if (!g) return;
  delete g->g;
  delete g;
}

} // extern "C"
