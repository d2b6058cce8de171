// origami_torch_ext.cpp -- PyTorch-ROCm extension module over the C ABI of
// liborigami_layout.so (include/origami_layout.h).
//
// It exports the function names of the reference's extension module
// origami_bitpack_cuda_v6 (csrc/origami/bitpack_layout_cuda.cpp:894-903) with
// their argument lists, plus the fused paths this library adds.  Tensors are
// checked and unwrapped here; the work is done by the extern "C" entry points
// on the calling thread's current HIP stream of the tensors' device, and a
// non-zero status becomes a RuntimeError carrying origami_last_error(), the
// way the reference's TORCH_CHECKs raise.  There is no device code here.
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "origami_layout.h"

namespace {

void check(int rc) {
  TORCH_CHECK(rc == ORIGAMI_OK, origami_last_error());
}

// ORIGAMI_ERR_UNSUPPORTED is returned to Python as False (the caller takes
// the two-step path); every other failure raises.
bool check_supported(int rc) {
  if (rc == ORIGAMI_ERR_UNSUPPORTED) return false;
  check(rc);
  return true;
}

origami_stream_t current_stream(const at::Tensor& t) {
  return reinterpret_cast<origami_stream_t>(
      c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void require_device(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void require_byte(const at::Tensor& t, const char* name) {
  require_device(t, name);
  TORCH_CHECK(t.scalar_type() == at::kByte, name, " must be uint8");
}

// Host int64 copy of a metadata tensor (no copy when it already is one).
// Device metadata costs one device-to-host copy, as in the reference
// (bitpack_layout_cuda.cpp:156, 350-351).
at::Tensor host_i64(const at::Tensor& t) {
  at::Tensor h = t;
  if (h.device().type() != at::kCPU || h.scalar_type() != at::kLong)
    h = h.to(at::kCPU, at::kLong);
  return h.contiguous();
}

const int64_t* i64p(const at::Tensor& t) { return t.data_ptr<int64_t>(); }

// Paged cache geometry of the layout entry points: [2, NB, bs, H, D] is
// recognised first, then [NB, 2, bs, H, D] (benchmark_utils.py:357,
// bitpack_layout_cuda.cpp:810-831).
struct CacheGeom {
  int64_t layout, num_blocks, block_size, heads, head_bytes;
};

CacheGeom layout_cache_geometry(const at::Tensor& c) {
  TORCH_CHECK(c.dim() == 5, "kv_cache must have rank 5");
  CacheGeom g{};
  if (c.size(0) == 2) {
    g.layout = ORIGAMI_CACHE_KV_FIRST;
    g.num_blocks = c.size(1);
  } else if (c.size(1) == 2) {
    g.layout = ORIGAMI_CACHE_BLOCKS_FIRST;
    g.num_blocks = c.size(0);
  } else {
    TORCH_CHECK(false, "kv_cache must be [num_blocks,2,block,heads,dim] or "
                       "[2,num_blocks,block,heads,dim]");
  }
  g.block_size = c.size(2);
  g.heads = c.size(3);
  g.head_bytes = c.size(4) * static_cast<int64_t>(c.element_size());
  return g;
}

// The dequantize entry points follow bitpack_layout_cuda.cpp:526-552, which
// recognises [NB, 2, bs, H, D] first.
CacheGeom dequant_cache_geometry(const at::Tensor& c, int64_t heads, int64_t head_dim) {
  TORCH_CHECK(c.dim() == 5, "kv_cache must have rank 5");
  CacheGeom g{};
  if (c.size(1) == 2) {
    g.layout = ORIGAMI_CACHE_BLOCKS_FIRST;
    g.num_blocks = c.size(0);
  } else if (c.size(0) == 2) {
    g.layout = ORIGAMI_CACHE_KV_FIRST;
    g.num_blocks = c.size(1);
  } else {
    TORCH_CHECK(false, "kv_cache must be [num_blocks,2,block,heads,dim] or "
                       "[2,num_blocks,block,heads,dim]");
  }
  TORCH_CHECK(c.size(3) == heads && c.size(4) == head_dim, "kv_cache head shape mismatch");
  g.block_size = c.size(2);
  return g;
}

int64_t dtype_code(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kHalf:
      return ORIGAMI_DTYPE_FLOAT16;
    case at::kBFloat16:
      return ORIGAMI_DTYPE_BFLOAT16;
    case at::kFloat:
      return ORIGAMI_DTYPE_FLOAT32;
    default:
      TORCH_CHECK(false, name, " has an unsupported dtype");
  }
  return 0;
}

void require_block_ids(const at::Tensor& ids, const at::Tensor& cache) {
  require_device(ids, "block_ids");
  TORCH_CHECK(ids.scalar_type() == at::kLong, "block_ids must be int64");
  TORCH_CHECK(ids.device() == cache.device(), "block_ids must be on the kv_cache device");
}

// ---------------------------------------------------------------------------
// Reference names (bitpack_layout_cuda.cpp:894-903)
// ---------------------------------------------------------------------------

// bitpack_layout_cuda.cpp:316-400: flat chunks -> new uint8 symbol tensor.
at::Tensor unpack_canonical_storage_chunks_cuda(at::Tensor flat_chunks, at::Tensor chunk_offsets,
                                                at::Tensor bits_per_chunk, at::Tensor source_shape,
                                                at::Tensor axis_positions, int64_t token_count,
                                                int64_t num_heads, int64_t head_dim,
                                                at::Tensor chunk_specs) {
  require_byte(flat_chunks, "flat_chunks");
  const at::Tensor offs = host_i64(chunk_offsets), bits = host_i64(bits_per_chunk);
  const at::Tensor specs = host_i64(chunk_specs), shape = host_i64(source_shape);
  const at::Tensor axes = host_i64(axis_positions);
  TORCH_CHECK(axes.numel() == 4,
              "axis_positions must be [token_axis, head_axis, head_dim_axis, layer_axis]");
  const int64_t n = bits.numel();
  TORCH_CHECK(offs.numel() == n + 1, "chunk_offsets length must be chunk count + 1");
  TORCH_CHECK(specs.numel() == 6 * n, "chunk_specs must be [num_chunks, 6]");
  int64_t total = 1;
  for (int64_t a = 0; a < shape.numel(); ++a) total *= std::max<int64_t>(i64p(shape)[a], 0);
  const c10::OptionalDeviceGuard guard(flat_chunks.device());
  at::Tensor out = at::empty({total}, flat_chunks.options());
  check(origami_unpack_canonical_storage_chunks(
      flat_chunks.data_ptr<uint8_t>(), flat_chunks.numel(), i64p(offs), i64p(bits), i64p(specs),
      n, i64p(shape), shape.numel(), i64p(axes), token_count, num_heads, head_dim,
      out.data_ptr<uint8_t>(), out.numel(), current_stream(flat_chunks)));
  return out;
}

// bitpack_layout_cuda.cpp:402-473: CacheGen layers -> float16 [L, 2, H, T, D].
at::Tensor cachegen_unpack_dequantize_cuda(at::Tensor bytestream, at::Tensor offsets,
                                           at::Tensor bits_per_layer, at::Tensor key_bins,
                                           at::Tensor value_bins, at::Tensor max_key,
                                           at::Tensor max_value, int64_t tokens, int64_t heads,
                                           int64_t head_dim) {
  at::Tensor flat = bytestream.reshape(-1).contiguous();
  require_byte(flat, "bytestream");
  const at::Tensor offs = host_i64(offsets), bits = host_i64(bits_per_layer);
  const at::Tensor kb = host_i64(key_bins), vb = host_i64(value_bins);
  TORCH_CHECK(bits.numel() % 2 == 0, "bits_per_layer length must be even");
  const int64_t layers = bits.numel() / 2;
  TORCH_CHECK(kb.numel() == layers, "key_bins length must match layers");
  TORCH_CHECK(vb.numel() == layers, "value_bins length must match layers");
  TORCH_CHECK(offs.numel() == bits.numel() + 1,
              "offsets length must be bits_per_layer length + 1");
  const at::Tensor mk = max_key.contiguous(), mv = max_value.contiguous();
  require_device(mk, "max_key");
  require_device(mv, "max_value");
  TORCH_CHECK(mk.scalar_type() == mv.scalar_type(),
              "max_key and max_value must have the same dtype");
  const c10::OptionalDeviceGuard guard(flat.device());
  at::Tensor out = at::empty({layers, 2, heads, tokens, head_dim},
                             flat.options().dtype(at::kHalf));
  check(origami_cachegen_unpack_dequantize(
      flat.data_ptr<uint8_t>(), flat.numel(), i64p(offs), i64p(bits), i64p(kb), i64p(vb), layers,
      mk.data_ptr(), mv.data_ptr(), mk.numel(), mv.numel(), dtype_code(mk.scalar_type(), "max_key"),
      tokens, heads, head_dim, out.data_ptr(), out.numel() * 2, current_stream(flat)));
  return out;
}

// bitpack_layout_cuda.cpp:475-581: CacheGen K/V streams -> paged cache.
void cachegen_unpack_dequantize_to_kv_cache_cuda(
    at::Tensor bytestream, int64_t key_offset, int64_t key_bytes, int64_t value_offset,
    int64_t value_bytes, int64_t key_bits, int64_t value_bits, int64_t key_bins,
    int64_t value_bins, at::Tensor max_key, at::Tensor max_value, at::Tensor kv_cache,
    at::Tensor block_ids, int64_t tokens, int64_t heads, int64_t head_dim) {
  at::Tensor flat = bytestream.reshape(-1).contiguous();
  require_byte(flat, "bytestream");
  require_device(kv_cache, "kv_cache");
  require_block_ids(block_ids, kv_cache);
  const at::Tensor mk = max_key.contiguous(), mv = max_value.contiguous();
  require_device(mk, "max_key");
  require_device(mv, "max_value");
  TORCH_CHECK(mk.scalar_type() == mv.scalar_type(),
              "max_key and max_value must have the same dtype");
  const CacheGeom g = dequant_cache_geometry(kv_cache, heads, head_dim);
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  check(origami_cachegen_unpack_dequantize_to_kv_cache(
      flat.data_ptr<uint8_t>(), flat.numel(), key_offset, key_bytes, value_offset, value_bytes,
      key_bits, value_bits, key_bins, value_bins, mk.data_ptr(), mv.data_ptr(), mk.numel(),
      mv.numel(), dtype_code(mk.scalar_type(), "max_key"), kv_cache.data_ptr(),
      dtype_code(kv_cache.scalar_type(), "kv_cache"), g.layout, g.num_blocks, g.block_size,
      block_ids.data_ptr<int64_t>(), block_ids.numel(), tokens, heads, head_dim,
      current_stream(kv_cache)));
}

void kivi_to_kv_cache(at::Tensor bytestream, int64_t key_offset, int64_t key_bytes,
                      int64_t value_offset, int64_t value_bytes, int64_t bits,
                      int64_t symbol_packing, int64_t group_size, int64_t sink_tokens,
                      at::Tensor key_scale, at::Tensor key_zero, at::Tensor value_scale,
                      at::Tensor value_zero, at::Tensor key_sink, at::Tensor value_sink,
                      at::Tensor kv_cache, at::Tensor block_ids, int64_t tokens, int64_t heads,
                      int64_t head_dim) {
  at::Tensor flat = bytestream.reshape(-1).contiguous();
  require_byte(flat, "bytestream");
  require_device(kv_cache, "kv_cache");
  require_block_ids(block_ids, kv_cache);
  const at::Tensor metas[6] = {key_scale.contiguous(), key_zero.contiguous(),
                               value_scale.contiguous(), value_zero.contiguous(),
                               key_sink.contiguous(), value_sink.contiguous()};
  const char* names[6] = {"key_scale", "key_zero", "value_scale", "value_zero", "key_sink",
                          "value_sink"};
  int64_t counts[6];
  for (int i = 0; i < 6; ++i) {
    require_device(metas[i], names[i]);
    TORCH_CHECK(metas[i].scalar_type() == metas[0].scalar_type(),
                "KIVI metadata tensors must have the same dtype");
    counts[i] = metas[i].numel();
  }
  const CacheGeom g = dequant_cache_geometry(kv_cache, heads, head_dim);
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  check(origami_kivi_dequantize_to_kv_cache(
      flat.data_ptr<uint8_t>(), flat.numel(), key_offset, key_bytes, value_offset, value_bytes,
      bits, symbol_packing, group_size, sink_tokens, metas[0].data_ptr(), metas[1].data_ptr(),
      metas[2].data_ptr(), metas[3].data_ptr(), metas[4].data_ptr(), metas[5].data_ptr(), counts,
      dtype_code(metas[0].scalar_type(), "KIVI metadata"), kv_cache.data_ptr(),
      dtype_code(kv_cache.scalar_type(), "kv_cache"), g.layout, g.num_blocks, g.block_size,
      block_ids.data_ptr<int64_t>(), block_ids.numel(), tokens, heads, head_dim,
      current_stream(kv_cache)));
}

// bitpack_layout_cuda.cpp:583-714: LSB-first symbols, as the reference kernel reads.
void kivi_dequantize_to_kv_cache_cuda(at::Tensor bytestream, int64_t key_offset,
                                      int64_t key_bytes, int64_t value_offset,
                                      int64_t value_bytes, int64_t bits, int64_t group_size,
                                      int64_t sink_tokens, at::Tensor key_scale,
                                      at::Tensor key_zero, at::Tensor value_scale,
                                      at::Tensor value_zero, at::Tensor key_sink,
                                      at::Tensor value_sink, at::Tensor kv_cache,
                                      at::Tensor block_ids, int64_t tokens, int64_t heads,
                                      int64_t head_dim) {
  kivi_to_kv_cache(bytestream, key_offset, key_bytes, value_offset, value_bytes, bits,
                   ORIGAMI_KIVI_PACKED_LSB, group_size, sink_tokens, key_scale, key_zero,
                   value_scale, value_zero, key_sink, value_sink, kv_cache, block_ids, tokens,
                   heads, head_dim);
}

void fused_prefix_attention_cuda(py::args, py::kwargs) {
  TORCH_CHECK(false, "fused prefix attention is outside the layout path");
}

// ---------------------------------------------------------------------------
// Fused paths (no reference counterpart under these names); chunk metadata
// as host int64 tensors.
// ---------------------------------------------------------------------------

// Packs a symbol tensor into `out` (the stub native_cpu.pack_canonical_storage_chunks).
void pack_canonical_storage_chunks(at::Tensor symbols, at::Tensor chunk_offsets,
                                   at::Tensor bits_per_chunk, at::Tensor chunk_specs,
                                   at::Tensor source_shape, at::Tensor axis_positions,
                                   int64_t token_count, int64_t num_heads, int64_t head_dim,
                                   at::Tensor out) {
  require_byte(symbols, "symbols");
  require_byte(out, "flat_chunks");
  const at::Tensor offs = host_i64(chunk_offsets), bits = host_i64(bits_per_chunk);
  const at::Tensor specs = host_i64(chunk_specs), shape = host_i64(source_shape);
  const at::Tensor axes = host_i64(axis_positions);
  TORCH_CHECK(offs.numel() == bits.numel() + 1, "chunk_offsets length must be chunk count + 1");
  const c10::OptionalDeviceGuard guard(symbols.device());
  check(origami_pack_canonical_storage_chunks(
      symbols.data_ptr<uint8_t>(), symbols.numel(), i64p(offs), i64p(bits), i64p(specs),
      bits.numel(), i64p(shape), shape.numel(), i64p(axes), token_count, num_heads, head_dim,
      out.data_ptr<uint8_t>(), out.numel(), current_stream(symbols)));
}

// One layer's stream -> paged cache through the block table.  Returns False
// when the chunk plan is not served by the fused kernel.
bool unpack_canonical_to_kv_cache(at::Tensor flat, at::Tensor chunk_offsets,
                                  at::Tensor bits_per_chunk, at::Tensor chunk_specs,
                                  int64_t tokens, at::Tensor kv_cache, at::Tensor block_ids) {
  require_byte(flat, "flat_chunks");
  require_device(kv_cache, "kv_cache");
  require_block_ids(block_ids, kv_cache);
  const CacheGeom g = layout_cache_geometry(kv_cache);
  const at::Tensor offs = host_i64(chunk_offsets), bits = host_i64(bits_per_chunk);
  const at::Tensor specs = host_i64(chunk_specs);
  TORCH_CHECK(offs.numel() == bits.numel() + 1, "chunk_offsets length must be chunk count + 1");
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  return check_supported(origami_unpack_canonical_to_kv_cache(
      flat.data_ptr<uint8_t>(), flat.numel(), i64p(offs), i64p(bits), i64p(specs), bits.numel(),
      tokens, kv_cache.data_ptr(), g.layout, g.num_blocks, g.block_size, g.heads, g.head_bytes,
      block_ids.data_ptr<int64_t>(), block_ids.numel(), current_stream(kv_cache)));
}

// Paged cache -> one layer's stream (`out`).  Returns False when the chunk
// plan is not served by the fused kernel.
bool pack_canonical_from_kv_cache(at::Tensor kv_cache, at::Tensor block_ids, int64_t tokens,
                                  at::Tensor chunk_offsets, at::Tensor bits_per_chunk,
                                  at::Tensor chunk_specs, at::Tensor out) {
  require_device(kv_cache, "kv_cache");
  require_block_ids(block_ids, kv_cache);
  require_byte(out, "flat_chunks");
  const CacheGeom g = layout_cache_geometry(kv_cache);
  const at::Tensor offs = host_i64(chunk_offsets), bits = host_i64(bits_per_chunk);
  const at::Tensor specs = host_i64(chunk_specs);
  TORCH_CHECK(offs.numel() == bits.numel() + 1, "chunk_offsets length must be chunk count + 1");
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  return check_supported(origami_pack_canonical_from_kv_cache(
      kv_cache.data_ptr(), g.layout, g.num_blocks, g.block_size, g.heads, g.head_bytes,
      block_ids.data_ptr<int64_t>(), block_ids.numel(), tokens, i64p(offs), i64p(bits),
      i64p(specs), bits.numel(), out.data_ptr<uint8_t>(), out.numel(),
      current_stream(kv_cache)));
}

// One layer of several requests into one cache.  Returns False when a plan
// is not served by the fused kernel.
bool unpack_canonical_to_kv_cache_batch(std::vector<at::Tensor> flats,
                                        std::vector<at::Tensor> chunk_offsets,
                                        std::vector<at::Tensor> bits_per_chunk,
                                        std::vector<at::Tensor> chunk_specs,
                                        std::vector<int64_t> tokens, at::Tensor kv_cache,
                                        std::vector<at::Tensor> block_ids,
                                        std::vector<int64_t> first_tokens) {
  const size_t n = flats.size();
  TORCH_CHECK(chunk_offsets.size() == n && bits_per_chunk.size() == n &&
                  chunk_specs.size() == n && tokens.size() == n && block_ids.size() == n &&
                  (first_tokens.empty() || first_tokens.size() == n),
              "one entry per request is required");
  require_device(kv_cache, "kv_cache");
  const CacheGeom g = layout_cache_geometry(kv_cache);
  std::vector<at::Tensor> offs(n), bits(n), specs(n);
  std::vector<const uint8_t*> fp(n);
  std::vector<const int64_t*> op(n), bp(n), sp(n), ip(n);
  std::vector<int64_t> fb(n), nc(n), bc(n);
  for (size_t r = 0; r < n; ++r) {
    require_byte(flats[r], "flat_chunks");
    require_block_ids(block_ids[r], kv_cache);
    offs[r] = host_i64(chunk_offsets[r]);
    bits[r] = host_i64(bits_per_chunk[r]);
    specs[r] = host_i64(chunk_specs[r]);
    TORCH_CHECK(offs[r].numel() == bits[r].numel() + 1,
                "chunk_offsets length must be chunk count + 1");
    fp[r] = flats[r].data_ptr<uint8_t>();
    fb[r] = flats[r].numel();
    op[r] = i64p(offs[r]);
    bp[r] = i64p(bits[r]);
    sp[r] = i64p(specs[r]);
    nc[r] = bits[r].numel();
    ip[r] = block_ids[r].data_ptr<int64_t>();
    bc[r] = block_ids[r].numel();
  }
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  return check_supported(origami_unpack_canonical_to_kv_cache_batch(
      static_cast<int64_t>(n), fp.data(), fb.data(), op.data(), bp.data(), sp.data(), nc.data(),
      tokens.data(), kv_cache.data_ptr(), g.layout, g.num_blocks, g.block_size, g.heads,
      g.head_bytes, ip.data(), bc.data(), first_tokens.empty() ? nullptr : first_tokens.data(),
      current_stream(kv_cache)));
}

// A prepared restore (origami_restore_plan_create) with the cache geometry it
// was made for and its device block table, which it keeps alive.
struct PreparedRestore {
  origami_restore_plan_t plan = nullptr;
  std::vector<int64_t> sizes;
  at::ScalarType dtype;
  at::Device device;
  at::Tensor block_ids;
  ~PreparedRestore() { origami_restore_plan_destroy(plan); }
};

// Returns a handle (an integer), or 0 when the chunk plan is not served by the
// fused kernel.
int64_t restore_plan_create(at::Tensor chunk_offsets, at::Tensor bits_per_chunk,
                            at::Tensor chunk_specs, int64_t tokens, at::Tensor kv_cache,
                            at::Tensor block_ids) {
  require_device(kv_cache, "kv_cache");
  require_block_ids(block_ids, kv_cache);
  const CacheGeom g = layout_cache_geometry(kv_cache);
  const at::Tensor offs = host_i64(chunk_offsets), bits = host_i64(bits_per_chunk);
  const at::Tensor specs = host_i64(chunk_specs);
  TORCH_CHECK(offs.numel() == bits.numel() + 1, "chunk_offsets length must be chunk count + 1");
  const c10::OptionalDeviceGuard guard(kv_cache.device());
  origami_restore_plan_t plan = nullptr;
  if (!check_supported(origami_restore_plan_create(
          i64p(offs), i64p(bits), i64p(specs), bits.numel(), tokens, g.layout, g.num_blocks,
          g.block_size, g.heads, g.head_bytes, block_ids.data_ptr<int64_t>(), block_ids.numel(),
          &plan)))
    return 0;
  auto* r = new PreparedRestore{plan, kv_cache.sizes().vec(), kv_cache.scalar_type(),
                                kv_cache.device(), block_ids};
  return reinterpret_cast<int64_t>(r);
}

// One layer: `flat` (this layer's stream) into `kv_cache` (a cache of the
// geometry the plan was made for), on the current stream.
void restore_plan_launch(int64_t handle, const at::Tensor& flat, const at::Tensor& kv_cache) {
  TORCH_CHECK(handle != 0, "restore plan is closed");
  const auto* r = reinterpret_cast<const PreparedRestore*>(handle);
  TORCH_CHECK(kv_cache.device() == r->device && kv_cache.scalar_type() == r->dtype &&
                  kv_cache.sizes().equals(r->sizes) && kv_cache.is_contiguous(),
              "kv_cache geometry differs from the prepared restore");
  TORCH_CHECK(flat.device() == r->device && flat.scalar_type() == at::kByte &&
                  flat.is_contiguous(),
              "flat_chunks must be a contiguous uint8 tensor on the cache's device");
  const c10::OptionalDeviceGuard guard(r->device);
  check(origami_restore_plan_launch(r->plan, flat.data_ptr<uint8_t>(), flat.numel(),
                                    kv_cache.data_ptr(), current_stream(kv_cache)));
}

void restore_plan_destroy(int64_t handle) {
  delete reinterpret_cast<PreparedRestore*>(handle);
}

// ---------------------------------------------------------------------------
// Operators on the paged cache that follow a restore.  The cache order is that of
// the layout entry points ([2, NB, bs, H, D] is recognised first).
// ---------------------------------------------------------------------------

int64_t paged_dtype_code(at::ScalarType t, const char* name) {
  if (t == at::kFloat8_e4m3fn) return ORIGAMI_DTYPE_FLOAT8_E4M3FN;
  TORCH_CHECK(t == at::kHalf || t == at::kBFloat16, name,
              " must be float16 or bfloat16 (a kv_cache may be float8_e4m3fn)");
  return dtype_code(t, name);
}

// No record is kept of operations: it would leave a launch on addresses out, and play back what
// this call gave.
void require_eager() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  bool recorded = torch::jit::tracer::isTracing();
  if (TorchDispatchModeTLS::any_modes_set())
    for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY,
                            TorchDispatchModeKey::FUNCTIONAL})
      recorded |= TorchDispatchModeTLS::get_mode(mode).has_value();
  TORCH_CHECK(!recorded, "this operator cannot be traced");
}

// A tensor whose memory holds its values, and of which no gradient or tangent is asked.
void require_plain(const at::Tensor& t, const char* name) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet kOdd(
      {DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
       DispatchKey::Batched, DispatchKey::Functionalize, DispatchKey::ZeroTensor,
       DispatchKey::Conjugate, DispatchKey::Negative});
  TORCH_CHECK(t.layout() == at::kStrided && !t.key_set().has_any(kOdd), name,
              " must be a plain tensor, not a wrapped, transformed or lazily negated one");
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires a gradient, which this operator does not have");
  TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
                t._fw_grad(0).defined()),
              name, " requires a gradient (it has a tangent), which this operator does not have");
}

// The bytes of a strided tensor: runs at every sum of count[i] multiples of step[i].
struct Extent {
  const char* base = nullptr;
  int64_t run = 0;  // bytes; 0: no elements
  int dims = 0;
  int64_t count[8], step[8];
  bool repeated = false;  // several indices have one address
};

Extent extent_of(const at::Tensor& t) {
  Extent e;
  if (t.numel() == 0) return e;
  e.base = static_cast<const char*>(t.data_ptr());
  e.run = t.element_size();
  const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
  TORCH_CHECK(sizes.size() <= 8, "tensors of more than 8 dimensions are not compared");
  const int64_t cell = e.run;
  for (size_t d = sizes.size(); d-- > 0;) {
    const int64_t n = sizes[d], step = strides[d] * cell;
    if (n == 1) continue;
    if (step == 0) {
      e.repeated = true;
    } else if (step == e.run && e.dims == 0) {
      e.run *= n;
    } else {
      e.count[e.dims] = n;
      e.step[e.dims++] = step;
    }
  }
  return e;
}

// Multiples first .. last of a step.
struct Multiples {
  int64_t step, first, last;
};

// Whether a sum of one multiple of each of p[0 .. n - 1] is in [low, high].  With the largest steps
// first, few multiples of each leave the rest a chance.
bool some_sum_within(const Multiples* p, int n, int64_t low, int64_t high) {
  if (n == 0) return low <= 0 && high >= 0;
  int64_t least = 0, most = 0;  // what the others add
  for (int i = 1; i < n; ++i) {
    least += p[i].first * p[i].step;
    most += p[i].last * p[i].step;
  }
  const auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t first = std::max(p->first, -floor_div(most - low, p->step));
  const int64_t last = std::min(p->last, floor_div(high - least, p->step));
  if (n == 1) return first <= last;
  for (int64_t i = first; i <= last; ++i)
    if (some_sum_within(p + 1, n - 1, low - i * p->step, high - i * p->step)) return true;
  return false;
}

void largest_first(Multiples* p, int n) {
  std::sort(p, p + n, [](const Multiples& a, const Multiples& b) { return a.step > b.step; });
}

bool share_bytes(const Extent& a, const Extent& b) {
  if (a.run == 0 || b.run == 0) return false;
  Multiples p[16];
  int n = 0;
  int64_t a_end = a.run, b_end = b.run;
  for (int i = 0; i < a.dims; ++i) {
    a_end += (a.count[i] - 1) * a.step[i];
    p[n++] = {a.step[i], 1 - a.count[i], 0};
  }
  const int from_a = n;
  for (int i = 0; i < b.dims; ++i) {
    b_end += (b.count[i] - 1) * b.step[i];
    int at = 0;
    while (at < from_a && p[at].step != b.step[i]) ++at;
    if (at < from_a)
      p[at].last += b.count[i] - 1;
    else
      p[n++] = {b.step[i], 0, b.count[i] - 1};
  }
  const int64_t apart = b.base - a.base;
  if (apart >= a_end || -apart >= b_end) return false;
  // a run of b starts less than a.run after one of a, or less than b.run before it
  largest_first(p, n);
  return some_sum_within(p, n, -apart - (b.run - 1), -apart + a.run - 1);
}

// Whether two elements of a tensor share bytes.
bool shares_with_itself(const Extent& e) {
  if (e.run == 0) return false;
  if (e.repeated) return true;
  Multiples p[8];
  for (int i = 0; i < e.dims; ++i) p[i] = {e.step[i], 1 - e.count[i], e.count[i] - 1};
  largest_first(p, e.dims);
  for (int i = 0; i < e.dims; ++i) {  // pairs that differ in p[i] first
    p[i].first = 1;
    if (some_sum_within(p + i, e.dims - i, 1 - e.run, e.run - 1)) return true;
  }
  return false;
}

bool same_elements(const at::Tensor& a, const at::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// What a call writes may not be what it reads: launches have no order between their workgroups.
void require_apart(const Extent& result, const char* result_name, const Extent& input,
                   const char* name) {
  TORCH_CHECK(!share_bytes(result, input), result_name, " must not overlap ", name);
}

// A [tokens, heads, head_dim] tensor whose channels are contiguous.
void require_rows(const at::Tensor& t, const char* name, const at::Tensor& cache,
                  at::ScalarType dtype) {
  require_plain(t, name);
  TORCH_CHECK(t.is_cuda() && t.device() == cache.device(), name,
              " must be on the kv_cache device");
  TORCH_CHECK(t.dim() == 3, name, " must be [tokens, heads, head_dim]");
  TORCH_CHECK(t.scalar_type() == dtype, name, " must have the same dtype as the other rows");
  TORCH_CHECK(t.size(2) == cache.size(4), name, " head_dim differs from the kv_cache's");
  TORCH_CHECK(t.stride(2) == 1 || t.numel() == 0, name, " channels must be contiguous");
}

// A contiguous int64 tensor of at least `count` values; null when it has none.
const int64_t* require_index(const at::Tensor& t, const char* name, const at::Tensor& cache,
                             int64_t count) {
  require_plain(t, name);
  TORCH_CHECK(t.is_cuda() && t.device() == cache.device(), name,
              " must be on the kv_cache device");
  TORCH_CHECK(t.scalar_type() == at::kLong && t.dim() == 1 && t.is_contiguous(), name,
              " must be a contiguous int64 vector");
  TORCH_CHECK(t.numel() == count, name, " must have ", count, " values, not ", t.numel());
  return count > 0 ? t.data_ptr<int64_t>() : nullptr;
}

// New tokens into the cache; returns the rotated queries (an undefined tensor, None in
// Python, without queries).
c10::optional<at::Tensor> append_kv_cache(
    at::Tensor key, at::Tensor value, at::Tensor kv_cache, at::Tensor slots,
    c10::optional<at::Tensor> query, c10::optional<at::Tensor> positions,
    c10::optional<at::Tensor> cos_sin, bool interleaved, c10::optional<at::Tensor> query_norm,
    c10::optional<at::Tensor> key_norm, double eps, double k_scale, double v_scale,
    c10::optional<at::Tensor> query_out) {
  require_eager();
  require_plain(kv_cache, "kv_cache");
  require_device(kv_cache, "kv_cache");
  const CacheGeom g = layout_cache_geometry(kv_cache);
  const int64_t dtype = paged_dtype_code(key.scalar_type(), "key");
  TORCH_CHECK(dtype != ORIGAMI_DTYPE_FLOAT8_E4M3FN, "key must be float16 or bfloat16");
  require_rows(key, "key", kv_cache, key.scalar_type());
  require_rows(value, "value", kv_cache, key.scalar_type());
  const int64_t tokens = key.size(0), D = kv_cache.size(4);
  TORCH_CHECK(key.size(1) == g.heads && value.size(1) == g.heads,
              "key and value heads differ from the kv_cache's");
  TORCH_CHECK(value.size(0) == tokens, "key and value must have the same tokens");
  const int64_t* const slot = require_index(slots, "slots", kv_cache, tokens);
  int64_t strides[8] = {key.stride(0), key.stride(1), value.stride(0), value.stride(1), 0, 0, 0, 0};
  const c10::OptionalDeviceGuard guard(kv_cache.device());

  c10::optional<at::Tensor> out;
  Extent out_extent;  // of a new tensor: none
  int64_t query_heads = 0;
  if (query) {
    require_rows(*query, "query", kv_cache, key.scalar_type());
    TORCH_CHECK(query->size(0) == tokens, "query and key must have the same tokens");
    query_heads = query->size(1);
    if (query_out) {
      require_rows(*query_out, "query_out", kv_cache, key.scalar_type());
      TORCH_CHECK(query_out->sizes() == query->sizes(), "query_out must have the query's shape");
      out_extent = extent_of(*query_out);
      TORCH_CHECK(!shares_with_itself(out_extent), "query_out must not overlap itself");
      if (!same_elements(*query_out, *query))
        require_apart(out_extent, "query_out", extent_of(*query), "another row's query");
    }
    out = query_out ? *query_out : at::empty({tokens, query_heads, D}, query->options());
    strides[4] = query->stride(0);
    strides[5] = query->stride(1);
    strides[6] = out->stride(0);
    strides[7] = out->stride(1);
  } else {
    TORCH_CHECK(!query_out, "query_out needs a query");
    TORCH_CHECK(!query_norm, "query_norm needs a query");
  }
  const int64_t* position = nullptr;
  int64_t table_rows = 0, rotary_dim = 0;
  TORCH_CHECK(positions.has_value() == cos_sin.has_value(),
              "rotation needs both positions and cos_sin");
  if (cos_sin) {
    position = require_index(*positions, "positions", kv_cache, tokens);
    require_plain(*cos_sin, "cos_sin");
    require_device(*cos_sin, "cos_sin");
    TORCH_CHECK(cos_sin->device() == kv_cache.device(), "cos_sin must be on the kv_cache device");
    TORCH_CHECK(cos_sin->scalar_type() == at::kFloat && cos_sin->dim() == 2,
                "cos_sin must be float32 [positions, rotary_dim]");
    table_rows = cos_sin->size(0);
    rotary_dim = cos_sin->size(1);
  }
  int64_t norm_dtype = dtype;
  for (const auto* norm : {&query_norm, &key_norm})
    if (*norm) {
      require_plain(**norm, "norm weights");
      require_device(**norm, "norm weights");
      TORCH_CHECK((*norm)->device() == kv_cache.device(),
                  "norm weights must be on the kv_cache device");
      TORCH_CHECK((*norm)->dim() == 1 && (*norm)->numel() == D,
                  "norm weights must have head_dim values");
      norm_dtype = dtype_code((*norm)->scalar_type(), "norm weights");
    }
  TORCH_CHECK(!query_norm || !key_norm || query_norm->scalar_type() == key_norm->scalar_type(),
              "norm weights must have the same dtype");
  const Extent cache_extent = extent_of(kv_cache);
  const auto apart = [&](const at::Tensor& t, const char* name) {
    const Extent e = extent_of(t);
    require_apart(cache_extent, "kv_cache", e, name);
    require_apart(out_extent, "query_out", e, name);
  };
  apart(key, "key");
  apart(value, "value");
  apart(slots, "slots");
  if (query) require_apart(cache_extent, "kv_cache", extent_of(*query), "query");
  require_apart(out_extent, "query_out", cache_extent, "kv_cache");
  if (cos_sin) {
    apart(*positions, "positions");
    apart(*cos_sin, "cos_sin");
  }
  if (query_norm) apart(*query_norm, "query_norm");
  if (key_norm) apart(*key_norm, "key_norm");
  check(origami_append_kv_cache(
      key.data_ptr(), value.data_ptr(), query ? query->data_ptr() : nullptr,
      out ? out->data_ptr() : nullptr, dtype, strides, tokens, query_heads, kv_cache.data_ptr(),
      paged_dtype_code(kv_cache.scalar_type(), "kv_cache"), g.layout, g.num_blocks, g.block_size,
      g.heads, D, slot, position, cos_sin ? cos_sin->data_ptr<float>() : nullptr, table_rows,
      rotary_dim, interleaved, query_norm ? query_norm->data_ptr() : nullptr,
      key_norm ? key_norm->data_ptr() : nullptr, norm_dtype, eps, k_scale, v_scale,
      current_stream(kv_cache)));
  return out;
}

// Attention of a batch over a shared prefix and each request's own tokens; fills lse where
// it is given and returns the output rows.
at::Tensor shared_prefix_attention(at::Tensor query, at::Tensor kv_cache,
                                   c10::optional<at::Tensor> prefix_block_ids,
                                   int64_t prefix_tokens, at::Tensor block_tables,
                                   at::Tensor own_tokens, c10::optional<at::Tensor> query_starts,
                                   c10::optional<int64_t> max_query_tokens,
                                   c10::optional<int64_t> max_own_tokens,
                                   c10::optional<double> scale, double k_scale, double v_scale,
                                   c10::optional<at::Tensor> out_, c10::optional<at::Tensor> lse) {
  require_eager();
  require_plain(kv_cache, "kv_cache");
  require_device(kv_cache, "kv_cache");
  const CacheGeom g = layout_cache_geometry(kv_cache);
  const int64_t dtype = paged_dtype_code(query.scalar_type(), "query");
  TORCH_CHECK(dtype != ORIGAMI_DTYPE_FLOAT8_E4M3FN, "query must be float16 or bfloat16");
  require_rows(query, "query", kv_cache, query.scalar_type());
  const int64_t tokens = query.size(0), Hq = query.size(1), D = kv_cache.size(4);
  require_plain(block_tables, "block_tables");
  TORCH_CHECK(block_tables.is_cuda() && block_tables.device() == kv_cache.device(),
              "block_tables must be on the kv_cache device");
  TORCH_CHECK(block_tables.scalar_type() == at::kLong && block_tables.dim() == 2 &&
                  (block_tables.stride(1) == 1 || block_tables.size(1) <= 1),
              "block_tables must be int64 [requests, blocks] with contiguous rows");
  const int64_t requests = block_tables.size(0), blocks = block_tables.size(1);
  const int64_t* const own = require_index(own_tokens, "own_tokens", kv_cache, requests);
  const int64_t *prefix = nullptr, *starts = nullptr;
  int64_t prefix_blocks = 0;
  if (prefix_block_ids) {
    prefix_blocks = prefix_block_ids->numel();
    prefix = require_index(*prefix_block_ids, "prefix_block_ids", kv_cache, prefix_blocks);
  }
  if (query_starts) starts = require_index(*query_starts, "query_starts", kv_cache, requests + 1);
  TORCH_CHECK(starts || tokens == requests,
              "without query_starts every request has one query token");
  const int64_t most =
      max_query_tokens ? *max_query_tokens : (starts ? tokens : std::min<int64_t>(tokens, 1));
  int64_t most_own;  // the block tables' slots; what 64 bits do not hold is refused as too many
  if (max_own_tokens)
    most_own = *max_own_tokens;
  else if (__builtin_mul_overflow(blocks, g.block_size, &most_own))
    most_own = INT64_MAX;
  const c10::OptionalDeviceGuard guard(kv_cache.device());

  at::Tensor out;
  Extent out_extent, lse_extent;  // of new tensors: none
  if (out_) {
    out = *out_;
    require_rows(out, "out", kv_cache, query.scalar_type());
    TORCH_CHECK(out.sizes() == query.sizes(), "out must have the query's shape");
    out_extent = extent_of(out);
    TORCH_CHECK(!shares_with_itself(out_extent), "out must not overlap itself");
  } else {
    // rows of no request are not written: zero in a new tensor
    out = starts ? at::zeros({tokens, Hq, D}, query.options())
                 : at::empty({tokens, Hq, D}, query.options());
  }
  if (lse) {
    require_plain(*lse, "lse");
    require_device(*lse, "lse");
    TORCH_CHECK(lse->device() == kv_cache.device() && lse->scalar_type() == at::kFloat &&
                    lse->dim() == 2 && lse->size(0) == tokens && lse->size(1) == Hq,
                "lse must be float32 [tokens, query heads] on the kv_cache device");
  }
  if (out_ || lse) {
    if (lse) lse_extent = extent_of(*lse);
    require_apart(out_extent, "out", lse_extent, "lse");
    const auto apart = [&](const at::Tensor& t, const char* name) {
      const Extent e = extent_of(t);
      require_apart(out_extent, "out", e, name);
      require_apart(lse_extent, "lse", e, name);
    };
    apart(query, "query");
    apart(kv_cache, "kv_cache");
    apart(block_tables, "block_tables");
    apart(own_tokens, "own_tokens");
    if (prefix_block_ids) apart(*prefix_block_ids, "prefix_block_ids");
    if (query_starts) apart(*query_starts, "query_starts");
  }
  const int64_t cache_dtype = paged_dtype_code(kv_cache.scalar_type(), "kv_cache");
  const int64_t bytes = origami_shared_prefix_attention_workspace(
      tokens, Hq, g.heads, D, prefix_tokens, requests, most, most_own, cache_dtype);
  TORCH_CHECK(bytes >= 0, origami_last_error());
  at::Tensor work;
  if (bytes > 0) work = at::empty({bytes}, query.options().dtype(at::kByte));
  const int64_t strides[4] = {query.stride(0), query.stride(1), out.stride(0), out.stride(1)};
  check(origami_shared_prefix_attention(
      query.data_ptr(), dtype, strides, tokens, Hq, kv_cache.data_ptr(), cache_dtype, g.layout,
      g.num_blocks, g.block_size, g.heads, D, prefix, prefix_blocks, prefix_tokens,
      block_tables.numel() ? block_tables.data_ptr<int64_t>() : nullptr, block_tables.stride(0),
      blocks, own, requests, starts, most, most_own,
      scale ? *scale : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(D, 1))), k_scale,
      v_scale, out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr,
      bytes > 0 ? work.data_ptr() : nullptr, bytes, current_stream(kv_cache)));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Origami KV codec-layout path on MI355X (liborigami_layout.so)";
  m.def("unpack_canonical_storage_chunks_cuda", &unpack_canonical_storage_chunks_cuda);
  m.def("cachegen_unpack_dequantize_cuda", &cachegen_unpack_dequantize_cuda);
  m.def("cachegen_unpack_dequantize_to_kv_cache_cuda",
        &cachegen_unpack_dequantize_to_kv_cache_cuda);
  m.def("kivi_dequantize_to_kv_cache_cuda", &kivi_dequantize_to_kv_cache_cuda);
  m.def("fused_prefix_attention_cuda", &fused_prefix_attention_cuda);
  m.def("kivi_dequantize_to_kv_cache", &kivi_to_kv_cache);
  m.def("pack_canonical_storage_chunks", &pack_canonical_storage_chunks);
  m.def("unpack_canonical_to_kv_cache", &unpack_canonical_to_kv_cache);
  m.def("pack_canonical_from_kv_cache", &pack_canonical_from_kv_cache);
  m.def("unpack_canonical_to_kv_cache_batch", &unpack_canonical_to_kv_cache_batch);
  m.def("restore_plan_create", &restore_plan_create);
  m.def("restore_plan_launch", &restore_plan_launch);
  m.def("restore_plan_destroy", &restore_plan_destroy);
  m.def("append_kv_cache", &append_kv_cache);
  m.def("shared_prefix_attention", &shared_prefix_attention);
  // how both find results that overlap inputs, for tests on any device
  m.def("_tensors_overlap", [](const at::Tensor& a, const at::Tensor& b) {
    return share_bytes(extent_of(a), extent_of(b));
  });
  m.def("_tensor_overlaps_itself",
        [](const at::Tensor& t) { return shares_with_itself(extent_of(t)); });
  m.def("abi_version", &origami_abi_version);
}
