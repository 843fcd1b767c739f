// PyTorch dispatcher binding of the Branchcraft gfx950 kernels.
//
// Mirrors bindings/torch_ops.cpp of the reference (schemas at :144-148,
// impls under the CUDA dispatch key at :150-154; on PyTorch-ROCm the CUDA
// key is the HIP device key).  Each impl validates its tensors with
// TORCH_CHECK (RuntimeError on failure, same rules as the reference), then
// calls the C ABI in include/branchcraft.h on the current HIP stream of the
// tensors' device, which it makes current for the call.
// Workspaces for split launches come from PyTorch's caching allocator, which
// keeps the ops safe under HIP graph capture.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <tuple>
#include <vector>

#include "bc_rules.h"
#include "branchcraft.h"

namespace {

void check_dev_contig(const at::Tensor& t, const char* name, at::ScalarType dtype) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == dtype, name, " has wrong dtype");
}

void check_launch(int err, const char* op) {
  TORCH_CHECK(err == 0, op, ": ",
              err == BC_ERROR_INVALID_VALUE ? "invalid argument"
                                            : hipGetErrorString((hipError_t)err));
}

bc_stream_t current_stream() {
  return reinterpret_cast<bc_stream_t>(c10::hip::getCurrentHIPStream().stream());
}

const bc_half* hptr(const at::Tensor& t) {
  return reinterpret_cast<const bc_half*>(t.data_ptr<at::Half>());
}

bc_half* hptr_mut(at::Tensor& t) {
  return reinterpret_cast<bc_half*>(t.data_ptr<at::Half>());
}

// Reference: tree_verify_cuda, bindings/torch_ops.cpp:22-67.
at::Tensor tree_verify_hip(const at::Tensor& q, const at::Tensor& prefix_k,
                           const at::Tensor& prefix_v, const at::Tensor& pages,
                           const at::Tensor& lengths, const at::Tensor& draft_k,
                           const at::Tensor& draft_v, const at::Tensor& parent) {
  check_dev_contig(q, "q", at::kHalf);
  check_dev_contig(prefix_k, "prefix_k", at::kHalf);
  check_dev_contig(prefix_v, "prefix_v", at::kHalf);
  check_dev_contig(draft_k, "draft_k", at::kHalf);
  check_dev_contig(draft_v, "draft_v", at::kHalf);
  check_dev_contig(pages, "pages", at::kInt);
  check_dev_contig(lengths, "lengths", at::kInt);
  check_dev_contig(parent, "parent", at::kInt);
  TORCH_CHECK(q.dim() == 4 && prefix_k.dim() == 4 && prefix_v.dim() == 4 &&
                  draft_k.dim() == 4 && draft_v.dim() == 4 && pages.dim() == 2 &&
                  lengths.dim() == 1 && parent.dim() == 2,
              "invalid tree tensor rank");
  const int64_t b = q.size(0), nodes = q.size(1), hq = q.size(2), d = q.size(3);
  const int64_t hkv = prefix_k.size(2);
  TORCH_CHECK(b > 0 && nodes > 0 && nodes <= BC_MAX_TREE_NODES && hq > 0 &&
                  hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128),
              "unsupported tree shape");
  TORCH_CHECK(prefix_k.size(1) == BC_PAGE_SIZE && prefix_k.size(3) == d &&
                  prefix_v.sizes() == prefix_k.sizes(),
              "prefix K/V shape mismatch");
  TORCH_CHECK(draft_k.sizes() == at::IntArrayRef({b, nodes, hkv, d}) &&
                  draft_v.sizes() == draft_k.sizes(),
              "draft K/V shape mismatch");
  TORCH_CHECK(pages.size(0) == b && lengths.size(0) == b &&
                  parent.sizes() == at::IntArrayRef({b, nodes}),
              "tree metadata shape mismatch");
  TORCH_CHECK(q.device() == prefix_k.device() && q.device() == prefix_v.device() &&
                  q.device() == draft_k.device() && q.device() == draft_v.device() &&
                  q.device() == pages.device() && q.device() == lengths.device() &&
                  q.device() == parent.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(q.device());
  auto output = at::empty(q.sizes(), q.options().dtype(at::kFloat));
  TORCH_CHECK(pages.size(1) >= 1, "pages must have at least one column");
  bc_shape shape{int(b), int(hq), int(hkv), int(d), int(pages.size(1)),
                 int(prefix_k.size(0))};
  bc_inputs prefix{nullptr, hptr(prefix_k), hptr(prefix_v), pages.data_ptr<int>(),
                   lengths.data_ptr<int>(), nullptr};
  bc_tree_inputs in{prefix, hptr(q), hptr(draft_k), hptr(draft_v),
                    parent.data_ptr<int>(), output.data_ptr<float>()};
  const size_t ws_bytes = bc_tree_verify_workspace_size(shape, int(nodes));
  at::Tensor ws;
  if (ws_bytes > 0)
    ws = at::empty({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  void* const wsp = ws_bytes ? ws.data_ptr() : nullptr;
  check_launch(bc_tree_verify_ws(shape, in, int(nodes), wsp, ws_bytes, current_stream()),
               "tree_verify");
  return output;
}

// Compute units of a device, cached (an immutable attribute).
int device_cus(int device) {
  static std::atomic<int> cache[64];
  if (device >= 0 && device < 64) {
    const int v = cache[device].load(std::memory_order_relaxed);
    if (v > 0) return v;
  }
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess ||
      n < 1)
    n = 256;
  if (device >= 0 && device < 64) cache[device].store(n, std::memory_order_relaxed);
  return n;
}

// Paged GQA decode with FP32 output.  The reference exposes it only as the
// C++ branchcraft::decode / auto_splits (include/branchcraft.hpp:39-41,
// src/paged_gqa.cu:122-142); this op takes the same tensors as Inputs
// (q [B,Hq,D], k/v [P,16,Hkv,D] FP16, pages [B,max_pages] and lengths [B]
// int32).  splits == 0 picks the split count from the shape alone:
// bc_auto_splits with the page table's capacity (max_pages * 16 tokens) as
// the context bound, so the op never reads lengths back to the host and
// can be captured in a HIP graph.  The split scratch comes from the caching
// allocator on the current stream.
at::Tensor paged_decode_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& pages, const at::Tensor& lengths,
                            int64_t splits) {
  check_dev_contig(q, "q", at::kHalf);
  check_dev_contig(k, "k", at::kHalf);
  check_dev_contig(v, "v", at::kHalf);
  check_dev_contig(pages, "pages", at::kInt);
  check_dev_contig(lengths, "lengths", at::kInt);
  TORCH_CHECK(q.dim() == 3 && k.dim() == 4 && pages.dim() == 2 && lengths.dim() == 1,
              "invalid paged decode tensor rank");
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2);
  TORCH_CHECK(b > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128),
              "unsupported paged decode shape");
  TORCH_CHECK(k.size(0) > 0 && k.size(1) == BC_PAGE_SIZE && k.size(3) == d &&
                  v.sizes() == k.sizes(),
              "K/V cache shape mismatch");
  TORCH_CHECK(pages.size(0) == b && pages.size(1) >= 1 && lengths.size(0) == b,
              "paged decode metadata mismatch");
  TORCH_CHECK(splits >= 0 && splits <= BC_MAX_SPLITS, "splits must be in [0, ",
              BC_MAX_SPLITS, "]");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device() &&
                  q.device() == pages.device() && q.device() == lengths.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(q.device());
  bc_shape shape{int(b), int(hq), int(hkv), int(d), int(pages.size(1)), int(k.size(0))};
  if (splits == 0) {
    const int64_t cap = std::min<int64_t>(pages.size(1) * BC_PAGE_SIZE, 1 << 30);
    splits = bc_auto_splits(shape, int(cap), device_cus(q.device().index()));
  }
  auto output = at::empty(q.sizes(), q.options().dtype(at::kFloat));
  at::Tensor scratch;
  bc_scratch scr{nullptr, nullptr};
  if (splits > 1) {
    const int64_t rows = splits * b * hq;
    scratch = at::empty({rows * (d + 2)}, q.options().dtype(at::kFloat));
    scr.partial_a = scratch.data_ptr<float>();
    scr.partial_ml = scr.partial_a + rows * d;
  }
  bc_inputs in{hptr(q), hptr(k), hptr(v), pages.data_ptr<int>(), lengths.data_ptr<int>(),
               output.data_ptr<float>()};
  check_launch(bc_decode(shape, in, scr, int(splits), current_stream()), "paged_decode");
  return output;
}

// Reference: packed_decode_out_cuda, bindings/torch_ops.cpp:69-104.
// packed_kv is either the reference's logical [P, Hkv, 16, 2D] view (V at
// +D, any outer strides) or [P, 2, 16, Hkv, D] (V at stride(1)); the head
// dimension must be contiguous.
at::Tensor packed_decode_out_hip(const at::Tensor& q, const at::Tensor& packed_kv,
                                 const at::Tensor& pages, const at::Tensor& lengths,
                                 at::Tensor& output, double scale) {
  check_dev_contig(q, "q", at::kHalf);
  check_dev_contig(pages, "pages", at::kInt);
  check_dev_contig(lengths, "lengths", at::kInt);
  check_dev_contig(output, "output", at::kHalf);
  TORCH_CHECK(q.dim() == 3 && pages.dim() == 2 && lengths.dim() == 1,
              "invalid packed decode tensor rank");
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  TORCH_CHECK(packed_kv.is_cuda() && packed_kv.scalar_type() == at::kHalf &&
                  (packed_kv.dim() == 4 || packed_kv.dim() == 5) &&
                  packed_kv.stride(-1) == 1,
              "packed_kv must be a GPU FP16 tensor with contiguous content dim");
  int64_t hkv, bs, hs, ss, kvs;
  if (packed_kv.dim() == 4) {
    hkv = packed_kv.size(1);
    TORCH_CHECK(packed_kv.size(2) == BC_PAGE_SIZE && packed_kv.size(3) == 2 * d,
                "packed KV shape mismatch");
    bs = packed_kv.stride(0);
    hs = packed_kv.stride(1);
    ss = packed_kv.stride(2);
    kvs = d;
  } else {
    hkv = packed_kv.size(3);
    TORCH_CHECK(packed_kv.size(1) == 2 && packed_kv.size(2) == BC_PAGE_SIZE &&
                    packed_kv.size(4) == d,
                "packed KV shape mismatch");
    bs = packed_kv.stride(0);
    kvs = packed_kv.stride(1);
    ss = packed_kv.stride(2);
    hs = packed_kv.stride(3);
  }
  TORCH_CHECK(b > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128),
              "unsupported packed decode shape");
  TORCH_CHECK(pages.size(0) == b && lengths.size(0) == b &&
                  output.numel() == q.numel() && pages.size(1) >= 1,
              "packed decode metadata/output mismatch");
  TORCH_CHECK(q.device() == packed_kv.device() && q.device() == pages.device() &&
                  q.device() == lengths.device() && q.device() == output.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(q.device());
  bc_shape shape{int(b), int(hq), int(hkv), int(d), int(pages.size(1)),
                 int(packed_kv.size(0))};
  const size_t ws_bytes = bc_packed_decode_workspace_size(shape);
  at::Tensor ws;
  if (ws_bytes > 0)
    ws = at::empty({int64_t(ws_bytes)}, q.options().dtype(at::kByte));
  check_launch(bc_packed_decode_ws(shape, hptr(q), hptr(packed_kv),
                                   pages.data_ptr<int>(), lengths.data_ptr<int>(),
                                   hptr_mut(output), bs, hs, ss, kvs, float(scale),
                                   ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                                   current_stream()),
               "packed_decode_out");
  return output;
}

// Reference: commit_path_cuda, bindings/torch_ops.cpp:106-140.
void commit_path_hip(at::Tensor& cache_k, at::Tensor& cache_v,
                     const at::Tensor& draft_k, const at::Tensor& draft_v,
                     const at::Tensor& path_nodes, const at::Tensor& dest_pages,
                     const at::Tensor& dest_slots, int64_t request) {
  check_dev_contig(cache_k, "cache_k", at::kHalf);
  check_dev_contig(cache_v, "cache_v", at::kHalf);
  check_dev_contig(draft_k, "draft_k", at::kHalf);
  check_dev_contig(draft_v, "draft_v", at::kHalf);
  check_dev_contig(path_nodes, "path_nodes", at::kInt);
  check_dev_contig(dest_pages, "dest_pages", at::kInt);
  check_dev_contig(dest_slots, "dest_slots", at::kInt);
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() &&
                  draft_k.dim() == 4 && draft_v.sizes() == draft_k.sizes() &&
                  path_nodes.dim() == 1 && dest_pages.sizes() == path_nodes.sizes() &&
                  dest_slots.sizes() == path_nodes.sizes(),
              "commit tensor shape mismatch");
  const int64_t b = draft_k.size(0), nodes = draft_k.size(1), hkv = draft_k.size(2);
  const int64_t d = draft_k.size(3);
  TORCH_CHECK(request >= 0 && request < b && path_nodes.numel() > 0 &&
                  path_nodes.numel() <= nodes && cache_k.size(1) == BC_PAGE_SIZE &&
                  cache_k.size(2) == hkv && cache_k.size(3) == d,
              "invalid commit destination");
  TORCH_CHECK(cache_k.device() == draft_k.device() && cache_k.device() == cache_v.device() &&
                  cache_k.device() == draft_v.device() &&
                  cache_k.device() == path_nodes.device() &&
                  cache_k.device() == dest_pages.device() &&
                  cache_k.device() == dest_slots.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(cache_k.device());
  bc_shape shape{int(b), int(hkv), int(hkv), int(d), 1, int(cache_k.size(0))};
  check_launch(bc_commit_path(shape, hptr(draft_k), hptr(draft_v), hptr_mut(cache_k),
                              hptr_mut(cache_v), path_nodes.data_ptr<int>(),
                              dest_pages.data_ptr<int>(), dest_slots.data_ptr<int>(),
                              int(request), int(nodes), int(path_nodes.numel()),
                              current_stream()),
               "commit_path_");
}

// Accepted paths of several requests in one launch (no reference op: it
// batches the per-request commit_path_ calls of a transaction,
// python/branchcraft_torch/transaction.py:144-148).
void commit_paths_hip(at::Tensor& cache_k, at::Tensor& cache_v,
                      const at::Tensor& draft_k, const at::Tensor& draft_v,
                      const at::Tensor& requests, const at::Tensor& path_nodes,
                      const at::Tensor& dest_pages, const at::Tensor& dest_slots) {
  check_dev_contig(cache_k, "cache_k", at::kHalf);
  check_dev_contig(cache_v, "cache_v", at::kHalf);
  check_dev_contig(draft_k, "draft_k", at::kHalf);
  check_dev_contig(draft_v, "draft_v", at::kHalf);
  check_dev_contig(requests, "requests", at::kInt);
  check_dev_contig(path_nodes, "path_nodes", at::kInt);
  check_dev_contig(dest_pages, "dest_pages", at::kInt);
  check_dev_contig(dest_slots, "dest_slots", at::kInt);
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() &&
                  draft_k.dim() == 4 && draft_v.sizes() == draft_k.sizes() &&
                  requests.dim() == 1 && path_nodes.sizes() == requests.sizes() &&
                  dest_pages.sizes() == requests.sizes() &&
                  dest_slots.sizes() == requests.sizes(),
              "commit tensor shape mismatch");
  const int64_t b = draft_k.size(0), nodes = draft_k.size(1), hkv = draft_k.size(2);
  const int64_t d = draft_k.size(3);
  TORCH_CHECK(b > 0 && nodes > 0 && cache_k.size(1) == BC_PAGE_SIZE &&
                  cache_k.size(2) == hkv && cache_k.size(3) == d,
              "invalid commit destination");
  TORCH_CHECK(cache_k.device() == draft_k.device() && cache_k.device() == cache_v.device() &&
                  cache_k.device() == draft_v.device() &&
                  cache_k.device() == requests.device() &&
                  cache_k.device() == path_nodes.device() &&
                  cache_k.device() == dest_pages.device() &&
                  cache_k.device() == dest_slots.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(cache_k.device());
  bc_shape shape{int(b), int(hkv), int(hkv), int(d), 1, int(cache_k.size(0))};
  check_launch(bc_commit_paths(shape, hptr(draft_k), hptr(draft_v), hptr_mut(cache_k),
                               hptr_mut(cache_v), requests.data_ptr<int>(),
                               path_nodes.data_ptr<int>(), dest_pages.data_ptr<int>(),
                               dest_slots.data_ptr<int>(), int(nodes),
                               int(requests.numel()), current_stream()),
               "commit_paths_");
}

// Copy-on-write page clone (no reference op: the reference transaction uses
// torch copy_, python/branchcraft_torch/transaction.py:133-134).
void copy_pages_hip(at::Tensor& cache_k, at::Tensor& cache_v,
                    const at::Tensor& src_pages, const at::Tensor& dst_pages) {
  check_dev_contig(cache_k, "cache_k", at::kHalf);
  check_dev_contig(cache_v, "cache_v", at::kHalf);
  check_dev_contig(src_pages, "src_pages", at::kInt);
  check_dev_contig(dst_pages, "dst_pages", at::kInt);
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() &&
                  cache_k.size(1) == BC_PAGE_SIZE && src_pages.dim() == 1 &&
                  dst_pages.sizes() == src_pages.sizes(),
              "copy_pages tensor shape mismatch");
  TORCH_CHECK(cache_k.device() == cache_v.device() &&
                  cache_k.device() == src_pages.device() &&
                  cache_k.device() == dst_pages.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(cache_k.device());
  bc_shape shape{1, int(cache_k.size(2)), int(cache_k.size(2)), int(cache_k.size(3)), 1,
                 int(cache_k.size(0))};
  check_launch(bc_copy_pages(shape, hptr_mut(cache_k), hptr_mut(cache_v),
                             src_pages.data_ptr<int>(), dst_pages.data_ptr<int>(),
                             int(src_pages.numel()), current_stream()),
               "copy_pages_");
}

// A prompt's K and V rows into the pages of a host-side list (the reference
// copies slice by slice, python/branchcraft_torch/transaction.py:64-81).
void write_prefix_hip(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                      const at::Tensor& v, at::IntArrayRef pages) {
  check_dev_contig(cache_k, "cache_k", at::kHalf);
  check_dev_contig(cache_v, "cache_v", at::kHalf);
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && k.scalar_type() == at::kHalf &&
                  v.scalar_type() == at::kHalf,
              "k and v must be GPU FP16 tensors");
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() &&
                  cache_k.size(1) == BC_PAGE_SIZE && k.dim() == 3 && v.sizes() == k.sizes() &&
                  k.size(1) == cache_k.size(2) && k.size(2) == cache_k.size(3) &&
                  k.stride(2) == 1 && v.stride(2) == 1 &&
                  int64_t(pages.size()) == (k.size(0) + BC_PAGE_SIZE - 1) / BC_PAGE_SIZE,
              "write_prefix shape mismatch");
  TORCH_CHECK(cache_k.device() == cache_v.device() && cache_k.device() == k.device() &&
                  cache_k.device() == v.device(),
              "all tensors must share a device");
  TORCH_CHECK(k.size(0) <= INT32_MAX, "write_prefix_: too many tokens");
  const c10::DeviceGuard guard(cache_k.device());
  // Ids past 32 bits are outside every pool, and skipped as such.
  c10::SmallVector<int32_t, 512> ids(pages.size());
  for (size_t i = 0; i < pages.size(); ++i)
    ids[i] = pages[i] >= 0 && pages[i] <= INT32_MAX ? int32_t(pages[i]) : -1;
  bc_shape shape{1, int(cache_k.size(2)), int(cache_k.size(2)), int(cache_k.size(3)), 1,
                 int(cache_k.size(0))};
  if (k.size(0) == 0) return;
  check_launch(bc_write_prefix(shape, hptr(k), hptr(v), k.stride(0), k.stride(1), v.stride(0),
                               v.stride(1), hptr_mut(cache_k), hptr_mut(cache_v), ids.data(),
                               int(k.size(0)), current_stream()),
               "write_prefix_");
}

// Above the kernel, with or without autograd above it (inference mode leaves it
// out for tensors that were made outside): the pools' version counters move.
void write_prefix_versions(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                           const at::Tensor& v, at::IntArrayRef pages) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("branchcraft::write_prefix_", "")
          .typed<void(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                      at::IntArrayRef)>();
  cache_k.unsafeGetTensorImpl()->bump_version();
  cache_v.unsafeGetTensorImpl()->bump_version();
  const at::AutoDispatchBelowADInplaceOrView below;
  op.call(cache_k, cache_v, k, v, pages);
}

// Pools or rows that autograd tracks, or that carry a tangent, are copied page
// by page with ops that have derivatives (and refuse a leaf pool).  Otherwise
// the pools' version counters move, so that a backward that saved a pool before
// a prompt entered it raises, as after those copies.
void write_prefix_autograd(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                           const at::Tensor& v, at::IntArrayRef pages) {
  auto tracked = [](const at::Tensor& x) {
    return (x.requires_grad() && at::GradMode::is_enabled()) || x._fw_grad(0).defined();
  };
  if (tracked(cache_k) || tracked(cache_v) || tracked(k) || tracked(v)) {
    for (size_t i = 0; i < pages.size(); ++i) {
      if (pages[i] < 0 || pages[i] >= cache_k.size(0)) continue;
      const int64_t t0 = int64_t(i) * BC_PAGE_SIZE;
      const int64_t n = std::min<int64_t>(BC_PAGE_SIZE, k.size(0) - t0);
      cache_k.select(0, pages[i]).narrow(0, 0, n).copy_(k.narrow(0, t0, n));
      cache_v.select(0, pages[i]).narrow(0, 0, n).copy_(v.narrow(0, t0, n));
    }
    return;
  }
  write_prefix_versions(cache_k, cache_v, k, v, pages);
}

// A host list as an int32 tensor on `like`'s device, written in stream order
// by kernels that carry the values as arguments.
at::Tensor int_tensor_hip(const at::Tensor& like, at::IntArrayRef values) {
  TORCH_CHECK(values.size() <= INT32_MAX, "int_tensor: too many values");
  std::vector<int32_t> host(values.size());
  for (size_t i = 0; i < values.size(); ++i) {
    TORCH_CHECK(values[i] >= INT32_MIN && values[i] <= INT32_MAX,
                "int_tensor: value out of range");
    host[i] = int32_t(values[i]);
  }
  const c10::DeviceGuard guard(like.device());
  auto out = at::empty({int64_t(host.size())},
                       at::TensorOptions().dtype(at::kInt).device(like.device()));
  if (!host.empty())
    check_launch(bc_write_ints(out.data_ptr<int>(), host.data(), int(host.size()),
                               current_stream()),
                 "int_tensor");
  return out;
}

// Memory straight from the allocator: a dispatched at::empty takes 0.8 us, and
// small calls' time is the host's.
at::Tensor new_tensor(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

// Block table, row offsets, slot map and positions of a step (see
// bc_build_tables); `tokens` rows, those behind the last request -1.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> build_tables_hip(
    const at::Tensor& page_ids, const at::Tensor& lengths, const at::Tensor& counts,
    int64_t max_pages, int64_t tokens) {
  check_dev_contig(page_ids, "page_ids", at::kInt);
  check_dev_contig(lengths, "lengths", at::kInt);
  check_dev_contig(counts, "counts", at::kInt);
  TORCH_CHECK(page_ids.dim() == 1 && lengths.dim() == 1 && counts.sizes() == lengths.sizes(),
              "build_tables shape mismatch");
  TORCH_CHECK(lengths.size(0) > 0, "build_tables: no requests");
  TORCH_CHECK(max_pages >= 1 && max_pages <= BC_MAX_TABLE_PAGES && tokens >= 0 &&
                  tokens < (1 << 27) && page_ids.numel() <= INT32_MAX &&
                  lengths.numel() <= BC_MAX_TABLE_REQUESTS,
              "build_tables: max_pages must be 1 to ", BC_MAX_TABLE_PAGES,
              ", tokens at least 0 and below 2**27, requests at most ", BC_MAX_TABLE_REQUESTS);
  TORCH_CHECK(page_ids.device() == lengths.device() && page_ids.device() == counts.device(),
              "all tensors must share a device");
  const c10::DeviceGuard guard(lengths.device());
  const int64_t b = lengths.size(0);
  auto ints = [&](at::IntArrayRef size) { return new_tensor(lengths, size, at::kInt); };
  auto pages = ints({b, max_pages}), starts = ints({b + 1});
  auto slots = ints({tokens}), positions = ints({tokens});
  check_launch(bc_build_tables(page_ids.data_ptr<int>(), int(page_ids.numel()),
                               lengths.data_ptr<int>(), counts.data_ptr<int>(), int(b),
                               int(max_pages), int(tokens), pages.data_ptr<int>(),
                               starts.data_ptr<int>(), slots.data_ptr<int>(),
                               positions.data_ptr<int>(), current_stream()),
               "build_tables");
  return {pages, starts, slots, positions};
}

// Strides of a [P, 16, Hkv, D] pool in any order of its outer dimensions (a
// dimension of one entry has none).
bc_pool_strides pool_strides(const at::Tensor& t) {
  auto at = [&](int i) { return (long long)(t.size(i) > 1 ? t.stride(i) : 0); };
  return {at(0), at(1), at(2)};
}

bc_row_strides row_strides(const at::Tensor& t) {
  auto at = [&](int i) { return (long long)(t.size(i) > 1 ? t.stride(i) : 0); };
  return {at(0), at(1)};
}

void check_rows(const at::Tensor& t, const char* name, int64_t rank) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name,
              " must be FP16 or BF16");
  TORCH_CHECK(t.dim() == rank, name, " must have ", rank, " dimensions");
  TORCH_CHECK(t.size(-1) == 64 || t.size(-1) == 128, name, ": head dimension must be 64 or 128");
  TORCH_CHECK(t.stride(-1) == 1, name, ": head dimension must be contiguous");
}

const bc_half* raw(const at::Tensor& t) { return static_cast<const bc_half*>(t.data_ptr()); }

// New tokens' K and V rows into the slots of a slot map (see bc_append_kv).
void append_kv_hip(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                   const at::Tensor& v, const at::Tensor& slots) {
  check_rows(cache_k, "cache_k", 4);
  check_rows(cache_v, "cache_v", 4);
  check_rows(k, "k", 3);
  check_rows(v, "v", 3);
  check_dev_contig(slots, "slots", at::kInt);
  TORCH_CHECK(cache_k.scalar_type() == cache_v.scalar_type() &&
                  cache_k.scalar_type() == k.scalar_type() &&
                  cache_k.scalar_type() == v.scalar_type(),
              "append_kv_: pools and rows must share a dtype");
  TORCH_CHECK(cache_k.size(0) > 0 && cache_k.size(1) == BC_PAGE_SIZE &&
                  cache_v.sizes() == cache_k.sizes() && v.sizes() == k.sizes() &&
                  k.size(1) > 0 && k.size(1) == cache_k.size(2) &&
                  k.size(2) == cache_k.size(3) && slots.dim() == 1 &&
                  slots.size(0) == k.size(0),
              "append_kv_ shape mismatch");
  TORCH_CHECK(cache_k.device() == cache_v.device() && cache_k.device() == k.device() &&
                  cache_k.device() == v.device() && cache_k.device() == slots.device(),
              "all tensors must share a device");
  TORCH_CHECK(k.size(0) <= INT32_MAX && cache_k.size(0) <= INT32_MAX &&
                  k.size(1) <= BC_MAX_CHUNK_HEADS,
              "append_kv_: too many tokens, heads or pages");
  at::assert_no_internal_overlap(cache_k);
  at::assert_no_internal_overlap(cache_v);
  at::assert_no_overlap(cache_k, cache_v);
  for (const at::Tensor* rows : {&k, &v}) {
    at::assert_no_overlap(cache_k, *rows);
    at::assert_no_overlap(cache_v, *rows);
  }
  if (k.size(0) == 0) return;
  const c10::DeviceGuard guard(cache_k.device());
  bc_shape shape{1, int(k.size(1)), int(k.size(1)), int(k.size(2)), 1, int(cache_k.size(0))};
  check_launch(bc_append_kv(shape, raw(k), raw(v), row_strides(k), row_strides(v),
                            static_cast<bc_half*>(cache_k.data_ptr()),
                            static_cast<bc_half*>(cache_v.data_ptr()), pool_strides(cache_k),
                            pool_strides(cache_v), slots.data_ptr<int>(), int(k.size(0)),
                            current_stream()),
               "append_kv_");
}

// Neither has a derivative.
void refuse_tracked(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* x : tensors)
    TORCH_CHECK(!(x->requires_grad() && at::GradMode::is_enabled()) && !x->_fw_grad(0).defined(),
                op, " is not differentiable: detach its tensors or call it under no_grad");
}

// Above the kernel, with or without autograd above it (inference mode leaves it
// out for tensors that were made outside): the pools' version counters move, so
// that a backward that saved a pool before the rows entered it raises.
void append_kv_versions(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                        const at::Tensor& v, const at::Tensor& slots) {
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("branchcraft::append_kv_", "")
          .typed<void(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&,
                      const at::Tensor&)>();
  cache_k.unsafeGetTensorImpl()->bump_version();
  cache_v.unsafeGetTensorImpl()->bump_version();
  const at::AutoDispatchBelowADInplaceOrView below;
  op.call(cache_k, cache_v, k, v, slots);
}

// Tensors that autograd tracks or that carry a tangent are refused.
void append_kv_autograd(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& k,
                        const at::Tensor& v, const at::Tensor& slots) {
  refuse_tracked("append_kv_", {&cache_k, &cache_v, &k, &v});
  append_kv_versions(cache_k, cache_v, k, v, slots);
}

// A pool of 8-bit codes, [P, 16, Hkv, D].
void check_codes(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn, name, " must be float8_e4m3fn");
  TORCH_CHECK(t.dim() == 4, name, " must have 4 dimensions");
  TORCH_CHECK(t.size(-1) == 64 || t.size(-1) == 128, name, ": head dimension must be 64 or 128");
  TORCH_CHECK(t.stride(-1) == 1, name, ": head dimension must be contiguous");
  const bc_pool_strides s = pool_strides(t);
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) | uintptr_t(s.page | s.slot | s.head)) % 16 == 0,
              name, " must be aligned to 16 bytes, and so must its pages, slots and heads");
}

// Its scales, [P, Hkv, 16, D / 32].
void check_scales(const at::Tensor& t, const char* name, const at::Tensor& codes) {
  check_dev_contig(t, name, at::kFloat8_e8m0fnu);
  TORCH_CHECK(t.sizes() == at::IntArrayRef({codes.size(0), codes.size(2), BC_PAGE_SIZE,
                                            codes.size(3) / BC_FP8_BLOCK}),
              name, " must be [pages, KV heads, 16, dim / 32]");
  TORCH_CHECK(t.device() == codes.device(), "all tensors must share a device");
}

uint8_t* bytes_of(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

// The checks of both calls on an 8-bit cache's rows, and the cache.
bc_fp8_pool fp8_pool(const char* op, const at::Tensor& cache_k, const at::Tensor& scale_k,
                     const at::Tensor& cache_v, const at::Tensor& scale_v, const at::Tensor& slots,
                     const char* slots_name = "slots") {
  check_codes(cache_k, "cache_k");
  check_codes(cache_v, "cache_v");
  check_scales(scale_k, "scale_k", cache_k);
  check_scales(scale_v, "scale_v", cache_v);
  check_dev_contig(slots, slots_name, at::kInt);
  TORCH_CHECK(cache_k.size(0) > 0 && cache_k.size(1) == BC_PAGE_SIZE && cache_k.size(2) > 0 &&
                  cache_v.sizes() == cache_k.sizes() && slots.dim() == 1,
              op, " shape mismatch");
  TORCH_CHECK(cache_k.device() == cache_v.device() && cache_k.device() == slots.device(),
              "all tensors must share a device");
  TORCH_CHECK(slots.size(0) <= INT32_MAX && cache_k.size(0) <= INT32_MAX &&
                  cache_k.size(2) <= BC_MAX_CHUNK_HEADS,
              op, ": too many tokens, heads or pages");
  return {bytes_of(cache_k), bytes_of(cache_v), bytes_of(scale_k), bytes_of(scale_v),
          pool_strides(cache_k), pool_strides(cache_v)};
}

bc_shape pool_shape(const at::Tensor& cache) {
  return {1, int(cache.size(2)), int(cache.size(2)), int(cache.size(3)), 1, int(cache.size(0))};
}

int dtype_of(at::ScalarType type) { return type == at::kHalf ? BC_FLOAT16 : BC_BFLOAT16; }

// New tokens' K and V rows into an 8-bit cache (see bc_append_fp8_kv).
void append_fp8_kv_hip(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                       at::Tensor& scale_v, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& slots) {
  const bc_fp8_pool pool = fp8_pool("append_fp8_kv_", cache_k, scale_k, cache_v, scale_v, slots);
  check_rows(k, "k", 3);
  check_rows(v, "v", 3);
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), "append_fp8_kv_: k and v must share a dtype");
  TORCH_CHECK(v.sizes() == k.sizes() && k.size(1) == cache_k.size(2) &&
                  k.size(2) == cache_k.size(3) && slots.size(0) == k.size(0),
              "append_fp8_kv_ shape mismatch");
  TORCH_CHECK(cache_k.device() == k.device() && cache_k.device() == v.device(),
              "all tensors must share a device");
  const at::Tensor* const written[] = {&cache_k, &scale_k, &cache_v, &scale_v};
  for (int i = 0; i < 4; ++i) {
    at::assert_no_internal_overlap(*written[i]);
    for (int j = 0; j < i; ++j) at::assert_no_overlap(*written[i], *written[j]);
    at::assert_no_overlap(*written[i], k);
    at::assert_no_overlap(*written[i], v);
  }
  if (k.size(0) == 0) return;
  const c10::DeviceGuard guard(cache_k.device());
  check_launch(bc_append_fp8_kv(pool_shape(cache_k), raw(k), raw(v), row_strides(k), row_strides(v),
                                dtype_of(k.scalar_type()), pool, slots.data_ptr<int>(),
                                int(k.size(0)), current_stream()),
               "append_fp8_kv_");
}

void append_fp8_kv_versions(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                            at::Tensor& scale_v, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& slots) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("branchcraft::append_fp8_kv_", "")
                             .typed<decltype(append_fp8_kv_hip)>();
  for (at::Tensor* x : {&cache_k, &scale_k, &cache_v, &scale_v})
    x->unsafeGetTensorImpl()->bump_version();
  const at::AutoDispatchBelowADInplaceOrView below;
  op.call(cache_k, scale_k, cache_v, scale_v, k, v, slots);
}

void append_fp8_kv_autograd(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                            at::Tensor& scale_v, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& slots) {
  refuse_tracked("append_fp8_kv_", {&cache_k, &scale_k, &cache_v, &scale_v, &k, &v});
  append_fp8_kv_versions(cache_k, scale_k, cache_v, scale_v, k, v, slots);
}

// Pages of an 8-bit cache (see bc_copy_fp8_pages).
void copy_fp8_pages_hip(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                        at::Tensor& scale_v, const at::Tensor& src_pages, const at::Tensor& dst_pages) {
  const bc_fp8_pool pool = fp8_pool("copy_fp8_pages_", cache_k, scale_k, cache_v, scale_v, src_pages,
                                    "src_pages");
  check_dev_contig(dst_pages, "dst_pages", at::kInt);
  TORCH_CHECK(dst_pages.sizes() == src_pages.sizes(), "copy_fp8_pages_ shape mismatch");
  TORCH_CHECK(dst_pages.device() == src_pages.device(), "all tensors must share a device");
  const at::Tensor* const written[] = {&cache_k, &scale_k, &cache_v, &scale_v};
  for (int i = 0; i < 4; ++i) {
    at::assert_no_internal_overlap(*written[i]);
    for (int j = 0; j < i; ++j) at::assert_no_overlap(*written[i], *written[j]);
  }
  if (src_pages.size(0) == 0) return;
  const c10::DeviceGuard guard(cache_k.device());
  check_launch(bc_copy_fp8_pages(pool_shape(cache_k), pool, src_pages.data_ptr<int>(),
                                 dst_pages.data_ptr<int>(), int(src_pages.size(0)), current_stream()),
               "copy_fp8_pages_");
}

void copy_fp8_pages_versions(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                             at::Tensor& scale_v, const at::Tensor& src_pages,
                             const at::Tensor& dst_pages) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("branchcraft::copy_fp8_pages_", "")
                             .typed<decltype(copy_fp8_pages_hip)>();
  for (at::Tensor* x : {&cache_k, &scale_k, &cache_v, &scale_v})
    x->unsafeGetTensorImpl()->bump_version();
  const at::AutoDispatchBelowADInplaceOrView below;
  op.call(cache_k, scale_k, cache_v, scale_v, src_pages, dst_pages);
}

void copy_fp8_pages_autograd(at::Tensor& cache_k, at::Tensor& scale_k, at::Tensor& cache_v,
                             at::Tensor& scale_v, const at::Tensor& src_pages,
                             const at::Tensor& dst_pages) {
  refuse_tracked("copy_fp8_pages_", {&cache_k, &scale_k, &cache_v, &scale_v});
  copy_fp8_pages_versions(cache_k, scale_k, cache_v, scale_v, src_pages, dst_pages);
}

// Rows of an 8-bit cache in 16 bits (see bc_read_fp8_kv).
std::tuple<at::Tensor, at::Tensor> read_fp8_kv_hip(const at::Tensor& cache_k, const at::Tensor& scale_k,
                                                   const at::Tensor& cache_v, const at::Tensor& scale_v,
                                                   const at::Tensor& slots, at::ScalarType dtype) {
  const bc_fp8_pool pool = fp8_pool("read_fp8_kv", cache_k, scale_k, cache_v, scale_v, slots);
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16, "dtype must be FP16 or BF16");
  const c10::DeviceGuard guard(cache_k.device());
  const at::DimVector size{slots.size(0), cache_k.size(2), cache_k.size(3)};
  auto k = new_tensor(cache_k, size, dtype), v = new_tensor(cache_k, size, dtype);
  if (slots.size(0) > 0)
    check_launch(bc_read_fp8_kv(pool_shape(cache_k), pool, slots.data_ptr<int>(), int(slots.size(0)),
                                dtype_of(dtype), static_cast<bc_half*>(k.data_ptr()),
                                static_cast<bc_half*>(v.data_ptr()), current_stream()),
                 "read_fp8_kv");
  return {k, v};
}

std::tuple<at::Tensor, at::Tensor> read_fp8_kv_autograd(const at::Tensor& cache_k,
                                                        const at::Tensor& scale_k,
                                                        const at::Tensor& cache_v,
                                                        const at::Tensor& scale_v,
                                                        const at::Tensor& slots, at::ScalarType dtype) {
  refuse_tracked("read_fp8_kv", {&cache_k, &scale_k, &cache_v, &scale_v});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("branchcraft::read_fp8_kv", "")
                             .typed<decltype(read_fp8_kv_hip)>();
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(cache_k, scale_k, cache_v, scale_v, slots, dtype);
}

// What the chunk attention ops take besides their caches.
struct ChunkOptions {
  std::optional<double> scale;
  bool causal;
  int64_t window;
  double cap;
  const std::optional<at::Tensor>&slopes, &prefix, &first;
};

// The checks of a chunk attention op over a 16-bit cache or, with scales, one of
// 8 bits, and `launch` with the call's shape, inputs and output.
template <typename F>
at::Tensor chunk_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool fp8,
                      const at::Tensor& pages, const at::Tensor& lengths, const at::Tensor& starts,
                      const ChunkOptions& o, F launch) {
  check_rows(q, "q", 3);
  if (fp8) {
    check_codes(k, "k");
    check_codes(v, "v");
  } else {
    check_rows(k, "k", 4);
    check_rows(v, "v", 4);
  }
  check_dev_contig(pages, "pages", at::kInt);
  check_dev_contig(lengths, "lengths", at::kInt);
  check_dev_contig(starts, "starts", at::kInt);
  TORCH_CHECK(fp8 || (q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type()),
              "q, k and v must share a dtype");
  TORCH_CHECK(pages.dim() == 2 && lengths.dim() == 1 && starts.dim() == 1,
              "invalid chunk attention tensor rank");
  const int64_t t = q.size(0), hq = q.size(1), d = q.size(2);
  const int64_t b = lengths.size(0), hkv = k.size(2);
  TORCH_CHECK(b > 0 && hq > 0 && hkv > 0 && hq % hkv == 0, "unsupported chunk attention shape");
  TORCH_CHECK(k.size(0) > 0 && k.size(1) == BC_PAGE_SIZE && k.size(3) == d &&
                  v.sizes() == k.sizes(),
              "K/V cache shape mismatch");
  TORCH_CHECK(pages.size(0) == b && pages.size(1) >= 1 && starts.size(0) == b + 1,
              "chunk attention metadata mismatch");
  TORCH_CHECK(t <= INT32_MAX && k.size(0) <= INT32_MAX && pages.size(1) <= BC_MAX_TABLE_PAGES &&
                  b < INT32_MAX && hq <= BC_MAX_CHUNK_HEADS,
              "chunk attention: too many rows, heads, pages or requests");
  const double s = o.scale.has_value() ? *o.scale : 1.0 / std::sqrt(double(d));
  TORCH_CHECK(float(s) >= BC_LEAST_SCALE && float(s) <= BC_MOST_SCALE,
              "scale must be positive, between ", BC_LEAST_SCALE, " and ", BC_MOST_SCALE);
  TORCH_CHECK(o.window >= 0, "window must not be negative");
  TORCH_CHECK(o.cap == 0 || (float(o.cap) >= BC_LEAST_SCALE && float(o.cap) <= BC_MOST_SCALE),
              "cap must be 0 (none), or between ", BC_LEAST_SCALE, " and ", BC_MOST_SCALE);
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device() &&
                  q.device() == pages.device() && q.device() == lengths.device() &&
                  q.device() == starts.device(),
              "all tensors must share a device");
  auto option = [&](const std::optional<at::Tensor>& x, const char* name, at::ScalarType type,
                    int64_t n) -> const void* {
    if (!x.has_value() || !x->defined()) return nullptr;
    check_dev_contig(*x, name, type);
    TORCH_CHECK(x->dim() == 1 && x->size(0) == n, name, " must have ", n, " entries");
    TORCH_CHECK(x->device() == q.device(), "all tensors must share a device");
    return x->data_ptr();
  };
  bc_chunk_inputs in{};
  in.slopes = static_cast<const float*>(option(o.slopes, "slopes", at::kFloat, hq));
  in.prefix = static_cast<const int32_t*>(option(o.prefix, "prefix", at::kInt, b));
  in.first = static_cast<const int32_t*>(option(o.first, "first", at::kInt, t));
  TORCH_CHECK(o.causal || !in.prefix, "prefix needs causal attention");
  const c10::DeviceGuard guard(q.device());
  auto output = new_tensor(q, q.sizes(), q.scalar_type());
  if (t == 0) return output;
  in.q = raw(q);
  in.k = raw(k);
  in.v = raw(v);
  in.pages = pages.data_ptr<int>();
  in.lengths = lengths.data_ptr<int>();
  in.starts = starts.data_ptr<int>();
  in.output = static_cast<bc_half*>(output.data_ptr());
  in.q_strides = row_strides(q);
  in.k_strides = pool_strides(k);
  in.v_strides = pool_strides(v);
  in.tokens = int(t);
  in.dtype = dtype_of(q.scalar_type());
  in.causal = o.causal;
  in.window = int(std::min<int64_t>(o.window, INT32_MAX));
  in.scale = float(s);
  in.cap = float(o.cap);
  launch(bc_shape{int(b), int(hq), int(hkv), int(d), int(pages.size(1)), int(k.size(0))}, in);
  return output;
}

// The workspace comes from the caching allocator on the current stream and its
// size from shapes alone, so that the ops never read lengths back and can be
// captured.
at::Tensor workspace_of(const at::Tensor& q, size_t bytes) {
  return bytes > 0 ? new_tensor(q, {int64_t(bytes)}, at::kByte) : at::Tensor();
}

// Attention of each request's new tokens over its pages (see
// bc_chunk_attention).
at::Tensor chunk_attention_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& pages, const at::Tensor& lengths,
                               const at::Tensor& starts, std::optional<double> scale,
                               bool causal, int64_t window, double cap,
                               const std::optional<at::Tensor>& slopes,
                               const std::optional<at::Tensor>& prefix,
                               const std::optional<at::Tensor>& first) {
  return chunk_call(q, k, v, false, pages, lengths, starts,
                    {scale, causal, window, cap, slopes, prefix, first},
                    [&](const bc_shape& shape, const bc_chunk_inputs& in) {
                      const size_t bytes = bc_chunk_attention_workspace_size(shape, in.tokens);
                      const at::Tensor ws = workspace_of(q, bytes);
                      check_launch(bc_chunk_attention(shape, in, bytes ? ws.data_ptr() : nullptr,
                                                      bytes, current_stream()),
                                   "chunk_attention");
                    });
}

// The same over an 8-bit cache (see bc_fp8_chunk_attention).
at::Tensor fp8_chunk_attention_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& scale_k,
                                   const at::Tensor& v, const at::Tensor& scale_v,
                                   const at::Tensor& pages, const at::Tensor& lengths,
                                   const at::Tensor& starts, std::optional<double> scale,
                                   bool causal, int64_t window, double cap,
                                   const std::optional<at::Tensor>& slopes,
                                   const std::optional<at::Tensor>& prefix,
                                   const std::optional<at::Tensor>& first) {
  check_codes(k, "k");
  check_codes(v, "v");
  check_scales(scale_k, "scale_k", k);
  check_scales(scale_v, "scale_v", v);
  return chunk_call(q, k, v, true, pages, lengths, starts,
                    {scale, causal, window, cap, slopes, prefix, first},
                    [&](const bc_shape& shape, const bc_chunk_inputs& in) {
                      const size_t bytes = bch::short_window(shape, in)
                                               ? 0
                                               : bc_fp8_chunk_attention_workspace_size(shape, in.tokens);
                      const at::Tensor ws = workspace_of(q, bytes);
                      check_launch(bc_fp8_chunk_attention(shape, in, bytes_of(scale_k), bytes_of(scale_v),
                                                          bytes ? ws.data_ptr() : nullptr, bytes,
                                                          current_stream()),
                                   "fp8_chunk_attention");
                    });
}

// The same for requests that begin with the same pages (see
// bc_shared_chunk_attention).
at::Tensor shared_chunk_attention_hip(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                      const at::Tensor& pages, const at::Tensor& lengths,
                                      const at::Tensor& starts, const at::Tensor& groups,
                                      const at::Tensor& shared, std::optional<double> scale,
                                      bool causal, int64_t window, double cap,
                                      const std::optional<at::Tensor>& slopes,
                                      const std::optional<at::Tensor>& prefix,
                                      const std::optional<at::Tensor>& first) {
  check_dev_contig(groups, "groups", at::kInt);
  check_dev_contig(shared, "shared", at::kInt);
  TORCH_CHECK(groups.dim() == 1 && shared.dim() == 1 && groups.size(0) == shared.size(0) + 1 &&
                  shared.size(0) <= lengths.size(0),
              "groups must have one entry more than shared, and shared at most one per request");
  TORCH_CHECK(groups.device() == q.device() && shared.device() == q.device(),
              "all tensors must share a device");
  const int count = int(shared.size(0));
  return chunk_call(q, k, v, false, pages, lengths, starts,
                    {scale, causal, window, cap, slopes, prefix, first},
                    [&](const bc_shape& shape, const bc_chunk_inputs& in) {
                      const bool once = count > 0 && bch::sharing_pays(shape, in.tokens, in.window);
                      const size_t bytes =
                          !once && bch::short_window(shape, in)
                              ? 0
                              : bc_shared_chunk_attention_workspace_size(shape, in.tokens, count);
                      const at::Tensor ws = workspace_of(q, bytes);
                      check_launch(bc_shared_chunk_attention(shape, in, groups.data_ptr<int>(),
                                                             shared.data_ptr<int>(), count,
                                                             bytes ? ws.data_ptr() : nullptr, bytes,
                                                             current_stream()),
                                   "shared_chunk_attention");
                    });
}

at::Tensor chunk_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                    const at::Tensor& pages, const at::Tensor& lengths,
                                    const at::Tensor& starts, std::optional<double> scale,
                                    bool causal, int64_t window, double cap,
                                    const std::optional<at::Tensor>& slopes,
                                    const std::optional<at::Tensor>& prefix,
                                    const std::optional<at::Tensor>& first) {
  refuse_tracked("chunk_attention", {&q, &k, &v});
  if (slopes.has_value() && slopes->defined()) refuse_tracked("chunk_attention", {&*slopes});
  static const auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("branchcraft::chunk_attention", "")
          .typed<decltype(chunk_attention_hip)>();
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, pages, lengths, starts, scale, causal, window, cap, slopes, prefix, first);
}

at::Tensor fp8_chunk_attention_autograd(const at::Tensor& q, const at::Tensor& k,
                                        const at::Tensor& scale_k, const at::Tensor& v,
                                        const at::Tensor& scale_v, const at::Tensor& pages,
                                        const at::Tensor& lengths, const at::Tensor& starts,
                                        std::optional<double> scale, bool causal, int64_t window,
                                        double cap, const std::optional<at::Tensor>& slopes,
                                        const std::optional<at::Tensor>& prefix,
                                        const std::optional<at::Tensor>& first) {
  refuse_tracked("fp8_chunk_attention", {&q, &k, &scale_k, &v, &scale_v});
  if (slopes.has_value() && slopes->defined()) refuse_tracked("fp8_chunk_attention", {&*slopes});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("branchcraft::fp8_chunk_attention", "")
                             .typed<decltype(fp8_chunk_attention_hip)>();
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, scale_k, v, scale_v, pages, lengths, starts, scale, causal, window, cap, slopes,
                 prefix, first);
}

at::Tensor shared_chunk_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                           const at::Tensor& pages, const at::Tensor& lengths,
                                           const at::Tensor& starts, const at::Tensor& groups,
                                           const at::Tensor& shared, std::optional<double> scale,
                                           bool causal, int64_t window, double cap,
                                           const std::optional<at::Tensor>& slopes,
                                           const std::optional<at::Tensor>& prefix,
                                           const std::optional<at::Tensor>& first) {
  refuse_tracked("shared_chunk_attention", {&q, &k, &v});
  if (slopes.has_value() && slopes->defined()) refuse_tracked("shared_chunk_attention", {&*slopes});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("branchcraft::shared_chunk_attention", "")
                             .typed<decltype(shared_chunk_attention_hip)>();
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, pages, lengths, starts, groups, shared, scale, causal, window, cap, slopes,
                 prefix, first);
}

}  // namespace

TORCH_LIBRARY(branchcraft, m) {
  m.def("tree_verify(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor pages, Tensor lengths, Tensor draft_k, Tensor draft_v, Tensor parent) -> Tensor");
  m.def("packed_decode_out(Tensor q, Tensor packed_kv, Tensor pages, Tensor lengths, Tensor(a!) output, float scale) -> Tensor(a!)");
  m.def("commit_path_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor draft_k, Tensor draft_v, Tensor path_nodes, Tensor dest_pages, Tensor dest_slots, int request) -> ()");
  m.def("copy_pages_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor src_pages, Tensor dst_pages) -> ()");
  m.def("commit_paths_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor draft_k, Tensor draft_v, Tensor requests, Tensor path_nodes, Tensor dest_pages, Tensor dest_slots) -> ()");
  m.def("write_prefix_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor k, Tensor v, int[] pages) -> ()");
  m.def("int_tensor(Tensor like, int[] values) -> Tensor");
  m.def("paged_decode(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor lengths, int splits=0) -> Tensor");
  m.def("build_tables(Tensor page_ids, Tensor lengths, Tensor counts, int max_pages, int tokens) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("append_kv_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor k, Tensor v, Tensor slots) -> ()");
  m.def("chunk_attention(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor lengths, Tensor starts, float? scale=None, bool causal=True, int window=0, float cap=0., Tensor? slopes=None, Tensor? prefix=None, Tensor? first=None) -> Tensor");
  m.def("append_fp8_kv_(Tensor(a!) cache_k, Tensor(b!) scale_k, Tensor(c!) cache_v, Tensor(d!) scale_v, Tensor k, Tensor v, Tensor slots) -> ()");
  m.def("copy_fp8_pages_(Tensor(a!) cache_k, Tensor(b!) scale_k, Tensor(c!) cache_v, Tensor(d!) scale_v, Tensor src_pages, Tensor dst_pages) -> ()");
  m.def("read_fp8_kv(Tensor cache_k, Tensor scale_k, Tensor cache_v, Tensor scale_v, Tensor slots, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("fp8_chunk_attention(Tensor q, Tensor k, Tensor scale_k, Tensor v, Tensor scale_v, Tensor pages, Tensor lengths, Tensor starts, float? scale=None, bool causal=True, int window=0, float cap=0., Tensor? slopes=None, Tensor? prefix=None, Tensor? first=None) -> Tensor");
  m.def("shared_chunk_attention(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor lengths, Tensor starts, Tensor groups, Tensor shared, float? scale=None, bool causal=True, int window=0, float cap=0., Tensor? slopes=None, Tensor? prefix=None, Tensor? first=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(branchcraft, CUDA, m) {
  m.impl("tree_verify", tree_verify_hip);
  m.impl("packed_decode_out", packed_decode_out_hip);
  m.impl("commit_path_", commit_path_hip);
  m.impl("copy_pages_", copy_pages_hip);
  m.impl("commit_paths_", commit_paths_hip);
  m.impl("write_prefix_", write_prefix_hip);
  m.impl("int_tensor", int_tensor_hip);
  m.impl("paged_decode", paged_decode_hip);
  m.impl("build_tables", build_tables_hip);
  m.impl("append_kv_", append_kv_hip);
  m.impl("chunk_attention", chunk_attention_hip);
  m.impl("append_fp8_kv_", append_fp8_kv_hip);
  m.impl("copy_fp8_pages_", copy_fp8_pages_hip);
  m.impl("read_fp8_kv", read_fp8_kv_hip);
  m.impl("fp8_chunk_attention", fp8_chunk_attention_hip);
  m.impl("shared_chunk_attention", shared_chunk_attention_hip);
}

TORCH_LIBRARY_IMPL(branchcraft, ADInplaceOrView, m) {
  m.impl("write_prefix_", write_prefix_versions);
  m.impl("append_kv_", append_kv_versions);
  m.impl("append_fp8_kv_", append_fp8_kv_versions);
  m.impl("copy_fp8_pages_", copy_fp8_pages_versions);
}

TORCH_LIBRARY_IMPL(branchcraft, Autograd, m) {
  m.impl("write_prefix_", write_prefix_autograd);
  m.impl("append_kv_", append_kv_autograd);
  m.impl("chunk_attention", chunk_attention_autograd);
  m.impl("append_fp8_kv_", append_fp8_kv_autograd);
  m.impl("copy_fp8_pages_", copy_fp8_pages_autograd);
  m.impl("read_fp8_kv", read_fp8_kv_autograd);
  m.impl("fp8_chunk_attention", fp8_chunk_attention_autograd);
  m.impl("shared_chunk_attention", shared_chunk_attention_autograd);
  // Whole numbers have no gradient: past autograd at once (0.8 of 8.7 us a call).
  m.impl("build_tables", torch::CppFunction::makeFallthrough());
}
