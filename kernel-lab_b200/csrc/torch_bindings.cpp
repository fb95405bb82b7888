// PyTorch operators torch.ops.kernel_lab.* over the C ABI in kernel_lab_b200.h.
//
// Registers the same TORCH_LIBRARY(kernel_lab) schemas as kernel-lab
// (csrc/torch_bindings.cpp:107-119 there), so `import kernel_lab._C` is a drop-in:
//   rms_norm(Tensor! out, Tensor x, Tensor weight, float eps) -> ()
//   fused_add_rms_norm(Tensor! out, Tensor x, Tensor! residual, Tensor weight, float eps) -> ()
//   paged_decode_attention(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache,
//                          Tensor block_table, Tensor seq_lens, float scale) -> ()
// plus one extension op that forces the number of KV splits:
//   paged_decode_attention_splits(..., float scale, int num_splits) -> ()
// Validation mirrors kernel-lab's (TORCH_CHECK -> RuntimeError); a non-zero status from
// the C ABI becomes "kernel_lab: <op> failed: <reason>". Meta kernels (no-ops: the ops
// only mutate their outputs) let torch.compile(fullgraph=True) trace the ops.
//
// The 8-bit serving step (kernel_lab_b200_block8.h): rms_norm_fp8, fused_add_rms_norm_fp8,
// paged_kv_append_block8, paged_decode_attention_block8 and paged_block_select.
//
// Decode scratch (split partials and arrival counters) is owned here, one pair of
// buffers per (device, stream), grown on demand. The counters are zeroed once at allocation; every call
// leaves them zero. Entries live as long as the process (a stream that is destroyed keeps its entry, so a
// host that creates streams per request should reuse a pool of them), and so do outgrown buffers, each
// less than 4/5 of the next: kernels in flight or another thread's launch may still use them.
//
// Calls that are captured into a CUDA graph have scratch of their own, one pair per capture and
// stream: a graph may be replayed on any stream, at the same time as other graphs and eager calls,
// and after the capturing stream's own buffers have grown. It is zeroed at once, outside of
// the capture (a recorded memset would clear the status word at each replay), and is the graph's until
// that is destroyed (a CUDA user object says when; it costs 2 to 3 us a replay, whatever the graph's size); then
// a later capture may have it.
//
// The buffers come from cudaMalloc, not from PyTorch's allocator: whichever pool serves the calling thread or
// stream there (a graph's private pool, torch.compile's) would count them as its own and could outlive or
// refuse them.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <ATen/record_function.h>
#include <torch/extension.h>

#include <atomic>
#include <map>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "kernel_lab_b200.h"
#include "kernel_lab_b200_block8.h"

namespace {

int to_dtype(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return KL_FLOAT32;
    case at::kHalf:
      return KL_FLOAT16;
    case at::kBFloat16:
      return KL_BFLOAT16;
    default:
      TORCH_CHECK(false, "kernel_lab: unsupported dtype ", t);
  }
}

void check_status(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "kernel_lab: ", what, " failed: ", kl_status_string(rc));
}

void rms_norm_impl(at::Tensor& out, const at::Tensor& x, at::Tensor* residual, const at::Tensor& weight,
                   double eps, const char* what) {
  TORCH_CHECK(x.is_cuda() && weight.is_cuda() && out.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(x.dim() >= 1 && x.stride(-1) == 1, "x must have a contiguous last dimension");
  TORCH_CHECK(out.is_contiguous() && weight.is_contiguous(), "out and weight must be contiguous");
  const int64_t hidden = x.size(-1);
  TORCH_CHECK(weight.numel() == hidden, "weight size ", weight.numel(), " != hidden ", hidden);
  TORCH_CHECK(out.sizes() == x.sizes(), "out must match x");
  TORCH_CHECK(x.scalar_type() == weight.scalar_type() && x.scalar_type() == out.scalar_type(),
              "x, weight and out must share a dtype");
  TORCH_CHECK(weight.device() == x.device() && out.device() == x.device(), "tensors must be on one device");
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, hidden});
  TORCH_CHECK(x2.stride(-1) == 1, "x cannot be viewed as rows with a contiguous last dim");
  void* res_ptr = nullptr;
  if (residual != nullptr) {
    TORCH_CHECK(residual->is_contiguous() && residual->sizes() == x.sizes() &&
                    residual->scalar_type() == x.scalar_type() && residual->device() == x.device(),
                "residual must be contiguous, same shape and dtype as x");
    res_ptr = residual->data_ptr();
  }
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(kl_rms_norm(to_dtype(x.scalar_type()), out.data_ptr(), x2.data_ptr(), res_ptr, weight.data_ptr(),
                           static_cast<int>(x2.size(0)), static_cast<int>(hidden), x2.stride(0),
                           static_cast<float>(eps), at::cuda::getCurrentCUDAStream().stream()),
               what);
}

void rms_norm(at::Tensor& out, const at::Tensor& x, const at::Tensor& weight, double eps) {
  rms_norm_impl(out, x, nullptr, weight, eps, "rms_norm");
}

void fused_add_rms_norm(at::Tensor& out, const at::Tensor& x, at::Tensor& residual, const at::Tensor& weight,
                        double eps) {
  rms_norm_impl(out, x, &residual, weight, eps, "fused_add_rms_norm");
}

struct Scratch {
  at::Tensor partials;  // uint8, no initialisation needed
  at::Tensor sync;      // uint8, zero at rest
};

size_t scratch_size(size_t bytes) { return std::max<size_t>(bytes, 256) * 5 / 4; }
bool holds(const at::Tensor& t, size_t bytes) { return t.defined() && static_cast<size_t>(t.numel()) >= bytes; }

// Scratch of one capture's calls on one stream; what was outgrown during the capture stays, for the nodes
// recorded with it.
struct GraphScratch {
  int device;
  cudaStream_t stream;
  unsigned long long capture;
  std::vector<Scratch> grown;  // the last is in use
};

struct ScratchPool {
  std::mutex mu;
  std::map<std::pair<int, cudaStream_t>, Scratch> streams;
  std::vector<at::Tensor> outgrown;
  std::vector<std::unique_ptr<GraphScratch>> graphs;
  std::map<int, std::vector<Scratch>> spare;  // of graphs that are gone
  std::map<int, uint32_t> spare_status;       // their status bits
  std::map<int, cudaStream_t> side;           // a stream of our own per device, for work outside of captures
  // Filled by the driver when a graph is gone; no CUDA call may be made there.
  std::mutex ended_mu;
  std::vector<GraphScratch*> ended;
  std::atomic<bool> any_ended{false};
};

// Never destroyed: a graph may outlive the other statics.
ScratchPool& scratch_pool() {
  static ScratchPool* const pool = new ScratchPool;
  return *pool;
}

void CUDART_CB graph_ended(void* scratch) {
  ScratchPool& pool = scratch_pool();
  const std::lock_guard<std::mutex> lock(pool.ended_mu);
  pool.ended.push_back(static_cast<GraphScratch*>(scratch));
  pool.any_ended.store(true, std::memory_order_release);
}

// The functions below hold pool.mu, with the device current and the thread's capture mode relaxed: while any
// stream captures, others forbid allocations and waits. Nothing here touches a capturing stream.
cudaStream_t side_stream(ScratchPool& pool, int device) {
  cudaStream_t& st = pool.side[device];
  if (st == nullptr) C10_CUDA_CHECK(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking));
  return st;
}

at::Tensor scratch_buffer(ScratchPool& pool, const at::Device& dev, size_t bytes) {
  const auto size = static_cast<int64_t>(scratch_size(bytes));
  const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
  void* p = nullptr;
  if (cudaMalloc(&p, static_cast<size_t>(size)) == cudaSuccess) return at::from_blob(p, {size}, opts);
  (void)cudaGetLastError();  // PyTorch may hold the memory that is left
  const c10::cuda::CUDAStreamGuard guard(c10::cuda::getStreamFromExternal(side_stream(pool, dev.index()), dev.index()));
  return at::empty({size}, opts);
}

// Takes back the scratch of graphs that are gone.
void collect_ended_graphs(ScratchPool& pool) {
  if (!pool.any_ended.load(std::memory_order_acquire)) return;
  std::vector<GraphScratch*> ended;
  {
    const std::lock_guard<std::mutex> lock(pool.ended_mu);
    ended.swap(pool.ended);
    pool.any_ended.store(false, std::memory_order_release);
  }
  for (GraphScratch* g : ended) {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(g->device));
    for (const Scratch& s : g->grown) {
      uint32_t status = 0;
      check_status(kl_paged_decode_read_status(s.sync.data_ptr(), &status, 1, side_stream(pool, g->device)), "scratch");
      pool.spare_status[g->device] |= status;
      pool.spare[g->device].push_back(s);
    }
    for (auto& p : pool.graphs) {
      if (p.get() == g) {
        std::swap(p, pool.graphs.back());
        pool.graphs.pop_back();
        break;
      }
    }
  }
}

// Scratch for a call that is being captured into `graph`.
Scratch graph_scratch(ScratchPool& pool, const at::Device& dev, cudaStream_t stream, unsigned long long capture,
                      cudaGraph_t graph, size_t partial_bytes, size_t sync_bytes) {
  const auto serves = [&](const Scratch& s) { return holds(s.partials, partial_bytes) && holds(s.sync, sync_bytes); };
  GraphScratch* own = nullptr;
  for (const auto& p : pool.graphs) {
    if (p->capture == capture && p->stream == stream && p->device == dev.index()) own = p.get();
  }
  if (own && serves(own->grown.back())) return own->grown.back();
  collect_ended_graphs(pool);
  Scratch s;
  std::vector<Scratch>& spare = pool.spare[dev.index()];
  for (Scratch& t : spare) {
    if (!serves(t)) continue;
    s = t;
    std::swap(t, spare.back());
    spare.pop_back();
    break;
  }
  if (!s.sync.defined()) {
    s.partials = scratch_buffer(pool, dev, partial_bytes);
    s.sync = scratch_buffer(pool, dev, sync_bytes);
    const cudaStream_t side = side_stream(pool, dev.index());
    C10_CUDA_CHECK(cudaMemsetAsync(s.sync.data_ptr(), 0, s.sync.numel(), side));
    C10_CUDA_CHECK(cudaStreamSynchronize(side));
  }
  if (own) {
    own->grown.push_back(s);
    return s;
  }
  pool.graphs.push_back(std::unique_ptr<GraphScratch>(new GraphScratch{dev.index(), stream, capture, {s}}));
  cudaUserObject_t object = nullptr;
  cudaError_t e = cudaUserObjectCreate(&object, pool.graphs.back().get(), graph_ended, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) {
    pool.graphs.pop_back();
  } else {
    e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) cudaUserObjectRelease(object, 1);  // graph_ended takes it from here
  }
  C10_CUDA_CHECK(e);
  return s;
}

// The buffers for a call on `stream`, the current one of `dev`.
Scratch scratch_for(const at::Device& dev, cudaStream_t stream, size_t partial_bytes, size_t sync_bytes) {
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  cudaGraph_t graph = nullptr;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &capturing, &capture, &graph, nullptr, nullptr));
  ScratchPool& pool = scratch_pool();
  const std::lock_guard<std::mutex> lock(pool.mu);
  if (capturing != cudaStreamCaptureStatusNone) {
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    return graph_scratch(pool, dev, stream, capture, graph, partial_bytes, sync_bytes);
  }
  Scratch& s = pool.streams[{dev.index(), stream}];
  if (holds(s.partials, partial_bytes) && holds(s.sync, sync_bytes)) return s;
  const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
  if (!holds(s.partials, partial_bytes)) {
    const at::Tensor grown = scratch_buffer(pool, dev, partial_bytes);
    if (s.partials.defined()) pool.outgrown.push_back(s.partials);
    s.partials = grown;
  }
  if (!holds(s.sync, sync_bytes)) {
    const at::Tensor grown = scratch_buffer(pool, dev, sync_bytes);
    C10_CUDA_CHECK(cudaMemsetAsync(grown.data_ptr(), 0, grown.numel(), stream));
    if (s.sync.defined()) {
      // Status word 0 is sticky until decode_status(clear=True): carry it into the larger buffer
      // (stream-ordered after every earlier call on this stream; the counters are zero at rest).
      C10_CUDA_CHECK(cudaMemcpyAsync(grown.data_ptr(), s.sync.data_ptr(), 4, cudaMemcpyDeviceToDevice, stream));
      pool.outgrown.push_back(s.sync);
    }
    s.sync = grown;
  }
  return s;
}

void paged_decode_impl(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                       const at::Tensor& block_table, const at::Tensor& seq_lens, double scale, int64_t num_splits) {
  TORCH_CHECK(q.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "q is [batch, heads, dim]; caches are 4-D");
  TORCH_CHECK(q.is_contiguous() && out.is_contiguous() && k_cache.is_contiguous() && v_cache.is_contiguous(),
              "q, out and both caches must be contiguous");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache shapes differ");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && seq_lens.scalar_type() == at::kInt,
              "block_table and seq_lens must be int32");
  TORCH_CHECK(block_table.dim() == 2 && block_table.stride(-1) == 1 && seq_lens.is_contiguous(),
              "block_table rows and seq_lens must be contiguous");
  TORCH_CHECK(q.scalar_type() == k_cache.scalar_type() && q.scalar_type() == v_cache.scalar_type() &&
                  q.scalar_type() == out.scalar_type(),
              "q, caches and out must share a dtype");
  TORCH_CHECK(out.sizes() == q.sizes(), "out must match q");
  TORCH_CHECK(k_cache.device() == q.device() && v_cache.device() == q.device() && out.device() == q.device() &&
                  block_table.device() == q.device() && seq_lens.device() == q.device(),
              "tensors must be on one device");
  TORCH_CHECK(num_splits >= 0 && num_splits <= (1 << 20), "num_splits must be >= 0");

  const int batch = static_cast<int>(q.size(0));
  const int num_q_heads = static_cast<int>(q.size(1));
  const int head_dim = static_cast<int>(q.size(2));
  const int page_size = static_cast<int>(k_cache.size(1));
  const int num_kv_heads = static_cast<int>(k_cache.size(2));
  TORCH_CHECK(k_cache.size(3) == head_dim, "cache head_dim differs from q");
  TORCH_CHECK(num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
              "num_q_heads must be a multiple of num_kv_heads");
  TORCH_CHECK(seq_lens.numel() == batch && block_table.size(0) == batch,
              "block_table and seq_lens need one row / entry per sequence");
  if (batch == 0) return;

  const int dtype = to_dtype(q.scalar_type());
  const int max_pages = static_cast<int>(block_table.size(1));
  const c10::cuda::CUDAGuard guard(q.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t partial_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_decode_workspace_size(dtype, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                                              max_pages, static_cast<int>(num_splits), &partial_bytes,
                                              &sync_bytes),
               "paged_decode_attention (workspace)");
  const Scratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
  check_status(kl_paged_decode(dtype, out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                               block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), batch, num_q_heads,
                               num_kv_heads, head_dim, page_size, block_table.stride(0), max_pages,
                               k_cache.size(0), static_cast<float>(scale), static_cast<int>(num_splits),
                               s.partials.data_ptr(), static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                               static_cast<size_t>(s.sync.numel()), stream),
               "paged_decode_attention");
}

void paged_decode_attention(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                            const at::Tensor& v_cache, const at::Tensor& block_table, const at::Tensor& seq_lens,
                            double scale) {
  paged_decode_impl(out, q, k_cache, v_cache, block_table, seq_lens, scale, 0);
}

void paged_decode_attention_splits(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                                   const at::Tensor& v_cache, const at::Tensor& block_table,
                                   const at::Tensor& seq_lens, double scale, int64_t num_splits) {
  paged_decode_impl(out, q, k_cache, v_cache, block_table, seq_lens, scale, num_splits);
}

// Write each sequence's new token's K/V rows into its pages (kl_paged_kv_append); bad page
// ids are skipped and flagged in the same status word as the decode calls of this stream.
void paged_kv_append(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& k_new, const at::Tensor& v_new,
                     const at::Tensor& block_table, const at::Tensor& positions) {
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_new.is_cuda() && v_new.is_cuda(),
              "tensors must be on CUDA");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.is_contiguous() &&
                  k_cache.sizes() == v_cache.sizes(),
              "caches are contiguous [num_pages, page_size, num_kv_heads, head_dim] of one shape");
  const int64_t num_kv_heads = k_cache.size(2), head_dim = k_cache.size(3);
  TORCH_CHECK(k_new.sizes() == v_new.sizes() && k_new.strides() == v_new.strides(),
              "k_new and v_new must have one shape and layout");
  TORCH_CHECK((k_new.dim() == 3 && k_new.size(1) == num_kv_heads && k_new.size(2) == head_dim &&
               k_new.stride(2) == 1 && k_new.stride(1) == head_dim) ||
                  (k_new.dim() == 2 && k_new.size(1) == num_kv_heads * head_dim && k_new.stride(1) == 1),
              "k_new is [batch, num_kv_heads, head_dim] (or [batch, num_kv_heads*head_dim]) with contiguous rows");
  TORCH_CHECK(k_new.scalar_type() == k_cache.scalar_type() && v_new.scalar_type() == k_cache.scalar_type() &&
                  v_cache.scalar_type() == k_cache.scalar_type(),
              "new rows and caches must share a dtype");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && positions.scalar_type() == at::kInt,
              "block_table and positions must be int32");
  TORCH_CHECK(block_table.dim() == 2 && block_table.stride(-1) == 1 && positions.is_contiguous(),
              "block_table rows and positions must be contiguous");
  const int64_t batch = k_new.size(0);
  TORCH_CHECK(positions.numel() == batch && block_table.size(0) == batch,
              "block_table and positions need one row / entry per sequence");
  TORCH_CHECK(k_cache.device() == k_new.device() && v_cache.device() == k_new.device() &&
                  v_new.device() == k_new.device() && block_table.device() == k_new.device() &&
                  positions.device() == k_new.device(),
              "tensors must be on one device");
  if (batch == 0) return;
  const c10::cuda::CUDAGuard guard(k_new.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const Scratch s = scratch_for(k_new.device(), stream, 0, 4);
  check_status(kl_paged_kv_append(to_dtype(k_cache.scalar_type()), k_cache.data_ptr(), v_cache.data_ptr(),
                                  k_new.data_ptr(), v_new.data_ptr(), block_table.data_ptr<int32_t>(),
                                  positions.data_ptr<int32_t>(), static_cast<int>(batch),
                                  static_cast<int>(num_kv_heads), static_cast<int>(head_dim),
                                  static_cast<int>(k_cache.size(1)), block_table.stride(0),
                                  static_cast<int>(block_table.size(1)), k_cache.size(0), k_new.stride(0),
                                  static_cast<uint32_t*>(s.sync.data_ptr()), stream),
               "paged_kv_append");
}

bool is_e4m3(const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte; }

void check_scales(const at::Tensor& k_scale, const at::Tensor& v_scale, int64_t num_kv_heads, const at::Device& dev) {
  TORCH_CHECK(k_scale.scalar_type() == at::kFloat && v_scale.scalar_type() == at::kFloat &&
                  k_scale.is_contiguous() && v_scale.is_contiguous() && k_scale.numel() == num_kv_heads &&
                  v_scale.numel() == num_kv_heads && k_scale.device() == dev && v_scale.device() == dev,
              "k_scale and v_scale are contiguous float32 [num_kv_heads] on the caches' device");
}

// Decode over an e4m3 cache with per-KV-head scales (kl_paged_decode_fp8).
void paged_decode_attention_fp8(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                                const at::Tensor& v_cache, const at::Tensor& k_scale, const at::Tensor& v_scale,
                                const at::Tensor& block_table, const at::Tensor& seq_lens, double scale) {
  TORCH_CHECK(q.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "q is [batch, heads, dim]; caches are 4-D");
  TORCH_CHECK(q.is_contiguous() && out.is_contiguous() && k_cache.is_contiguous() && v_cache.is_contiguous(),
              "q, out and both caches must be contiguous");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache shapes differ");
  TORCH_CHECK(is_e4m3(k_cache) && is_e4m3(v_cache), "caches must be float8_e4m3fn (or uint8 e4m3 codes)");
  TORCH_CHECK((q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) &&
                  out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes(),
              "q and out are fp16 or bf16 of one shape");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && seq_lens.scalar_type() == at::kInt &&
                  block_table.dim() == 2 && block_table.stride(-1) == 1 && seq_lens.is_contiguous(),
              "block_table rows and seq_lens must be contiguous int32");
  TORCH_CHECK(k_cache.device() == q.device() && v_cache.device() == q.device() && out.device() == q.device() &&
                  block_table.device() == q.device() && seq_lens.device() == q.device(),
              "tensors must be on one device");
  const int batch = static_cast<int>(q.size(0));
  const int num_q_heads = static_cast<int>(q.size(1));
  const int head_dim = static_cast<int>(q.size(2));
  const int page_size = static_cast<int>(k_cache.size(1));
  const int num_kv_heads = static_cast<int>(k_cache.size(2));
  TORCH_CHECK(k_cache.size(3) == head_dim, "cache head_dim differs from q");
  TORCH_CHECK(num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, "num_q_heads must be a multiple of num_kv_heads");
  TORCH_CHECK(seq_lens.numel() == batch && block_table.size(0) == batch,
              "block_table and seq_lens need one row / entry per sequence");
  check_scales(k_scale, v_scale, num_kv_heads, q.device());
  if (batch == 0) return;
  const int dtype = to_dtype(q.scalar_type());
  const int max_pages = static_cast<int>(block_table.size(1));
  const c10::cuda::CUDAGuard guard(q.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t partial_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_decode_workspace_size(dtype, batch, num_q_heads, num_kv_heads, head_dim, page_size,
                                              max_pages, 0, &partial_bytes, &sync_bytes),
               "paged_decode_attention_fp8 (workspace)");
  const Scratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
  check_status(kl_paged_decode_fp8(dtype, out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                   k_scale.data_ptr<float>(), v_scale.data_ptr<float>(),
                                   block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), batch,
                                   num_q_heads, num_kv_heads, head_dim, page_size, block_table.stride(0), max_pages,
                                   k_cache.size(0), static_cast<float>(scale), 0, s.partials.data_ptr(),
                                   static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                                   static_cast<size_t>(s.sync.numel()), stream),
               "paged_decode_attention_fp8");
}

// Quantising append into an e4m3 cache (kl_paged_kv_append_fp8).
void paged_kv_append_fp8(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& k_new, const at::Tensor& v_new,
                         const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                         const at::Tensor& positions) {
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_new.is_cuda() && v_new.is_cuda(),
              "tensors must be on CUDA");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.is_contiguous() &&
                  k_cache.sizes() == v_cache.sizes() && is_e4m3(k_cache) && is_e4m3(v_cache),
              "caches are contiguous e4m3 [num_pages, page_size, num_kv_heads, head_dim] of one shape");
  const int64_t num_kv_heads = k_cache.size(2), head_dim = k_cache.size(3);
  TORCH_CHECK(k_new.sizes() == v_new.sizes() && k_new.strides() == v_new.strides() &&
                  k_new.scalar_type() == v_new.scalar_type(),
              "k_new and v_new must have one shape, layout and dtype");
  TORCH_CHECK((k_new.dim() == 3 && k_new.size(1) == num_kv_heads && k_new.size(2) == head_dim &&
               k_new.stride(2) == 1 && k_new.stride(1) == head_dim) ||
                  (k_new.dim() == 2 && k_new.size(1) == num_kv_heads * head_dim && k_new.stride(1) == 1),
              "k_new is [batch, num_kv_heads, head_dim] (or [batch, num_kv_heads*head_dim]) with contiguous rows");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && positions.scalar_type() == at::kInt &&
                  block_table.dim() == 2 && block_table.stride(-1) == 1 && positions.is_contiguous(),
              "block_table rows and positions must be contiguous int32");
  const int64_t batch = k_new.size(0);
  TORCH_CHECK(positions.numel() == batch && block_table.size(0) == batch,
              "block_table and positions need one row / entry per sequence");
  TORCH_CHECK(v_cache.device() == k_cache.device() && k_new.device() == k_cache.device() &&
                  v_new.device() == k_cache.device() && block_table.device() == k_cache.device() &&
                  positions.device() == k_cache.device(),
              "tensors must be on one device");
  check_scales(k_scale, v_scale, num_kv_heads, k_cache.device());
  if (batch == 0) return;
  const c10::cuda::CUDAGuard guard(k_new.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const Scratch s = scratch_for(k_new.device(), stream, 0, 4);
  check_status(kl_paged_kv_append_fp8(to_dtype(k_new.scalar_type()), k_cache.data_ptr(), v_cache.data_ptr(),
                                      k_new.data_ptr(), v_new.data_ptr(), k_scale.data_ptr<float>(),
                                      v_scale.data_ptr<float>(), block_table.data_ptr<int32_t>(),
                                      positions.data_ptr<int32_t>(), static_cast<int>(batch),
                                      static_cast<int>(num_kv_heads), static_cast<int>(head_dim),
                                      static_cast<int>(k_cache.size(1)), block_table.stride(0),
                                      static_cast<int>(block_table.size(1)), k_cache.size(0), k_new.stride(0),
                                      static_cast<uint32_t*>(s.sync.data_ptr()), stream),
               "paged_kv_append_fp8");
}

// Cascade (shared-prefix) decode (kl_paged_decode_cascade): the sequences of group p,
// [prefix_indptr[p], prefix_indptr[p+1]), attend to the prefix_lens[p] tokens in the pages of
// prefix_block_table row p and then to their own. The caches are q's dtype, or e4m3 with
// per-KV-head scales when k_scale / v_scale are given.
void paged_decode_attention_cascade(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                                    const at::Tensor& v_cache, const at::Tensor& prefix_block_table,
                                    const at::Tensor& prefix_lens, const at::Tensor& prefix_indptr,
                                    const at::Tensor& block_table, const at::Tensor& seq_lens, double scale,
                                    const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale) {
  TORCH_CHECK(q.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "q is [batch, heads, dim]; caches are 4-D");
  TORCH_CHECK(q.is_contiguous() && out.is_contiguous() && k_cache.is_contiguous() && v_cache.is_contiguous(),
              "q, out and both caches must be contiguous");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.scalar_type() == v_cache.scalar_type(),
              "k_cache and v_cache differ in shape or dtype");
  TORCH_CHECK(k_scale.has_value() == v_scale.has_value(), "give both k_scale and v_scale, or neither");
  const bool fp8 = k_scale.has_value();
  if (fp8) {
    TORCH_CHECK(is_e4m3(k_cache), "with scales the caches must be float8_e4m3fn (or uint8 e4m3 codes)");
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q is fp16 or bf16");
  } else {
    TORCH_CHECK(q.scalar_type() == k_cache.scalar_type(), "q and caches must share a dtype");
  }
  TORCH_CHECK(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes(), "out must match q");
  for (const at::Tensor* t : {&prefix_block_table, &prefix_lens, &prefix_indptr, &block_table, &seq_lens}) {
    TORCH_CHECK(t->scalar_type() == at::kInt && t->device() == q.device(),
                "block tables, lengths and prefix_indptr must be int32 on q's device");
  }
  TORCH_CHECK(block_table.dim() == 2 && block_table.stride(-1) == 1 && prefix_block_table.dim() == 2 &&
                  prefix_block_table.stride(-1) == 1 && seq_lens.is_contiguous() && prefix_lens.is_contiguous() &&
                  prefix_indptr.is_contiguous(),
              "block-table rows, lengths and prefix_indptr must be contiguous");
  TORCH_CHECK(k_cache.device() == q.device() && v_cache.device() == q.device() && out.device() == q.device(),
              "tensors must be on one device");
  const int batch = static_cast<int>(q.size(0));
  const int num_q_heads = static_cast<int>(q.size(1));
  const int head_dim = static_cast<int>(q.size(2));
  const int page_size = static_cast<int>(k_cache.size(1));
  const int num_kv_heads = static_cast<int>(k_cache.size(2));
  TORCH_CHECK(k_cache.size(3) == head_dim, "cache head_dim differs from q");
  TORCH_CHECK(num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, "num_q_heads must be a multiple of num_kv_heads");
  TORCH_CHECK(seq_lens.numel() == batch && block_table.size(0) == batch,
              "block_table and seq_lens need one row / entry per sequence");
  const int64_t groups = prefix_lens.numel();
  TORCH_CHECK(prefix_block_table.size(0) == groups && prefix_indptr.numel() == groups + 1,
              "prefix_block_table needs one row and prefix_indptr groups + 1 entries per prefix group");
  if (fp8) check_scales(*k_scale, *v_scale, num_kv_heads, q.device());
  if (batch == 0) return;
  const int dtype = to_dtype(q.scalar_type());
  const int max_pages = static_cast<int>(block_table.size(1));
  const int max_prefix_pages = static_cast<int>(prefix_block_table.size(1));
  const c10::cuda::CUDAGuard guard(q.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t partial_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_decode_cascade_workspace_size(dtype, batch, static_cast<int>(groups), num_q_heads,
                                                      num_kv_heads, head_dim, page_size, max_pages, max_prefix_pages,
                                                      &partial_bytes, &sync_bytes),
               "paged_decode_attention_cascade (workspace)");
  const Scratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
  check_status(
      kl_paged_decode_cascade(dtype, out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                              fp8 ? k_scale->data_ptr<float>() : nullptr, fp8 ? v_scale->data_ptr<float>() : nullptr,
                              prefix_block_table.data_ptr<int32_t>(), prefix_lens.data_ptr<int32_t>(),
                              prefix_indptr.data_ptr<int32_t>(), static_cast<int>(groups), prefix_block_table.stride(0),
                              max_prefix_pages, block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), batch,
                              num_q_heads, num_kv_heads, head_dim, page_size, block_table.stride(0), max_pages,
                              k_cache.size(0), static_cast<float>(scale), s.partials.data_ptr(),
                              static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                              static_cast<size_t>(s.sync.numel()), stream),
      "paged_decode_attention_cascade");
}

// RMSNorm with an e4m3 output and a scale a row (group_size 0) or a group of columns
// (kl_rms_norm_fp8); with a residual, residual_out receives x + residual (it may be `residual`).
void rms_norm_fp8_impl(at::Tensor& codes, at::Tensor& scales, at::Tensor* residual_out, const at::Tensor& x,
                       const at::Tensor* residual, const at::Tensor& weight, double eps, int64_t group_size,
                       const char* what) {
  TORCH_CHECK(x.is_cuda() && weight.is_cuda() && codes.is_cuda() && scales.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(x.dim() >= 1 && x.stride(-1) == 1, "x must have a contiguous last dimension");
  TORCH_CHECK(codes.is_contiguous() && scales.is_contiguous() && weight.is_contiguous(),
              "codes, scales and weight must be contiguous");
  const int64_t hidden = x.size(-1);
  TORCH_CHECK(hidden > 0 && hidden <= INT32_MAX, "x must have columns");
  TORCH_CHECK(weight.numel() == hidden, "weight size ", weight.numel(), " != hidden ", hidden);
  TORCH_CHECK(x.scalar_type() == weight.scalar_type(), "x and weight must share a dtype");
  TORCH_CHECK(is_e4m3(codes) && codes.sizes() == x.sizes(), "codes must be float8_e4m3fn (or uint8) and match x");
  TORCH_CHECK(group_size >= 0 && group_size <= INT32_MAX, "group_size must be >= 0");
  const int64_t groups = group_size == 0 ? 1 : (hidden + group_size - 1) / group_size;
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.numel() == x.numel() / hidden * groups,
              "scales must be float32 with ", groups, " per row");
  TORCH_CHECK(weight.device() == x.device() && codes.device() == x.device() && scales.device() == x.device(),
              "tensors must be on one device");
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, hidden});
  TORCH_CHECK(x2.stride(-1) == 1, "x cannot be viewed as rows with a contiguous last dim");
  TORCH_CHECK(x2.size(0) <= INT32_MAX, "too many rows");
  for (const at::Tensor* t : {residual, static_cast<const at::Tensor*>(residual_out)}) {
    TORCH_CHECK(t == nullptr || (t->is_contiguous() && t->sizes() == x.sizes() && t->scalar_type() == x.scalar_type() &&
                                 t->device() == x.device()),
                "residual must be contiguous, same shape and dtype as x");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  check_status(kl_rms_norm_fp8(to_dtype(x.scalar_type()), codes.data_ptr(), scales.data_ptr<float>(),
                               residual_out ? residual_out->data_ptr() : nullptr, x2.data_ptr(),
                               residual ? residual->data_ptr() : nullptr, weight.data_ptr(),
                               static_cast<int>(x2.size(0)), static_cast<int>(hidden), x2.stride(0),
                               static_cast<int>(group_size), static_cast<float>(eps),
                               at::cuda::getCurrentCUDAStream().stream()),
               what);
}

void rms_norm_fp8(at::Tensor& codes, at::Tensor& scales, const at::Tensor& x, const at::Tensor& weight, double eps,
                  int64_t group_size) {
  rms_norm_fp8_impl(codes, scales, nullptr, x, nullptr, weight, eps, group_size, "rms_norm_fp8");
}

void fused_add_rms_norm_fp8(at::Tensor& codes, at::Tensor& scales, at::Tensor& residual_out, const at::Tensor& x,
                            const at::Tensor& residual, const at::Tensor& weight, double eps, int64_t group_size) {
  rms_norm_fp8_impl(codes, scales, &residual_out, x, &residual, weight, eps, group_size, "fused_add_rms_norm_fp8");
}

int code_type_of(const at::Tensor& cache) {
  TORCH_CHECK(cache.scalar_type() == at::kFloat8_e4m3fn || cache.scalar_type() == at::kChar,
              "block-scaled caches are float8_e4m3fn or int8");
  return cache.scalar_type() == at::kChar ? KL_CODE_INT8 : KL_CODE_E4M3;
}

// [num_pages, page_size, num_kv_heads, head_dim] caches of one layout (pages, tokens and heads in any
// order, head_dim contiguous) with [num_pages, num_kv_heads] scales.
void check_block8_cache(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& k_scale,
                        const at::Tensor& v_scale) {
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_scale.is_cuda() && v_scale.is_cuda(),
              "tensors must be on CUDA");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() && k_cache.strides() == v_cache.strides() &&
                  k_cache.scalar_type() == v_cache.scalar_type(),
              "caches are [num_pages, page_size, num_kv_heads, head_dim] of one shape, layout and dtype");
  TORCH_CHECK(k_cache.size(3) > 0 && k_cache.stride(3) == 1, "caches need a contiguous head_dim");
  for (const at::Tensor* t : {&k_scale, &v_scale}) {
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 &&
                    t->size(0) == k_cache.size(0) && t->size(1) == k_cache.size(2),
                "k_scale and v_scale are contiguous float32 [num_pages, num_kv_heads]");
  }
  TORCH_CHECK(v_cache.device() == k_cache.device() && k_scale.device() == k_cache.device() &&
                  v_scale.device() == k_cache.device(),
              "tensors must be on one device");
  for (int64_t d : k_cache.sizes()) TORCH_CHECK(d <= INT32_MAX, "cache dimensions must fit 32 bits");
}

// A dimension's stride; 0 where it has one entry (its stride means nothing there).
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

void check_bounds(const at::Tensor& k_bounds, const at::Tensor& k_cache) {
  TORCH_CHECK(k_bounds.scalar_type() == at::kChar && k_bounds.is_contiguous() && k_bounds.dim() == 4 &&
                  k_bounds.size(0) == k_cache.size(0) && k_bounds.size(1) == k_cache.size(2) &&
                  k_bounds.size(2) == 2 && k_bounds.size(3) == k_cache.size(3) &&
                  k_bounds.device() == k_cache.device(),
              "k_bounds is contiguous int8 [num_pages, num_kv_heads, 2, head_dim] on the caches' device");
}

void check_tables(const at::Tensor& block_table, const at::Tensor& per_sequence, int64_t batch, const at::Device& dev,
                  const char* name) {
  TORCH_CHECK(block_table.scalar_type() == at::kInt && per_sequence.scalar_type() == at::kInt &&
                  block_table.dim() == 2 && block_table.stride(-1) == 1 && per_sequence.is_contiguous(),
              "block_table rows and ", name, " must be contiguous int32");
  TORCH_CHECK(per_sequence.numel() == batch && block_table.size(0) == batch, "block_table and ", name,
              " need one row / entry per sequence");
  TORCH_CHECK(block_table.device() == dev && per_sequence.device() == dev, "tensors must be on one device");
}

// Append into a block-scaled 8-bit cache (kl_paged_kv_append_block8): one token a sequence, or with
// indptr [batch + 1] the rows indptr[b] .. indptr[b + 1] - 1 at positions[b], positions[b] + 1, ...
void paged_kv_append_block8(at::Tensor& k_cache, at::Tensor& v_cache, at::Tensor& k_scale, at::Tensor& v_scale,
                            const std::optional<at::Tensor>& k_bounds, const at::Tensor& k_new,
                            const at::Tensor& v_new, const at::Tensor& block_table, const at::Tensor& positions,
                            const std::optional<at::Tensor>& indptr) {
  check_block8_cache(k_cache, v_cache, k_scale, v_scale);
  const int code_type = code_type_of(k_cache);
  const int64_t num_kv_heads = k_cache.size(2), head_dim = k_cache.size(3);
  TORCH_CHECK(k_new.sizes() == v_new.sizes() && k_new.strides() == v_new.strides() &&
                  k_new.scalar_type() == v_new.scalar_type(),
              "k_new and v_new must have one shape, layout and dtype");
  TORCH_CHECK((k_new.dim() == 3 && k_new.size(1) == num_kv_heads && k_new.size(2) == head_dim &&
               k_new.stride(2) == 1 && (k_new.stride(1) == head_dim || num_kv_heads == 1)) ||
                  (k_new.dim() == 2 && k_new.size(1) == num_kv_heads * head_dim && k_new.stride(1) == 1),
              "k_new is [tokens, num_kv_heads, head_dim] (or [tokens, num_kv_heads*head_dim]) with contiguous rows");
  const int64_t tokens = k_new.size(0), batch = positions.numel();
  check_tables(block_table, positions, batch, k_cache.device(), "positions");
  TORCH_CHECK(k_new.device() == k_cache.device() && v_new.device() == k_cache.device(),
              "tensors must be on one device");
  if (indptr) {
    TORCH_CHECK(indptr->scalar_type() == at::kInt && indptr->is_contiguous() && indptr->numel() == batch + 1 &&
                    indptr->device() == k_cache.device(),
                "indptr is contiguous int32 [batch + 1] on the caches' device");
  } else {
    TORCH_CHECK(tokens == batch, "without indptr there is one new row per sequence");
  }
  if (k_bounds) check_bounds(*k_bounds, k_cache);
  if (batch == 0 || tokens == 0) return;
  // A row stride is arbitrary where there is one row.
  const int64_t row_stride = tokens == 1 ? num_kv_heads * head_dim : k_new.stride(0);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const Scratch s = scratch_for(k_cache.device(), stream, 0, 4);
  check_status(
      kl_paged_kv_append_block8(to_dtype(k_new.scalar_type()), code_type, k_cache.data_ptr(), v_cache.data_ptr(),
                                k_scale.data_ptr<float>(), v_scale.data_ptr<float>(),
                                k_bounds ? k_bounds->data_ptr() : nullptr, k_new.data_ptr(), v_new.data_ptr(),
                                block_table.data_ptr<int32_t>(), positions.data_ptr<int32_t>(),
                                indptr ? indptr->data_ptr<int32_t>() : nullptr, static_cast<int>(batch), tokens,
                                static_cast<int>(num_kv_heads), static_cast<int>(head_dim),
                                static_cast<int>(k_cache.size(1)), stride_of(k_cache, 0), stride_of(k_cache, 1),
                                stride_of(k_cache, 2), block_table.stride(0), static_cast<int>(block_table.size(1)),
                                k_cache.size(0), row_stride, static_cast<uint32_t*>(s.sync.data_ptr()), stream),
      "paged_kv_append_block8");
}

// Decode over a block-scaled 8-bit cache (kl_paged_decode_block8), over every page or over the
// block-table columns in `selected` [batch, num_kv_heads, n].
void paged_decode_attention_block8(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache,
                                   const at::Tensor& v_cache, const at::Tensor& k_scale, const at::Tensor& v_scale,
                                   const at::Tensor& block_table, const at::Tensor& seq_lens, double scale,
                                   const std::optional<at::Tensor>& selected) {
  check_block8_cache(k_cache, v_cache, k_scale, v_scale);
  const int code_type = code_type_of(k_cache);
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.is_contiguous() && out.is_contiguous() && out.sizes() == q.sizes() &&
                  out.scalar_type() == q.scalar_type(),
              "q is a contiguous [batch, heads, dim] and out matches it");
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q and out are fp16 or bf16");
  TORCH_CHECK(q.device() == k_cache.device() && out.device() == k_cache.device(), "tensors must be on one device");
  const int64_t batch = q.size(0), num_q_heads = q.size(1), num_kv_heads = k_cache.size(2);
  TORCH_CHECK(k_cache.size(3) == q.size(2), "cache head_dim differs from q");
  TORCH_CHECK(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
              "num_q_heads must be a multiple of num_kv_heads");
  check_tables(block_table, seq_lens, batch, q.device(), "seq_lens");
  int num_selected = 0;
  if (selected) {
    TORCH_CHECK(selected->scalar_type() == at::kInt && selected->is_contiguous() && selected->dim() == 3 &&
                    selected->size(0) == batch && selected->size(1) == num_kv_heads && selected->size(2) > 0 &&
                    selected->size(2) <= INT32_MAX && selected->device() == q.device(),
                "selected is contiguous int32 [batch, num_kv_heads, n] on q's device");
    num_selected = static_cast<int>(selected->size(2));
  }
  if (batch == 0) return;
  const int d = static_cast<int>(q.size(2)), page = static_cast<int>(k_cache.size(1));
  const int max_pages = static_cast<int>(block_table.size(1));
  const c10::cuda::CUDAGuard guard(q.device());
  // A view may start anywhere; the kernel reads q 16 bytes at a time.
  const at::Tensor rows = reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 ? q : q.clone();
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t partial_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_decode_block8_workspace_size(static_cast<int>(batch), static_cast<int>(num_q_heads),
                                                     static_cast<int>(num_kv_heads), d, page, max_pages, num_selected,
                                                     &partial_bytes, &sync_bytes),
               "paged_decode_attention_block8 (workspace)");
  const Scratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
  check_status(
      kl_paged_decode_block8(to_dtype(q.scalar_type()), code_type, out.data_ptr(), rows.data_ptr(), k_cache.data_ptr(),
                             v_cache.data_ptr(), k_scale.data_ptr<float>(), v_scale.data_ptr<float>(),
                             block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(),
                             selected ? selected->data_ptr<int32_t>() : nullptr, static_cast<int>(batch),
                             static_cast<int>(num_q_heads), static_cast<int>(num_kv_heads), d, page,
                             stride_of(k_cache, 0), stride_of(k_cache, 1), stride_of(k_cache, 2), block_table.stride(0), max_pages,
                             k_cache.size(0), num_selected, static_cast<float>(scale), s.partials.data_ptr(),
                             static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                             static_cast<size_t>(s.sync.numel()), stream),
      "paged_decode_attention_block8");
}

// The pages a decode step should read, by their key bounds (kl_paged_block_select).
void paged_block_select(at::Tensor& selected, const at::Tensor& q, const at::Tensor& k_cache,
                        const at::Tensor& k_scale, const at::Tensor& k_bounds, const at::Tensor& block_table,
                        const at::Tensor& seq_lens, int64_t sink_pages, int64_t recent_pages) {
  check_block8_cache(k_cache, k_cache, k_scale, k_scale);
  const int code_type = code_type_of(k_cache);
  check_bounds(k_bounds, k_cache);
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.is_contiguous() && q.device() == k_cache.device(),
              "q is a contiguous [batch, heads, dim] on the cache's device");
  const int64_t batch = q.size(0), num_q_heads = q.size(1), num_kv_heads = k_cache.size(2);
  TORCH_CHECK(k_cache.size(3) == q.size(2), "cache head_dim differs from q");
  TORCH_CHECK(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
              "num_q_heads must be a multiple of num_kv_heads");
  check_tables(block_table, seq_lens, batch, q.device(), "seq_lens");
  TORCH_CHECK(selected.scalar_type() == at::kInt && selected.is_contiguous() && selected.dim() == 3 &&
                  selected.size(0) == batch && selected.size(1) == num_kv_heads && selected.size(2) > 0 &&
                  selected.size(2) <= INT32_MAX && selected.device() == q.device(),
              "selected is contiguous int32 [batch, num_kv_heads, n] on q's device");
  TORCH_CHECK(sink_pages >= 0 && recent_pages >= 0 && sink_pages <= selected.size(2) &&
                  recent_pages <= selected.size(2) - sink_pages,
              "sink_pages and recent_pages must fit in the selection");
  if (batch == 0) return;
  const int max_pages = static_cast<int>(block_table.size(1));
  const c10::cuda::CUDAGuard guard(q.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t scratch_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_block_select_workspace_size(static_cast<int>(batch), static_cast<int>(num_kv_heads), max_pages,
                                                    &scratch_bytes, &sync_bytes),
               "paged_block_select (workspace)");
  const Scratch s = scratch_for(q.device(), stream, scratch_bytes, sync_bytes);
  check_status(
      kl_paged_block_select(to_dtype(q.scalar_type()), code_type, selected.data_ptr<int32_t>(), q.data_ptr(),
                            k_bounds.data_ptr(), k_scale.data_ptr<float>(), block_table.data_ptr<int32_t>(),
                            seq_lens.data_ptr<int32_t>(), static_cast<int>(batch), static_cast<int>(num_q_heads),
                            static_cast<int>(num_kv_heads), static_cast<int>(q.size(2)),
                            static_cast<int>(k_cache.size(1)), block_table.stride(0), max_pages, k_cache.size(0),
                            static_cast<int>(selected.size(2)), static_cast<int>(sink_pages),
                            static_cast<int>(recent_pages), s.partials.data_ptr(),
                            static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                            static_cast<size_t>(s.sync.numel()), stream),
      "paged_block_select");
}

// Status bits (KL_STATUS_*) left by decode calls on the current device and stream and by the graphs
// captured on the device.
int64_t decode_status(bool clear) {
  const at::Device dev(at::kCUDA, c10::cuda::current_device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  std::vector<at::Tensor> words;
  uint32_t status = 0;
  {
    ScratchPool& pool = scratch_pool();
    const std::lock_guard<std::mutex> lock(pool.mu);
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    collect_ended_graphs(pool);
    const auto it = pool.streams.find({dev.index(), stream});
    if (it != pool.streams.end() && it->second.sync.defined()) words.push_back(it->second.sync);
    for (const auto& p : pool.graphs) {
      if (p->device != dev.index()) continue;
      for (const Scratch& s : p->grown) words.push_back(s.sync);
    }
    uint32_t& gone = pool.spare_status[dev.index()];
    status = gone;
    if (clear) gone = 0;
  }
  for (const at::Tensor& sync : words) {
    uint32_t bits = 0;
    check_status(kl_paged_decode_read_status(sync.data_ptr(), &bits, clear ? 1 : 0, stream), "decode_status");
    status |= bits;
  }
  return status;
}

// Whether a call on these tensors (or None) may go past the dispatcher without anyone's noticing: plain CUDA tensors, and no
// dispatch mode, transform or profiler that would see the operator.
bool direct(const pybind11::args& tensors) {
  c10::DispatchKeySet keys;
  for (const pybind11::handle& t : tensors) {
    if (t.is_none()) continue;
    if (!THPVariable_Check(t.ptr())) return false;
    const at::Tensor& tensor = THPVariable_Unpack(t.ptr());
    if (!tensor.is_cuda()) return false;
    keys = keys | tensor.key_set();
  }
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  // Keys that these operators fall through: no kernels for them.
  const c10::DispatchKeySet through = c10::autograd_dispatch_keyset_with_ADInplaceOrView | c10::autocast_dispatch_keyset |
                                      c10::DispatchKeySet(c10::DispatchKey::BackendSelect);
  const c10::DispatchKeySet seen = ((keys | tls.included_) - tls.excluded_) - through;
  return seen.highestPriorityTypeId() == c10::DispatchKey::CUDA && !at::hasCallbacks();
}

// Functional forms of the 8-bit ops for eager callers (kernel_lab.cuda_ops) whose call is direct(): outputs
// allocated here and the implementation called directly, which costs a host 4-8 us less a call than
// allocating in Python and going through the dispatcher. Others take the torch.ops, which have Meta kernels.
std::pair<at::Tensor, at::Tensor> fp8_outputs(const at::Tensor& x, int64_t group_size) {
  TORCH_CHECK(group_size >= 0, "group_size must be >= 0");
  TORCH_CHECK(x.dim() >= 1 && x.is_cuda(), "x must be rows on CUDA");
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  at::Tensor codes = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
  shape.back() = group_size == 0 ? 1 : (x.size(-1) + group_size - 1) / group_size;
  return {codes, at::empty(shape, x.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> rms_norm_fp8_new(const at::Tensor& x, const at::Tensor& weight, double eps,
                                                    int64_t group_size) {
  auto [codes, scales] = fp8_outputs(x, group_size);
  rms_norm_fp8(codes, scales, x, weight, eps, group_size);
  return {codes, scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> fused_add_rms_norm_fp8_new(const at::Tensor& x,
                                                                          const at::Tensor& residual,
                                                                          const at::Tensor& weight, double eps,
                                                                          int64_t group_size) {
  auto [codes, scales] = fp8_outputs(x, group_size);
  at::Tensor residual_out = at::empty(x.sizes(), x.options());
  fused_add_rms_norm_fp8(codes, scales, residual_out, x, residual.contiguous(), weight, eps, group_size);
  return {codes, scales, residual_out};
}

at::Tensor paged_decode_attention_block8_new(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                             const at::Tensor& k_scale, const at::Tensor& v_scale,
                                             const at::Tensor& block_table, const at::Tensor& seq_lens, double scale,
                                             const std::optional<at::Tensor>& selected) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  paged_decode_attention_block8(out, q.contiguous(), k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, scale, selected);
  return out;
}

at::Tensor paged_block_select_new(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& k_scale,
                                  const at::Tensor& k_bounds, const at::Tensor& block_table,
                                  const at::Tensor& seq_lens, int64_t num_selected, int64_t sink_pages,
                                  int64_t recent_pages) {
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4 && num_selected > 0,
              "q is [batch, heads, dim], the cache is 4-D and num_selected is positive");
  at::Tensor selected = at::empty({q.size(0), k_cache.size(2), num_selected}, q.options().dtype(at::kInt));
  paged_block_select(selected, q.contiguous(), k_cache, k_scale, k_bounds, block_table, seq_lens, sink_pages,
                     recent_pages);
  return selected;
}

void noop_rms_norm(at::Tensor&, const at::Tensor&, const at::Tensor&, double) {}
void noop_fused(at::Tensor&, const at::Tensor&, at::Tensor&, const at::Tensor&, double) {}
void noop_decode(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                 const at::Tensor&, double) {}
void noop_decode_splits(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const at::Tensor&, double, int64_t) {}
void noop_append(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                 const at::Tensor&) {}
void noop_decode_fp8(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                     const at::Tensor&, const at::Tensor&, const at::Tensor&, double) {}
void noop_append_fp8(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                     const at::Tensor&, const at::Tensor&, const at::Tensor&) {}
void noop_cascade(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                  const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, double,
                  const std::optional<at::Tensor>&, const std::optional<at::Tensor>&) {}

void noop_norm_fp8(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, double, int64_t) {}
void noop_fused_fp8(at::Tensor&, at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                    double, int64_t) {}
void noop_append_block8(at::Tensor&, at::Tensor&, at::Tensor&, at::Tensor&, const std::optional<at::Tensor>&,
                        const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const std::optional<at::Tensor>&) {}
void noop_decode_block8(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const at::Tensor&, const at::Tensor&, const at::Tensor&, double,
                        const std::optional<at::Tensor>&) {}
void noop_select(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                 const at::Tensor&, const at::Tensor&, int64_t, int64_t) {}

}  // namespace

TORCH_LIBRARY(kernel_lab, m) {
  m.def("rms_norm(Tensor! out, Tensor x, Tensor weight, float eps) -> ()");
  m.def("fused_add_rms_norm(Tensor! out, Tensor x, Tensor! residual, Tensor weight, float eps) -> ()");
  m.def(
      "paged_decode_attention(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor block_table, Tensor seq_lens, float scale) -> ()");
  m.def(
      "paged_decode_attention_splits(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor block_table, Tensor seq_lens, float scale, int num_splits) -> ()");
  m.def(
      "paged_kv_append(Tensor! k_cache, Tensor! v_cache, Tensor k_new, Tensor v_new, "
      "Tensor block_table, Tensor positions) -> ()");
  m.def(
      "paged_decode_attention_fp8(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, "
      "Tensor v_scale, Tensor block_table, Tensor seq_lens, float scale) -> ()");
  m.def(
      "paged_kv_append_fp8(Tensor! k_cache, Tensor! v_cache, Tensor k_new, Tensor v_new, Tensor k_scale, "
      "Tensor v_scale, Tensor block_table, Tensor positions) -> ()");
  m.def(
      "paged_decode_attention_cascade(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, "
      "Tensor prefix_block_table, Tensor prefix_lens, Tensor prefix_indptr, Tensor block_table, "
      "Tensor seq_lens, float scale, Tensor? k_scale=None, Tensor? v_scale=None) -> ()");
  m.def("rms_norm_fp8(Tensor! codes, Tensor! scales, Tensor x, Tensor weight, float eps, int group_size) -> ()");
  m.def(
      "fused_add_rms_norm_fp8(Tensor! codes, Tensor! scales, Tensor! residual_out, Tensor x, Tensor residual, "
      "Tensor weight, float eps, int group_size) -> ()");
  m.def(
      "paged_kv_append_block8(Tensor! k_cache, Tensor! v_cache, Tensor! k_scale, Tensor! v_scale, "
      "Tensor(a!)? k_bounds, Tensor k_new, Tensor v_new, Tensor block_table, Tensor positions, "
      "Tensor? indptr=None) -> ()");
  m.def(
      "paged_decode_attention_block8(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, "
      "Tensor v_scale, Tensor block_table, Tensor seq_lens, float scale, Tensor? selected=None) -> ()");
  m.def(
      "paged_block_select(Tensor! selected, Tensor q, Tensor k_cache, Tensor k_scale, Tensor k_bounds, "
      "Tensor block_table, Tensor seq_lens, int sink_pages, int recent_pages) -> ()");
}

TORCH_LIBRARY_IMPL(kernel_lab, CUDA, m) {
  m.impl("rms_norm", &rms_norm);
  m.impl("fused_add_rms_norm", &fused_add_rms_norm);
  m.impl("paged_decode_attention", &paged_decode_attention);
  m.impl("paged_decode_attention_splits", &paged_decode_attention_splits);
  m.impl("paged_kv_append", &paged_kv_append);
  m.impl("paged_decode_attention_fp8", &paged_decode_attention_fp8);
  m.impl("paged_kv_append_fp8", &paged_kv_append_fp8);
  m.impl("paged_decode_attention_cascade", &paged_decode_attention_cascade);
  m.impl("rms_norm_fp8", &rms_norm_fp8);
  m.impl("fused_add_rms_norm_fp8", &fused_add_rms_norm_fp8);
  m.impl("paged_kv_append_block8", &paged_kv_append_block8);
  m.impl("paged_decode_attention_block8", &paged_decode_attention_block8);
  m.impl("paged_block_select", &paged_block_select);
}

TORCH_LIBRARY_IMPL(kernel_lab, Meta, m) {
  m.impl("rms_norm", &noop_rms_norm);
  m.impl("fused_add_rms_norm", &noop_fused);
  m.impl("paged_decode_attention", &noop_decode);
  m.impl("paged_decode_attention_splits", &noop_decode_splits);
  m.impl("paged_kv_append", &noop_append);
  m.impl("paged_decode_attention_fp8", &noop_decode_fp8);
  m.impl("paged_kv_append_fp8", &noop_append_fp8);
  m.impl("paged_decode_attention_cascade", &noop_cascade);
  m.impl("rms_norm_fp8", &noop_norm_fp8);
  m.impl("fused_add_rms_norm_fp8", &noop_fused_fp8);
  m.impl("paged_kv_append_block8", &noop_append_block8);
  m.impl("paged_decode_attention_block8", &noop_decode_block8);
  m.impl("paged_block_select", &noop_select);
}

// Importing kernel_lab._C runs the registrations above.
PYBIND11_MODULE(_C, m) {
  m.def("decode_status", &decode_status, pybind11::arg("clear") = false,
        "Status bits left by calls on the current device and stream and by the graphs captured on the device.");
  m.def("direct", &direct);
  m.def("rms_norm_fp8", &rms_norm_fp8_new);
  m.def("fused_add_rms_norm_fp8", &fused_add_rms_norm_fp8_new);
  m.def("paged_kv_append_block8", &paged_kv_append_block8);
  m.def("paged_decode_attention_block8", &paged_decode_attention_block8_new);
  m.def("paged_block_select", &paged_block_select_new);
  m.attr("version") = kl_version();
}
