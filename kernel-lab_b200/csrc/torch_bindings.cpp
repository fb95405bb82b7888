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
// The chunked step (kernel_lab_b200_chunk.h): paged_kv_append_chunks(_fp8), paged_chunk_attention(_fp8,
// _block8), paged_copy_pages, paged_reserve and paged_compact.
//
// Decode scratch (split partials and arrival counters) is owned here, one pair of
// buffers per (device, stream), grown on demand. The counters are zeroed once at allocation; every call
// leaves them zero. Entries live as long as the process (a stream that is destroyed keeps its entry, so a
// host that creates streams per request should reuse a pool of them), and so do outgrown buffers, each
// less than 4/5 of the next: kernels in flight or another thread's launch may still use them.
// Some calls launch kernels that hand data on through the scratch (a cascade's prefix, the marks and the plan of
// paged_reserve and paged_compact). So a call has its stream's scratch to itself until all of them are launched, whatever
// other threads put on that stream.
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

#include <algorithm>
#include <atomic>
#include <map>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "kernel_lab_b200.h"
#include "kernel_lab_b200_block8.h"
#include "kernel_lab_b200_chunk.h"

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

// Scratch for one call, and the right to launch kernels that use it.
struct HeldScratch : Scratch {
  std::unique_lock<std::mutex> launching;
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
  std::map<std::pair<int, cudaStream_t>, std::mutex> launching;  // one of these is taken before mu, never after it
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

// A call whose wait ran out leaves counters behind that later calls would go on from: zeroed once its status has been read.
void zero_after_timeout(const at::Tensor& sync, uint32_t status, cudaStream_t stream) {
  if (!(status & KL_STATUS_WAIT_TIMEOUT)) return;
  C10_CUDA_CHECK(cudaMemsetAsync(sync.data_ptr(), 0, sync.numel(), stream));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
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
      const cudaStream_t side = side_stream(pool, g->device);
      check_status(kl_paged_decode_read_status(s.sync.data_ptr(), &status, 1, side), "scratch");
      zero_after_timeout(s.sync, status, side);
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

// The right to launch on `stream` with its scratch (of its own or of what it captures).
std::unique_lock<std::mutex> launching_on(ScratchPool& pool, const at::Device& dev, cudaStream_t stream) {
  std::mutex* mu;
  {
    const std::lock_guard<std::mutex> lock(pool.mu);
    mu = &pool.launching[{dev.index(), stream}];
  }
  return std::unique_lock<std::mutex>(*mu);
}

// The buffers for a call on `stream`, the current one of `dev`; the result lives until the call has launched its kernels.
HeldScratch scratch_for(const at::Device& dev, cudaStream_t stream, size_t partial_bytes, size_t sync_bytes) {
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  cudaGraph_t graph = nullptr;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &capturing, &capture, &graph, nullptr, nullptr));
  ScratchPool& pool = scratch_pool();
  std::unique_lock<std::mutex> launching = launching_on(pool, dev, stream);
  const std::lock_guard<std::mutex> lock(pool.mu);
  if (capturing != cudaStreamCaptureStatusNone) {
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    return {graph_scratch(pool, dev, stream, capture, graph, partial_bytes, sync_bytes), std::move(launching)};
  }
  Scratch& s = pool.streams[{dev.index(), stream}];
  if (holds(s.partials, partial_bytes) && holds(s.sync, sync_bytes)) return {s, std::move(launching)};
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
  return {s, std::move(launching)};
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
  const HeldScratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
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
  const HeldScratch s = scratch_for(k_new.device(), stream, 0, 4);
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
  const HeldScratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
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
  const HeldScratch s = scratch_for(k_new.device(), stream, 0, 4);
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
  const HeldScratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
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
  const HeldScratch s = scratch_for(k_cache.device(), stream, 0, 4);
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
  const HeldScratch s = scratch_for(q.device(), stream, partial_bytes, sync_bytes);
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
  const HeldScratch s = scratch_for(q.device(), stream, scratch_bytes, sync_bytes);
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

// Rows of chunks: sequence b's are indptr[b] .. indptr[b + 1] - 1.
void check_indptr(const at::Tensor& indptr, int64_t batch, const at::Device& dev) {
  TORCH_CHECK(indptr.scalar_type() == at::kInt && indptr.is_contiguous() && indptr.dim() == 1 && indptr.numel() == batch + 1 &&
                  indptr.device() == dev,
              "indptr is contiguous int32 [batch + 1] on the caches' device");
}

// Append of chunks (kl_paged_kv_append_chunks; with scales kl_paged_kv_append_chunks_fp8).
void append_chunks_impl(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& k_new, const at::Tensor& v_new,
                        const at::Tensor* k_scale, const at::Tensor* v_scale, const at::Tensor& block_table,
                        const at::Tensor& positions, const at::Tensor& indptr, const char* what) {
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_new.is_cuda() && v_new.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.is_contiguous() && k_cache.sizes() == v_cache.sizes() &&
                  k_cache.scalar_type() == v_cache.scalar_type(),
              "caches are contiguous [num_pages, page_size, num_kv_heads, head_dim] of one shape and dtype");
  const int64_t num_kv_heads = k_cache.size(2), head_dim = k_cache.size(3);
  TORCH_CHECK(k_new.sizes() == v_new.sizes() && k_new.strides() == v_new.strides() && k_new.scalar_type() == v_new.scalar_type(),
              "k_new and v_new must have one shape, layout and dtype");
  TORCH_CHECK((k_new.dim() == 3 && k_new.size(1) == num_kv_heads && k_new.size(2) == head_dim && k_new.stride(2) == 1 &&
               (k_new.stride(1) == head_dim || num_kv_heads == 1)) ||
                  (k_new.dim() == 2 && k_new.size(1) == num_kv_heads * head_dim && k_new.stride(1) == 1),
              "k_new is [tokens, num_kv_heads, head_dim] (or [tokens, num_kv_heads*head_dim]) with contiguous rows");
  const at::Device dev = k_cache.device();
  const int64_t tokens = k_new.size(0), batch = positions.numel();
  check_tables(block_table, positions, batch, dev, "positions");
  check_indptr(indptr, batch, dev);
  TORCH_CHECK(v_cache.device() == dev && k_new.device() == dev && v_new.device() == dev, "tensors must be on one device");
  for (int64_t d : k_cache.sizes()) TORCH_CHECK(d <= INT32_MAX, "cache dimensions must fit 32 bits");
  TORCH_CHECK(batch <= INT32_MAX && block_table.size(1) <= INT32_MAX, "too many sequences or pages");
  if (k_scale) {
    TORCH_CHECK(is_e4m3(k_cache), "caches must be float8_e4m3fn (or uint8 e4m3 codes)");
    check_scales(*k_scale, *v_scale, num_kv_heads, dev);
  } else {
    TORCH_CHECK(k_new.scalar_type() == k_cache.scalar_type(), "new rows and caches must share a dtype");
  }
  if (batch == 0 || tokens == 0) return;
  // A row stride is arbitrary where there is one row.
  const int64_t row_stride = tokens == 1 ? num_kv_heads * head_dim : k_new.stride(0);
  const c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const HeldScratch s = scratch_for(dev, stream, 0, 4);
  uint32_t* const status = static_cast<uint32_t*>(s.sync.data_ptr());
  const int dtype = to_dtype(k_new.scalar_type()), heads = static_cast<int>(num_kv_heads), dim = static_cast<int>(head_dim);
  const int page = static_cast<int>(k_cache.size(1)), width = static_cast<int>(block_table.size(1)), b = static_cast<int>(batch);
  check_status(
      k_scale ? kl_paged_kv_append_chunks_fp8(dtype, k_cache.data_ptr(), v_cache.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
                                              k_scale->data_ptr<float>(), v_scale->data_ptr<float>(),
                                              block_table.data_ptr<int32_t>(), positions.data_ptr<int32_t>(),
                                              indptr.data_ptr<int32_t>(), b, tokens, heads, dim, page, block_table.stride(0),
                                              width, k_cache.size(0), row_stride, status, stream)
              : kl_paged_kv_append_chunks(dtype, k_cache.data_ptr(), v_cache.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
                                          block_table.data_ptr<int32_t>(), positions.data_ptr<int32_t>(),
                                          indptr.data_ptr<int32_t>(), b, tokens, heads, dim, page, block_table.stride(0), width,
                                          k_cache.size(0), row_stride, status, stream),
      what);
}

void paged_kv_append_chunks(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& k_new, const at::Tensor& v_new,
                            const at::Tensor& block_table, const at::Tensor& positions, const at::Tensor& indptr) {
  append_chunks_impl(k_cache, v_cache, k_new, v_new, nullptr, nullptr, block_table, positions, indptr, "paged_kv_append_chunks");
}

void paged_kv_append_chunks_fp8(at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& k_new, const at::Tensor& v_new,
                                const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                                const at::Tensor& positions, const at::Tensor& indptr) {
  append_chunks_impl(k_cache, v_cache, k_new, v_new, &k_scale, &v_scale, block_table, positions, indptr,
                     "paged_kv_append_chunks_fp8");
}

// Attention of chunks of new tokens (kl_paged_chunk_attention). Without scales the caches are q's dtype; scales are
// [num_kv_heads], or per page [num_pages, num_kv_heads].
void chunk_attention_impl(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                          const at::Tensor* k_scale, const at::Tensor* v_scale, const at::Tensor& block_table,
                          const at::Tensor& seq_lens, const at::Tensor& indptr, double scale, bool causal, int code_type,
                          bool per_page, const char* what) {
  TORCH_CHECK(q.is_cuda() && out.is_cuda() && k_cache.is_cuda() && v_cache.is_cuda(), "tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 && k_cache.dim() == 4, "q is [tokens, heads, dim]; caches are 4-D");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.strides() == v_cache.strides() &&
                  k_cache.scalar_type() == v_cache.scalar_type() && k_cache.size(3) > 0 && k_cache.stride(3) == 1,
              "caches are [num_pages, page_size, num_kv_heads, head_dim] of one shape, layout and dtype, head_dim contiguous");
  const int64_t tokens = q.size(0), hq = q.size(1), dim = q.size(2), hkv = k_cache.size(2);
  TORCH_CHECK(dim == k_cache.size(3), "cache head_dim differs from q");
  TORCH_CHECK(hkv > 0 && hq > 0 && hq % hkv == 0, "num_q_heads must be a multiple of num_kv_heads");
  TORCH_CHECK(q.stride(2) == 1 && (q.stride(1) == dim || hq == 1), "a row of q must be contiguous");
  TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(),
              "out must be contiguous and match q");
  if (code_type == KL_CODE_NONE) {
    TORCH_CHECK(q.scalar_type() == k_cache.scalar_type(), "q and caches must share a dtype");
  } else {
    TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16, "q and out are fp16 or bf16");
  }
  const at::Device dev = q.device();
  TORCH_CHECK(out.device() == dev && k_cache.device() == dev && v_cache.device() == dev, "tensors must be on one device");
  const int64_t batch = seq_lens.numel();
  check_tables(block_table, seq_lens, batch, dev, "seq_lens");
  check_indptr(indptr, batch, dev);
  for (int64_t d : k_cache.sizes()) TORCH_CHECK(d <= INT32_MAX, "cache dimensions must fit 32 bits");
  TORCH_CHECK(batch <= 65535 && tokens <= INT32_MAX - 256 && hq <= INT32_MAX && block_table.size(1) <= INT32_MAX,
              "too many sequences, tokens, heads or pages");
  if (batch == 0 || tokens == 0) return;
  const c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const int dtype = to_dtype(q.scalar_type()), b = static_cast<int>(batch), d = static_cast<int>(dim);
  size_t partial_bytes = 0, sync_bytes = 0;
  check_status(kl_paged_chunk_attention_workspace_size(dtype, code_type, tokens, b, static_cast<int>(hq), static_cast<int>(hkv), d,
                                                       &partial_bytes, &sync_bytes),
               what);
  const HeldScratch s = scratch_for(dev, stream, partial_bytes, sync_bytes);
  check_status(
      kl_paged_chunk_attention(dtype, code_type, out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                               k_scale ? k_scale->data_ptr<float>() : nullptr, v_scale ? v_scale->data_ptr<float>() : nullptr,
                               block_table.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(), indptr.data_ptr<int32_t>(), b, tokens,
                               static_cast<int>(hq), static_cast<int>(hkv), d, static_cast<int>(k_cache.size(1)),
                               tokens == 1 ? hq * dim : q.stride(0), stride_of(k_cache, 0), stride_of(k_cache, 1),
                               stride_of(k_cache, 2), per_page ? hkv : 0, block_table.stride(0),
                               static_cast<int>(block_table.size(1)), k_cache.size(0), causal, static_cast<float>(scale),
                               s.partials.data_ptr(), static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                               static_cast<size_t>(s.sync.numel()), stream),
      what);
}

void paged_chunk_attention(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& indptr, double scale,
                           bool causal) {
  chunk_attention_impl(out, q, k_cache, v_cache, nullptr, nullptr, block_table, seq_lens, indptr, scale, causal, KL_CODE_NONE,
                       false, "paged_chunk_attention");
}

void paged_chunk_attention_fp8(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                               const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                               const at::Tensor& seq_lens, const at::Tensor& indptr, double scale, bool causal) {
  TORCH_CHECK(k_cache.dim() == 4 && is_e4m3(k_cache), "caches must be float8_e4m3fn (or uint8 e4m3 codes)");
  check_scales(k_scale, v_scale, k_cache.size(2), k_cache.device());
  chunk_attention_impl(out, q, k_cache, v_cache, &k_scale, &v_scale, block_table, seq_lens, indptr, scale, causal, KL_CODE_E4M3,
                       false, "paged_chunk_attention_fp8");
}

void paged_chunk_attention_block8(at::Tensor& out, const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                  const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                                  const at::Tensor& seq_lens, const at::Tensor& indptr, double scale, bool causal) {
  check_block8_cache(k_cache, v_cache, k_scale, v_scale);
  chunk_attention_impl(out, q, k_cache, v_cache, &k_scale, &v_scale, block_table, seq_lens, indptr, scale, causal,
                       code_type_of(k_cache), true, "paged_chunk_attention_block8");
}

// The pools of the page operators: tensors whose first dimension is the page, each page's elements filling one
// piece of memory (in any order of its dimensions).
struct Pools {
  std::vector<void*> base;
  std::vector<int64_t> stride, bytes;
  int64_t num_pages = 0;
  at::Device device = at::kCPU;
  kl_page_pools_t c() const { return {static_cast<int>(base.size()), base.data(), stride.data(), bytes.data()}; }
};

Pools check_pools(at::TensorList caches) {
  TORCH_CHECK(!caches.empty(), "there must be at least one cache");
  Pools p;
  p.num_pages = caches[0].dim() > 0 ? caches[0].size(0) : 0;
  p.device = caches[0].device();
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (const at::Tensor& t : caches) {
    TORCH_CHECK(t.is_cuda() && t.device() == p.device, "caches must be on one CUDA device");
    TORCH_CHECK(t.dim() >= 1 && t.size(0) == p.num_pages && p.num_pages <= INT32_MAX - 8, "caches must have one number of pages");
    dims.clear();
    int64_t elements = 1;
    for (int64_t i = 1; i < t.dim(); ++i) {
      elements *= t.size(i);
      if (t.size(i) > 1) dims.emplace_back(t.stride(i), t.size(i));
    }
    std::sort(dims.begin(), dims.end());
    int64_t filled = 1;
    for (const auto& d : dims) {
      TORCH_CHECK(elements == 0 || d.first == filled, "a page of a cache must fill one piece of memory");
      filled *= d.second;
    }
    const int64_t e = t.element_size();
    TORCH_CHECK(p.num_pages <= 1 || t.stride(0) >= elements, "pages of a cache must not overlap");
    if (elements == 0 || p.num_pages == 0) continue;
    p.base.push_back(t.data_ptr());
    p.stride.push_back((p.num_pages > 1 ? t.stride(0) : elements) * e);
    p.bytes.push_back(elements * e);
  }
  return p;
}

bool is_index(const at::Tensor& t, const at::Device& dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.device() == dev;
}

void paged_copy_pages(at::TensorList caches, const at::Tensor& src, const at::Tensor& dst) {
  const Pools p = check_pools(caches);
  TORCH_CHECK(is_index(src, p.device) && is_index(dst, p.device) && src.numel() == dst.numel() && src.numel() <= INT32_MAX,
              "src and dst are contiguous int32 of one length on the caches' device");
  if (src.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(p.device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  const HeldScratch s = scratch_for(p.device, stream, 0, 4);
  const kl_page_pools_t pools = p.c();
  check_status(kl_paged_copy_pages(&pools, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), src.numel(), p.num_pages,
                                   static_cast<uint32_t*>(s.sync.data_ptr()), stream),
               "paged_copy_pages");
}

void check_page_table(const at::Tensor& out_table, const at::Tensor& block_table, const at::Tensor& seq_lens, int64_t rows,
                      const at::Device& dev) {
  check_tables(block_table, seq_lens, seq_lens.numel(), dev, "seq_lens");
  TORCH_CHECK(out_table.scalar_type() == at::kInt && out_table.is_contiguous() && out_table.dim() == 2 && out_table.size(0) == rows &&
                  out_table.size(1) == block_table.size(1) && out_table.device() == dev,
              "out_table is contiguous int32 [rows, width of block_table] on the caches' device");
  TORCH_CHECK(seq_lens.numel() <= INT32_MAX && rows <= (1 << 24) && block_table.size(1) <= INT32_MAX, "too many sequences or pages");
}

// Pages for new tokens, and forks (kl_paged_reserve).
void paged_reserve(at::Tensor& out_table, at::Tensor& out_lens, at::Tensor& served, at::TensorList caches,
                   const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& new_tokens,
                   const std::optional<at::Tensor>& parents, int64_t page_size) {
  const Pools p = check_pools(caches);
  const int64_t batch = seq_lens.numel(), rows = parents ? parents->numel() : batch;
  check_page_table(out_table, block_table, seq_lens, rows, p.device);
  TORCH_CHECK(page_size > 0 && page_size <= INT32_MAX, "page_size must be positive");
  TORCH_CHECK(is_index(new_tokens, p.device) && new_tokens.numel() == rows && (!parents || is_index(*parents, p.device)),
              "new_tokens and parents are contiguous int32 [rows] on the caches' device");
  TORCH_CHECK(is_index(out_lens, p.device) && out_lens.numel() == rows && served.scalar_type() == at::kBool && served.dim() == 1 &&
                  served.is_contiguous() && served.numel() == rows && served.device() == p.device,
              "out_lens is int32 [rows] and served bool [rows] on the caches' device");
  if (rows == 0) return;
  const c10::cuda::CUDAGuard guard(p.device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t bytes = 0, sync_bytes = 0;
  check_status(kl_paged_reserve_workspace_size(p.num_pages, static_cast<int>(rows), &bytes, &sync_bytes), "paged_reserve (workspace)");
  const HeldScratch s = scratch_for(p.device, stream, bytes, sync_bytes);
  const kl_page_pools_t pools = p.c();
  check_status(kl_paged_reserve(&pools, out_table.data_ptr<int32_t>(), out_lens.data_ptr<int32_t>(),
                                reinterpret_cast<uint8_t*>(served.data_ptr<bool>()), block_table.data_ptr<int32_t>(),
                                seq_lens.data_ptr<int32_t>(), new_tokens.data_ptr<int32_t>(),
                                parents ? parents->data_ptr<int32_t>() : nullptr, static_cast<int>(batch), static_cast<int>(rows),
                                static_cast<int>(block_table.size(1)), static_cast<int>(page_size), block_table.stride(0), p.num_pages,
                                s.partials.data_ptr(), static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                                static_cast<size_t>(s.sync.numel()), stream),
               "paged_reserve");
}

// The pages in use moved to the lowest ids (kl_paged_compact).
void paged_compact(at::Tensor& out_table, at::Tensor& used, at::TensorList caches, const at::Tensor& block_table,
                   const at::Tensor& seq_lens, int64_t page_size) {
  const Pools p = check_pools(caches);
  const int64_t batch = seq_lens.numel();
  check_page_table(out_table, block_table, seq_lens, batch, p.device);
  TORCH_CHECK(page_size > 0 && page_size <= INT32_MAX, "page_size must be positive");
  TORCH_CHECK(used.scalar_type() == at::kInt && used.numel() == 1 && used.device() == p.device, "used is one int32 on the caches' device");
  const c10::cuda::CUDAGuard guard(p.device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  size_t bytes = 0, sync_bytes = 0;
  check_status(kl_paged_compact_workspace_size(p.num_pages, &bytes, &sync_bytes), "paged_compact (workspace)");
  const HeldScratch s = scratch_for(p.device, stream, bytes, sync_bytes);
  const kl_page_pools_t pools = p.c();
  check_status(kl_paged_compact(&pools, out_table.data_ptr<int32_t>(), used.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(),
                                seq_lens.data_ptr<int32_t>(), static_cast<int>(batch), static_cast<int>(block_table.size(1)),
                                static_cast<int>(page_size), block_table.stride(0), p.num_pages, s.partials.data_ptr(),
                                static_cast<size_t>(s.partials.numel()), s.sync.data_ptr(),
                                static_cast<size_t>(s.sync.numel()), stream),
               "paged_compact");
}

// The sync buffers of the current device and stream and of the graphs captured on the device. With pool.mu held.
std::vector<at::Tensor> sync_buffers(ScratchPool& pool, const at::Device& dev, cudaStream_t stream) {
  std::vector<at::Tensor> buffers;
  const auto it = pool.streams.find({dev.index(), stream});
  if (it != pool.streams.end() && it->second.sync.defined()) buffers.push_back(it->second.sync);
  for (const auto& p : pool.graphs) {
    if (p->device != dev.index()) continue;
    for (const Scratch& s : p->grown) buffers.push_back(s.sync);
  }
  return buffers;
}

// Status bits (KL_STATUS_*) left by decode calls on the current device and stream and by the graphs
// captured on the device.
int64_t decode_status(bool clear) {
  const at::Device dev(at::kCUDA, c10::cuda::current_device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  std::vector<at::Tensor> words;
  uint32_t status = 0;
  ScratchPool& pool = scratch_pool();
  const std::unique_lock<std::mutex> launching = launching_on(pool, dev, stream);
  {
    const std::lock_guard<std::mutex> lock(pool.mu);
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    collect_ended_graphs(pool);
    words = sync_buffers(pool, dev, stream);
    uint32_t& gone = pool.spare_status[dev.index()];
    status = gone;
    if (clear) gone = 0;
  }
  for (const at::Tensor& sync : words) {
    uint32_t bits = 0;
    check_status(kl_paged_decode_read_status(sync.data_ptr(), &bits, clear ? 1 : 0, stream), "decode_status");
    if (clear) zero_after_timeout(sync, bits, stream);
    status |= bits;
  }
  return status;
}

// The buffers that decode_status() reads, for tests.
std::vector<at::Tensor> current_sync_buffers() {
  const at::Device dev(at::kCUDA, c10::cuda::current_device());
  ScratchPool& pool = scratch_pool();
  const std::lock_guard<std::mutex> lock(pool.mu);
  return sync_buffers(pool, dev, at::cuda::getCurrentCUDAStream().stream());
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

// The chunked step's functional forms, under the same rule.
at::Tensor rows_of_q(const at::Tensor& q) {
  const bool rows = q.dim() == 3 && q.stride(2) == 1 && (q.stride(1) == q.size(2) || q.size(1) == 1) &&
                    (q.stride(0) >= q.size(1) * q.size(2) || q.size(0) <= 1);
  return rows ? q : q.contiguous();
}

at::Tensor paged_chunk_attention_new(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                     const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& indptr,
                                     double scale, bool causal) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  paged_chunk_attention(out, rows_of_q(q), k_cache, v_cache, block_table, seq_lens, indptr, scale, causal);
  return out;
}

at::Tensor paged_chunk_attention_fp8_new(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                         const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                                         const at::Tensor& seq_lens, const at::Tensor& indptr, double scale, bool causal) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  paged_chunk_attention_fp8(out, rows_of_q(q), k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr, scale, causal);
  return out;
}

at::Tensor paged_chunk_attention_block8_new(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                            const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                                            const at::Tensor& seq_lens, const at::Tensor& indptr, double scale, bool causal) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  paged_chunk_attention_block8(out, rows_of_q(q), k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr, scale, causal);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> paged_reserve_new(const std::vector<at::Tensor>& caches,
                                                                 const at::Tensor& block_table, const at::Tensor& seq_lens,
                                                                 const at::Tensor& new_tokens,
                                                                 const std::optional<at::Tensor>& parents, int64_t page_size) {
  TORCH_CHECK(block_table.dim() == 2, "block_table is [batch, width]");
  const int64_t rows = parents ? parents->numel() : seq_lens.numel();
  at::Tensor table = at::empty({rows, block_table.size(1)}, block_table.options().dtype(at::kInt));
  at::Tensor lens = at::empty({rows}, table.options()), served = at::empty({rows}, table.options().dtype(at::kBool));
  paged_reserve(table, lens, served, caches, block_table, seq_lens, new_tokens, parents, page_size);
  return {table, lens, served};
}

std::tuple<at::Tensor, at::Tensor> paged_compact_new(const std::vector<at::Tensor>& caches, const at::Tensor& block_table,
                                                     const at::Tensor& seq_lens, int64_t page_size) {
  TORCH_CHECK(block_table.dim() == 2, "block_table is [batch, width]");
  at::Tensor table = at::empty({seq_lens.numel(), block_table.size(1)}, block_table.options().dtype(at::kInt));
  at::Tensor used = at::empty({}, table.options());
  paged_compact(table, used, caches, block_table, seq_lens, page_size);
  return {table, used};
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
void noop_append_chunks(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const at::Tensor&) {}
void noop_append_chunks_fp8(at::Tensor&, at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&) {}
void noop_chunk(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                const at::Tensor&, double, bool) {}
void noop_chunk8(at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                 const at::Tensor&, const at::Tensor&, const at::Tensor&, double, bool) {}
void noop_copy_pages(at::TensorList, const at::Tensor&, const at::Tensor&) {}
void noop_reserve(at::Tensor&, at::Tensor&, at::Tensor&, at::TensorList, const at::Tensor&, const at::Tensor&,
                  const at::Tensor&, const std::optional<at::Tensor>&, int64_t) {}
void noop_compact(at::Tensor&, at::Tensor&, at::TensorList, const at::Tensor&, const at::Tensor&, int64_t) {}

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
  m.def(
      "paged_kv_append_chunks(Tensor! k_cache, Tensor! v_cache, Tensor k_new, Tensor v_new, Tensor block_table, "
      "Tensor positions, Tensor indptr) -> ()");
  m.def(
      "paged_kv_append_chunks_fp8(Tensor! k_cache, Tensor! v_cache, Tensor k_new, Tensor v_new, Tensor k_scale, "
      "Tensor v_scale, Tensor block_table, Tensor positions, Tensor indptr) -> ()");
  m.def(
      "paged_chunk_attention(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
      "Tensor seq_lens, Tensor indptr, float scale, bool causal) -> ()");
  m.def(
      "paged_chunk_attention_fp8(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
      "Tensor block_table, Tensor seq_lens, Tensor indptr, float scale, bool causal) -> ()");
  m.def(
      "paged_chunk_attention_block8(Tensor! out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, "
      "Tensor v_scale, Tensor block_table, Tensor seq_lens, Tensor indptr, float scale, bool causal) -> ()");
  m.def("paged_copy_pages(Tensor(a!)[] caches, Tensor src, Tensor dst) -> ()");
  m.def(
      "paged_reserve(Tensor! out_table, Tensor! out_lens, Tensor! served, Tensor(a!)[] caches, Tensor block_table, "
      "Tensor seq_lens, Tensor new_tokens, Tensor? parents, int page_size) -> ()");
  m.def(
      "paged_compact(Tensor! out_table, Tensor! used, Tensor(a!)[] caches, Tensor block_table, Tensor seq_lens, "
      "int page_size) -> ()");
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
  m.impl("paged_kv_append_chunks", &paged_kv_append_chunks);
  m.impl("paged_kv_append_chunks_fp8", &paged_kv_append_chunks_fp8);
  m.impl("paged_chunk_attention", &paged_chunk_attention);
  m.impl("paged_chunk_attention_fp8", &paged_chunk_attention_fp8);
  m.impl("paged_chunk_attention_block8", &paged_chunk_attention_block8);
  m.impl("paged_copy_pages", &paged_copy_pages);
  m.impl("paged_reserve", &paged_reserve);
  m.impl("paged_compact", &paged_compact);
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
  m.impl("paged_kv_append_chunks", &noop_append_chunks);
  m.impl("paged_kv_append_chunks_fp8", &noop_append_chunks_fp8);
  m.impl("paged_chunk_attention", &noop_chunk);
  m.impl("paged_chunk_attention_fp8", &noop_chunk8);
  m.impl("paged_chunk_attention_block8", &noop_chunk8);
  m.impl("paged_copy_pages", &noop_copy_pages);
  m.impl("paged_reserve", &noop_reserve);
  m.impl("paged_compact", &noop_compact);
}

// Importing kernel_lab._C runs the registrations above.
PYBIND11_MODULE(_C, m) {
  m.def("decode_status", &decode_status, pybind11::arg("clear") = false,
        "Status bits left by calls on the current device and stream and by the graphs captured on the device.");
  m.def("current_sync_buffers", &current_sync_buffers, "The scratch that decode_status() reads and clears, for tests.");
  m.def("direct", &direct);
  m.def("rms_norm_fp8", &rms_norm_fp8_new);
  m.def("fused_add_rms_norm_fp8", &fused_add_rms_norm_fp8_new);
  m.def("paged_kv_append_block8", &paged_kv_append_block8);
  m.def("paged_decode_attention_block8", &paged_decode_attention_block8_new);
  m.def("paged_block_select", &paged_block_select_new);
  m.def("paged_kv_append_chunks", &paged_kv_append_chunks);
  m.def("paged_kv_append_chunks_fp8", &paged_kv_append_chunks_fp8);
  m.def("paged_chunk_attention", &paged_chunk_attention_new);
  m.def("paged_chunk_attention_fp8", &paged_chunk_attention_fp8_new);
  m.def("paged_chunk_attention_block8", &paged_chunk_attention_block8_new);
  m.def("paged_copy_pages", [](const std::vector<at::Tensor>& caches, const at::Tensor& src, const at::Tensor& dst) {
    paged_copy_pages(caches, src, dst);
  });
  m.def("paged_reserve", &paged_reserve_new);
  m.def("paged_compact", &paged_compact_new);
  m.attr("version") = kl_version();
}
