// Host side of the uncompressed paged cache (lc_paged_*) and of beam
// selection (lc_beam_*): argument checks, workspaces, stream order.
#include <algorithm>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "paged.h"

using namespace lc;

namespace {

int element_size(int32_t dtype) { return dtype == LC_F32 ? 4 : 2; }

void check_dtype(int32_t dtype, const char* what) {
  LC_REQUIRE(dtype == LC_F32 || dtype == LC_BF16 || dtype == LC_F16, LC_ERR_INVALID,
             std::string(what) + ": unknown dtype " + std::to_string(dtype));
}

// Memory that kernels on `device` may read: that device's own, or managed.
void check_device(const void* p, int device, const char* what, size_t align) {
  LC_REQUIRE(p, LC_ERR_INVALID, std::string(what) + ": null pointer");
  cudaPointerAttributes at;
  const cudaError_t e = cudaPointerGetAttributes(&at, p);
  if (e != cudaSuccess) cudaGetLastError();
  LC_REQUIRE(e == cudaSuccess && (at.type == cudaMemoryTypeManaged ||
                                  (at.type == cudaMemoryTypeDevice && at.device == device)),
             LC_ERR_INVALID, std::string(what) + ": not memory of the handle's device");
  LC_REQUIRE((reinterpret_cast<uintptr_t>(p) & (align - 1)) == 0, LC_ERR_INVALID,
             std::string(what) + ": pointer not aligned to its elements");
}

bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

// An output may be its input, not a part of it.
void check_in_place(const void* in, const void* out, size_t bytes, const char* what) {
  LC_REQUIRE(in == out || !overlap(in, bytes, out, bytes), LC_ERR_INVALID,
             std::string(what) + ": output overlaps input, but is not the same");
}

// The calling thread's device, put back at the end of a call.
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(int device) {
    LC_CUDA(cudaGetDevice(&before));
    if (before != device) LC_CUDA(cudaSetDevice(device));
    now = device;
  }
  ~DeviceScope() {
    if (before >= 0 && before != now) cudaSetDevice(before);
  }
  int now = -1;
};

// Workspaces come from a memory pool of the library's own for each device, which
// keeps up to kKeptBytes of what is freed: a handle made for every request pays
// for its memory once a process, not once a handle.
constexpr uint64_t kKeptBytes = 256ull << 20;
cudaMemPool_t workspace_pool(int device) {
  static std::mutex mu;
  static std::map<int, cudaMemPool_t> pools;
  std::lock_guard<std::mutex> lock(mu);
  cudaMemPool_t& pool = pools[device];
  if (!pool) {
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = device;
    LC_CUDA(cudaMemPoolCreate(&pool, &props));
    uint64_t keep = kKeptBytes;
    LC_CUDA(cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep));
  }
  return pool;
}

bool capturing(cudaStream_t s) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  LC_CUDA(cudaStreamIsCapturing(s, &capture));
  return capture != cudaStreamCaptureStatusNone;
}

// A device buffer that grows, in the order of the handle's calls. One that a
// captured call was given is kept when it is outgrown, until the handle is
// destroyed: the graph has its address.
struct Workspace {
  void* p = nullptr;
  size_t bytes = 0;
  bool in_graph = false;
  std::vector<void*> outgrown;
  ~Workspace() {  // the device is idle: the handle is being destroyed
    if (p) cudaFreeAsync(p, cudaStreamLegacy);
    for (void* x : outgrown) cudaFreeAsync(x, cudaStreamLegacy);
  }
  void* get(size_t need, int device, cudaStream_t s, bool captured, bool zeroed = false) {
    if (need > bytes) {
      LC_REQUIRE(!captured, LC_ERR_STATE, "the first call of this size allocates: make it outside the capture");
      if (p && in_graph)
        outgrown.push_back(p);
      else if (p)
        LC_CUDA(cudaFreeAsync(p, s));
      p = nullptr;
      bytes = 0;
      in_graph = false;
      const cudaError_t e = cudaMallocFromPoolAsync(&p, need, workspace_pool(device), s);
      if (e != cudaSuccess) {
        cudaGetLastError();
        p = nullptr;
        LC_THROW(LC_ERR_NOMEM, "workspace of " + std::to_string(need) + " bytes: " + cudaGetErrorString(e));
      }
      bytes = need;
      if (zeroed) LC_CUDA(cudaMemsetAsync(p, 0, need, s));
    }
    in_graph |= captured;
    return p;
  }
};

// Status words in mapped host memory, a cache line a handle, from pages that are kept.
struct StatusWords {
  std::mutex mu;
  std::vector<int32_t*> free;
  int32_t* take() {
    std::lock_guard<std::mutex> lock(mu);
    if (free.empty()) {
      constexpr int kLines = 256;
      int32_t* page = nullptr;
      LC_CUDA(cudaHostAlloc(reinterpret_cast<void**>(&page), kLines * 64, cudaHostAllocMapped | cudaHostAllocPortable));
      for (int i = 0; i < kLines; ++i) free.push_back(page + 16 * i);
    }
    int32_t* w = free.back();
    free.pop_back();
    std::fill(w, w + kStatusBits, 0);
    return w;
  }
  void give(int32_t* w) {
    std::lock_guard<std::mutex> lock(mu);
    free.push_back(w);
  }
};
StatusWords& status_words() {
  static auto* words = new StatusWords;  // outlives every handle
  return *words;
}

// Calls of one handle share its workspace and write its pools: a call on another
// stream than the last one's waits for that call's event. The event is recorded
// behind every call (0.4 us of its issue; kernels overlap across it as
// before), so that the last one's stream is not touched again: it may have been
// destroyed since, or be in capture, which a later record would join. A stream
// that is being captured takes no part: a graph may not wait for work outside
// it, so its replays are the caller's to order.
struct Order {
  cudaStream_t own = nullptr;
  unsigned long long last = 0;  // the last call's stream by its id, which no other stream is given
  cudaEvent_t ev = nullptr;     // null before the first call
  ~Order() {
    if (ev) cudaEventDestroy(ev);
    if (own) cudaStreamDestroy(own);
  }
};

// One call's place in the order, from its first launch to its last.
struct Turn {
  Order& order;
  cudaStream_t s;
  bool captured = false;
  Turn(Order& o, void* stream) : order(o) {
    if (!stream && !o.own) LC_CUDA(cudaStreamCreateWithFlags(&o.own, cudaStreamNonBlocking));
    s = stream ? static_cast<cudaStream_t>(stream) : o.own;
    unsigned long long id = s == o.own ? ~0ull : ~1ull;  // these two are no one's to capture or destroy
    if (s != o.own && s != cudaStreamLegacy) {
      captured = capturing(s);
      if (captured) return;
      LC_CUDA(cudaStreamGetId(s, &id));
    }
    if (!o.ev)
      LC_CUDA(cudaEventCreateWithFlags(&o.ev, cudaEventDisableTiming));
    else if (o.last != id)
      LC_CUDA(cudaStreamWaitEvent(s, o.ev, 0));
    o.last = id;
  }
  ~Turn() {
    if (!captured) cudaEventRecord(order.ev, s);
  }
  Turn(const Turn&) = delete;
  Turn& operator=(const Turn&) = delete;
};

// A handle's status words and their address on the device.
struct Status {
  int32_t* words = nullptr;
  int32_t* on_device = nullptr;
  ~Status() {
    if (words) status_words().give(words);
  }
  void make() {
    words = status_words().take();
    LC_CUDA(cudaHostGetDevicePointer(reinterpret_cast<void**>(&on_device), words, 0));
  }
  void check() const {
    const int code = status_code(words);
    LC_REQUIRE(code == LC_OK, code, status_message(code));
  }
};

int sm_count(int device) {
  int n = 0;
  LC_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
  return n;
}

}  // namespace

struct lc_paged {
  lc_paged_config cfg{};
  PagedView view{};
  PagedMaps maps{};
  int sms = 0, esize = 0;
  Order order;
  Workspace part, counters, scores, evict;
  Status status;

  PagedView call(const int32_t* tables, int32_t width, const int32_t* lens, int32_t rows) const {
    LC_REQUIRE(rows >= 1 && rows <= cfg.max_seqs, LC_ERR_INVALID,
               "n_seqs " + std::to_string(rows) + " outside 1.." + std::to_string(cfg.max_seqs));
    LC_REQUIRE(width >= 1 && width <= cfg.max_pages_per_seq, LC_ERR_INVALID,
               "table width " + std::to_string(width) + " outside 1.." + std::to_string(cfg.max_pages_per_seq));
    check_device(tables, cfg.device, "tables", 4);
    check_device(lens, cfg.device, "lens", 4);
    PagedView v = view;
    v.tables = tables;
    v.lens = lens;
    v.width = width;
    return v;
  }
  void check_layer(int32_t layer) const {
    LC_REQUIRE(layer >= 0 && layer < cfg.n_layers, LC_ERR_INVALID, "layer out of range");
  }
};

struct lc_beam {
  int32_t n_groups = 0, n_beams = 0, n_out = 0, device = 0, sms = 0;
  int64_t vocab = 0;
  size_t lists = 0;
  Order order;
  Workspace ws;
  Status status;
};

extern "C" {

int lc_paged_create(const lc_paged_config* config, void* k_pages, void* v_pages, lc_paged** out) {
  return abi_guard([&] {
    LC_REQUIRE(out, LC_ERR_INVALID, "null out");
    *out = nullptr;
    LC_REQUIRE(config, LC_ERR_INVALID, "null config");
    lc_paged_config c = *config;
    check_dtype(c.dtype, "pool");
    LC_REQUIRE(c.n_layers >= 1 && c.n_layers <= 65535 && c.n_kv_heads >= 1 && c.n_kv_heads <= 1024, LC_ERR_INVALID,
               "n_layers must be 1..65535 and n_kv_heads 1..1024");
    LC_REQUIRE(c.head_dim >= 1 && c.head_dim <= kPagedMaxDim, LC_ERR_INVALID,
               "head_dim must be 1.." + std::to_string(kPagedMaxDim));
    LC_REQUIRE(c.page_tokens >= 1 && c.page_tokens <= 4096, LC_ERR_INVALID, "page_tokens must be 1..4096");
    LC_REQUIRE(c.n_pages >= 1 && c.n_pages <= INT32_MAX, LC_ERR_INVALID, "n_pages must be 1..2^31-1");
    LC_REQUIRE(c.max_seqs >= 1 && c.max_seqs <= kPagedMaxSeqs, LC_ERR_INVALID,
               "max_seqs must be 1.." + std::to_string(kPagedMaxSeqs));
    LC_REQUIRE(c.max_pages_per_seq >= 1 && (int64_t)c.max_pages_per_seq * c.page_tokens < (1ll << 30), LC_ERR_INVALID,
               "a sequence must hold 1..2^30-1 slots");
    LC_REQUIRE(c.max_q_heads >= c.n_kv_heads && c.max_q_heads <= 4096, LC_ERR_INVALID,
               "max_q_heads must be n_kv_heads..4096");
    LC_REQUIRE(c.reserved == 0, LC_ERR_INVALID, "reserved must be 0");
    if (!c.layer_stride && !c.page_stride && !c.head_stride && !c.token_stride) {
      c.token_stride = c.head_dim;
      c.head_stride = c.token_stride * c.page_tokens;
      c.page_stride = c.head_stride * c.n_kv_heads;
      c.layer_stride = c.page_stride * c.n_pages;
    }
    // rows must not overlap: the writing calls would race
    std::pair<int64_t, int64_t> dims[4] = {{c.layer_stride, c.n_layers},
                                           {c.page_stride, c.n_pages},
                                           {c.head_stride, c.n_kv_heads},
                                           {c.token_stride, c.page_tokens}};
    std::sort(dims, dims + 4);
    int64_t span = c.head_dim;
    for (const auto& [stride, n] : dims) {
      if (n == 1) continue;
      LC_REQUIRE(stride >= span, LC_ERR_INVALID, "pool strides overlap");
      LC_REQUIRE(stride <= (1ll << 60) / n, LC_ERR_INVALID, "pool strides too large");
      span = stride * (n - 1) + span;
    }
    DeviceScope scope(c.device);
    check_device(k_pages, c.device, "k_pages", element_size(c.dtype));
    check_device(v_pages, c.device, "v_pages", element_size(c.dtype));
    auto p = std::make_unique<lc_paged>();
    p->cfg = c;
    p->esize = element_size(c.dtype);
    p->sms = sm_count(c.device);
    p->status.make();
    p->view.k = k_pages;
    p->view.v = v_pages;
    p->view.layer = c.n_layers == 1 ? 0 : c.layer_stride;
    p->view.page = c.n_pages == 1 ? 0 : c.page_stride;
    p->view.head = c.n_kv_heads == 1 ? 0 : c.head_stride;
    p->view.token = c.page_tokens == 1 ? 0 : c.token_stride;
    p->view.n_layers = c.n_layers;
    p->view.hkv = c.n_kv_heads;
    p->view.d = c.head_dim;
    p->view.page_tokens = c.page_tokens;
    p->view.n_pages = c.n_pages;
    p->view.status = p->status.on_device;
    p->maps = make_paged_maps(p->view, c.dtype);
    *out = p.release();
  });
}

void lc_paged_destroy(lc_paged* p) {
  if (!p) return;
  int before = -1;
  cudaGetDevice(&before);
  cudaSetDevice(p->cfg.device);
  cudaDeviceSynchronize();
  const int device = p->cfg.device;
  delete p;
  if (before >= 0 && before != device) cudaSetDevice(before);
}

int lc_paged_status(const lc_paged* p) {
  return abi_guard([&] {
    LC_REQUIRE(p, LC_ERR_INVALID, "null handle");
    p->status.check();
  });
}

int lc_paged_append(lc_paged* p, int32_t layer, int32_t n_seqs, const int32_t* tables, int32_t width,
                    const int32_t* lens, const void* keys, const void* values, int32_t dtype, int64_t n_tokens,
                    int32_t* pos, int64_t pos_stride, const int32_t* pos0, void* stream) {
  return abi_guard([&] {
    LC_REQUIRE(p, LC_ERR_INVALID, "null handle");
    check_dtype(dtype, "keys");
    p->check_layer(layer);
    LC_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 30), LC_ERR_INVALID, "n_tokens must be 0..2^30-1");
    DeviceScope scope(p->cfg.device);
    PagedAppendArgs a{};
    a.c = p->call(tables, width, lens, n_seqs);
    if (n_tokens == 0) return;
    check_device(keys, p->cfg.device, "keys", element_size(dtype));
    check_device(values, p->cfg.device, "values", element_size(dtype));
    if (pos) {
      check_device(pos, p->cfg.device, "pos", 4);
      check_device(pos0, p->cfg.device, "pos0", 4);
      LC_REQUIRE(pos_stride >= (int64_t)width * p->cfg.page_tokens, LC_ERR_INVALID, "pos rows shorter than the table");
    }
    a.keys = keys;
    a.values = values;
    a.dtype = dtype;
    a.pool_dtype = p->cfg.dtype;
    a.layer = layer;
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.pos = pos;
    a.pos0 = pos0;
    a.pos_stride = pos_stride;
    const Turn turn(p->order, stream);
    launch_paged_append(a, p->sms, turn.s);
  });
}

static void paged_attn(lc_paged* p, int32_t layer, int32_t n_seqs, const int32_t* tables, int32_t width,
                       const int32_t* lens, const void* q, int32_t q_dtype, int32_t n_q_heads, float scale,
                       int32_t window, void* out, int32_t out_dtype, const float* acc_in, float* acc_out,
                       int64_t acc_stride, float decay, void* stream) {
  LC_REQUIRE(p, LC_ERR_INVALID, "null handle");
  check_dtype(q_dtype, "q");
  check_dtype(out_dtype, "out");
  p->check_layer(layer);
  LC_REQUIRE(n_q_heads >= 1 && n_q_heads <= p->cfg.max_q_heads && n_q_heads % p->cfg.n_kv_heads == 0, LC_ERR_INVALID,
             "n_q_heads must be a multiple of n_kv_heads and at most max_q_heads");
  LC_REQUIRE(window >= 0, LC_ERR_INVALID, "window must be >= 0");
  LC_REQUIRE(scale == scale && scale - scale == 0.f, LC_ERR_INVALID, "scale must be finite");
  DeviceScope scope(p->cfg.device);
  PagedAttnArgs a{};
  a.c = p->call(tables, width, lens, n_seqs);
  check_device(q, p->cfg.device, "q", element_size(q_dtype));
  check_device(out, p->cfg.device, "out", element_size(out_dtype));
  const size_t values = (size_t)n_seqs * n_q_heads * p->cfg.head_dim;
  const size_t out_bytes = values * element_size(out_dtype);
  LC_REQUIRE(!overlap(q, values * element_size(q_dtype), out, out_bytes), LC_ERR_INVALID, "out overlaps q");
  a.q = q;
  a.out = out;
  a.q_dtype = q_dtype;
  a.out_dtype = out_dtype;
  a.n_seqs = n_seqs;
  a.group = n_q_heads / p->cfg.n_kv_heads;
  a.layer = layer;
  a.window = window;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  const int64_t cap = (int64_t)width * p->cfg.page_tokens;
  const Turn turn(p->order, stream);
  const cudaStream_t s = turn.s;
  a.part = static_cast<float*>(p->part.get((size_t)paged_part_floats(p->sms) * 4, p->cfg.device, s, turn.captured));
  a.counters = static_cast<int32_t*>(p->counters.get((size_t)p->cfg.max_seqs * p->cfg.max_q_heads * 4, p->cfg.device, s,
                                                     turn.captured, true));
  if (acc_out) {
    check_device(acc_in, p->cfg.device, "acc_in", 4);
    check_device(acc_out, p->cfg.device, "acc_out", 4);
    LC_REQUIRE(acc_stride >= cap, LC_ERR_INVALID, "acc rows shorter than the table");
    const size_t acc_bytes = (size_t)n_seqs * p->cfg.n_kv_heads * acc_stride * 4;
    check_in_place(acc_in, acc_out, acc_bytes, "acc");
    LC_REQUIRE(!overlap(out, out_bytes, acc_in, acc_bytes) && !overlap(out, out_bytes, acc_out, acc_bytes) &&
                   !overlap(q, values * element_size(q_dtype), acc_out, acc_bytes),
               LC_ERR_INVALID, "acc overlaps q or out");
    const size_t rows = (size_t)n_seqs * n_q_heads;
    a.score_tokens = cap;
    a.scores =
        static_cast<float*>(p->scores.get((rows * cap + 2 * rows) * 4, p->cfg.device, s, turn.captured));
    a.stats = a.scores + rows * cap;
  }
  launch_paged_attn(a, p->maps, p->cfg.dtype, p->cfg.device, p->sms, s);
  if (acc_out) {
    PagedWeightArgs w{};
    w.scores = a.scores;
    w.stats = a.stats;
    w.acc_in = acc_in;
    w.acc_out = acc_out;
    w.lens = lens;
    w.score_tokens = cap;
    w.acc_stride = acc_stride;
    w.n_seqs = n_seqs;
    w.hkv = p->cfg.n_kv_heads;
    w.group = a.group;
    w.window = window;
    w.cap = (int32_t)cap;
    w.decay = decay;
    launch_paged_weights(w, s);
  }
}

int lc_paged_attn(lc_paged* p, int32_t layer, int32_t n_seqs, const int32_t* tables, int32_t width,
                  const int32_t* lens, const void* q, int32_t q_dtype, int32_t n_q_heads, float scale, int32_t window,
                  void* out, int32_t out_dtype, void* stream) {
  return abi_guard([&] {
    paged_attn(p, layer, n_seqs, tables, width, lens, q, q_dtype, n_q_heads, scale, window, out, out_dtype, nullptr,
               nullptr, 0, 0.f, stream);
  });
}

int lc_paged_attn_weights(lc_paged* p, int32_t layer, int32_t n_seqs, const int32_t* tables, int32_t width,
                          const int32_t* lens, const void* q, int32_t q_dtype, int32_t n_q_heads, float scale,
                          int32_t window, void* out, int32_t out_dtype, const float* acc_in, float* acc_out,
                          int64_t acc_stride, float decay, void* stream) {
  return abi_guard([&] {
    LC_REQUIRE(acc_in && acc_out, LC_ERR_INVALID, "acc_in and acc_out must be given");
    LC_REQUIRE(decay >= 0.f && decay <= 1.f, LC_ERR_INVALID, "decay must be in [0, 1]");
    paged_attn(p, layer, n_seqs, tables, width, lens, q, q_dtype, n_q_heads, scale, window, out, out_dtype, acc_in,
               acc_out, acc_stride, decay, stream);
  });
}

int lc_paged_evict(lc_paged* p, int32_t layer, int32_t n_seqs, const int32_t* tables, int32_t width,
                   const int32_t* lens, int32_t budget, int32_t n_sink, int32_t n_recent, const float* acc_in,
                   const int32_t* pos_in, float* acc_out, int32_t* pos_out, int64_t stride, void* stream) {
  return abi_guard([&] {
    LC_REQUIRE(p, LC_ERR_INVALID, "null handle");
    p->check_layer(layer);
    LC_REQUIRE(budget >= 1 && n_sink >= 0 && n_recent >= 0 && (int64_t)n_sink + n_recent <= budget, LC_ERR_INVALID,
               "budget must be >= 1 and hold n_sink + n_recent");
    DeviceScope scope(p->cfg.device);
    PagedEvictArgs a{};
    a.c = p->call(tables, width, lens, n_seqs);
    check_device(acc_in, p->cfg.device, "acc_in", 4);
    check_device(pos_in, p->cfg.device, "pos_in", 4);
    check_device(acc_out, p->cfg.device, "acc_out", 4);
    check_device(pos_out, p->cfg.device, "pos_out", 4);
    const int64_t cap = (int64_t)width * p->cfg.page_tokens;
    LC_REQUIRE(stride >= cap, LC_ERR_INVALID, "acc and pos rows shorter than the table");
    const size_t row_bytes = (size_t)n_seqs * p->cfg.n_kv_heads * stride * 4;
    check_in_place(acc_in, acc_out, row_bytes, "acc");
    check_in_place(pos_in, pos_out, row_bytes, "pos");
    LC_REQUIRE(!overlap(acc_out, row_bytes, pos_out, row_bytes), LC_ERR_INVALID, "acc_out overlaps pos_out");
    LC_REQUIRE(!overlap(acc_out, row_bytes, pos_in, row_bytes) && !overlap(pos_out, row_bytes, acc_in, row_bytes),
               LC_ERR_INVALID, "an output overlaps the other's input");
    a.layer = layer;
    a.n_seqs = n_seqs;
    a.esize = p->esize;
    a.budget = budget;
    a.n_sink = n_sink;
    a.n_recent = n_recent;
    a.stride = stride;
    a.acc_in = acc_in;
    a.pos_in = pos_in;
    a.acc_out = acc_out;
    a.pos_out = pos_out;
    // at most min(budget, cap - budget) slots move in a row
    const int64_t rows = (int64_t)n_seqs * p->cfg.n_kv_heads;
    a.list_cap = std::max<int64_t>(1, std::min<int64_t>(budget, cap - budget));
    const int cl = paged_evict_cluster(cap, (int)rows, p->sms);
    const int64_t keys = paged_evict_keys_in_smem(cap, cl) ? 0 : rows * stride;
    const Turn turn(p->order, stream);
    const cudaStream_t s = turn.s;
    int32_t* ws = static_cast<int32_t*>(
        p->evict.get((size_t)(rows * (4 * a.list_cap + 1) + keys) * 4, p->cfg.device, s, turn.captured));
    a.list = ws;
    a.pairs = ws + rows * 4 * a.list_cap;
    a.keys = reinterpret_cast<uint32_t*>(a.pairs + rows);
    launch_paged_evict(a, p->cfg.device, p->sms, s);
  });
}

int lc_paged_reorder(lc_paged* p, int32_t n_groups, int32_t n_beams, const int32_t* tables, int32_t width,
                     const int32_t* lens, const int32_t* parents, int32_t* tables_out, void* stream) {
  return abi_guard([&] {
    LC_REQUIRE(p, LC_ERR_INVALID, "null handle");
    LC_REQUIRE(n_groups >= 1 && n_beams >= 1 && n_beams <= kBeamMaxBeams, LC_ERR_INVALID,
               "n_groups must be >= 1 and n_beams 1.." + std::to_string(kBeamMaxBeams));
    LC_REQUIRE((int64_t)n_groups * n_beams <= p->cfg.max_seqs, LC_ERR_INVALID, "more rows than max_seqs");
    DeviceScope scope(p->cfg.device);
    PagedReorderArgs a{};
    a.c = p->call(tables, width, lens, n_groups * n_beams);
    check_device(parents, p->cfg.device, "parents", 4);
    check_device(tables_out, p->cfg.device, "tables_out", 4);
    const size_t bytes = (size_t)n_groups * n_beams * width * 4;
    LC_REQUIRE(!overlap(tables, bytes, tables_out, bytes) &&
                   !overlap(parents, (size_t)n_groups * n_beams * 4, tables_out, bytes) &&
                   !overlap(lens, (size_t)n_groups * 4, tables_out, bytes),
               LC_ERR_INVALID, "tables_out overlaps an input");
    a.n_groups = n_groups;
    a.n_beams = n_beams;
    a.esize = p->esize;
    a.parents = parents;
    a.tables_out = tables_out;
    const Turn turn(p->order, stream);
    launch_paged_reorder(a, p->sms, turn.s);
  });
}

int lc_beam_create(int32_t n_groups, int32_t n_beams, int64_t vocab, int32_t n_out, int32_t device, lc_beam** out) {
  return abi_guard([&] {
    LC_REQUIRE(out, LC_ERR_INVALID, "null out");
    *out = nullptr;
    LC_REQUIRE(n_groups >= 1 && n_beams >= 1 && n_beams <= kBeamMaxBeams && (int64_t)n_groups * n_beams <= 65535,
               LC_ERR_INVALID, "n_beams must be 1.." + std::to_string(kBeamMaxBeams) + " and the rows at most 65535");
    LC_REQUIRE(n_out >= 1 && n_out <= kBeamMaxOut, LC_ERR_INVALID, "n_out must be 1.." + std::to_string(kBeamMaxOut));
    LC_REQUIRE(vocab >= 1 && vocab <= (1 << 24), LC_ERR_INVALID, "vocab must be 1..2^24");
    const int64_t slices = (vocab + beam_slice(LC_F32) - 1) / beam_slice(LC_F32);
    DeviceScope scope(device);
    auto b = std::make_unique<lc_beam>();
    b->n_groups = n_groups;
    b->n_beams = n_beams;
    b->n_out = n_out;
    b->device = device;
    b->vocab = vocab;
    b->sms = sm_count(device);
    // a row has at most one part a slice, and a group no more candidates than one merge takes
    const size_t rows = (size_t)n_groups * n_beams;
    const size_t lists = rows * std::min<int64_t>(slices, std::max(1, kBeamMaxMerge / (n_beams * n_out)));
    b->lists = lists;
    b->status.make();
    *out = b.release();
  });
}

void lc_beam_destroy(lc_beam* b) {
  if (!b) return;
  int before = -1;
  cudaGetDevice(&before);
  const int device = b->device;
  cudaSetDevice(device);
  cudaDeviceSynchronize();
  delete b;
  if (before >= 0 && before != device) cudaSetDevice(before);
}

int lc_beam_status(const lc_beam* b) {
  return abi_guard([&] {
    LC_REQUIRE(b, LC_ERR_INVALID, "null handle");
    b->status.check();
  });
}

int lc_beam_select(lc_beam* b, int32_t n_groups, const void* logits, int32_t dtype, int64_t row_stride,
                   const float* scores, const uint8_t* finished, int32_t eos, int32_t pad, float* scores_out,
                   int32_t* parents, int32_t* tokens, uint8_t* finished_out, void* stream) {
  return abi_guard([&] {
    LC_REQUIRE(b, LC_ERR_INVALID, "null handle");
    check_dtype(dtype, "logits");
    LC_REQUIRE(n_groups >= 1 && n_groups <= b->n_groups, LC_ERR_INVALID,
               "n_groups outside 1.." + std::to_string(b->n_groups));
    LC_REQUIRE(row_stride >= b->vocab && row_stride < (1ll << 40), LC_ERR_INVALID, "row_stride shorter than vocab");
    LC_REQUIRE(pad >= 0 && pad < b->vocab, LC_ERR_INVALID, "pad outside the vocabulary");
    DeviceScope scope(b->device);
    check_device(logits, b->device, "logits", element_size(dtype));
    check_device(scores, b->device, "scores", 4);
    if (finished) check_device(finished, b->device, "finished", 1);
    check_device(scores_out, b->device, "scores_out", 4);
    check_device(parents, b->device, "parents", 4);
    check_device(tokens, b->device, "tokens", 4);
    check_device(finished_out, b->device, "finished_out", 1);
    const size_t in = (size_t)n_groups * b->n_beams, out = (size_t)n_groups * b->n_out;
    const std::pair<const void*, size_t> ins[3] = {
        {logits, ((in - 1) * row_stride + b->vocab) * element_size(dtype)}, {scores, in * 4}, {finished, in}};
    const std::pair<const void*, size_t> outs[4] = {
        {scores_out, out * 4}, {parents, out * 4}, {tokens, out * 4}, {finished_out, out}};
    for (int o = 0; o < 4; ++o) {
      for (const auto& [p, bytes] : ins)
        LC_REQUIRE(!p || !overlap(p, bytes, outs[o].first, outs[o].second), LC_ERR_INVALID, "outputs overlap inputs");
      for (int other = 0; other < o; ++other)
        LC_REQUIRE(!overlap(outs[other].first, outs[other].second, outs[o].first, outs[o].second), LC_ERR_INVALID,
                   "outputs overlap each other");
    }
    const Turn turn(b->order, stream);
    const cudaStream_t s = turn.s;
    const size_t keys = b->lists * b->n_out;
    uint8_t* w = static_cast<uint8_t*>(
        b->ws.get(keys * 8 + (4 * b->lists + b->n_groups) * 4, b->device, s, turn.captured, true));
    BeamArgs a{};
    a.slice_key = reinterpret_cast<uint64_t*>(w);
    a.slice_stats = reinterpret_cast<float*>(a.slice_key + keys);
    a.slice_next = a.slice_stats + 2 * b->lists;
    a.counters = reinterpret_cast<int32_t*>(a.slice_next + 2 * b->lists);
    a.logits = logits;
    a.dtype = dtype;
    a.row_stride = row_stride;
    a.n_groups = n_groups;
    a.n_beams = b->n_beams;
    a.n_out = b->n_out;
    a.vocab = (int32_t)b->vocab;
    a.slice = beam_slice(dtype);
    a.slices = (int32_t)((b->vocab + a.slice - 1) / a.slice);
    a.scores = scores;
    a.finished = finished;
    a.eos = eos;
    a.pad = pad;
    a.scores_out = scores_out;
    a.parents = parents;
    a.tokens = tokens;
    a.finished_out = finished_out;
    a.status = b->status.on_device;
    launch_beam(a, b->device, b->sms, s);
  });
}

}  // extern "C"
