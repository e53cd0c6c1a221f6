// extern "C" surface of the engine; see include/cuhnsw_b200.h for the contract.
#include <exception>
#include <new>

#include "../../include/cuhnsw_b200.h"
#include "engine.h"
#include "replicas.h"
#include "table.h"

struct cuhnsw_handle {
  hnsw::Engine engine;         // the index on the first (or only) GPU
  hnsw::ReplicaSet replicas;   // copies on the other GPUs of the option `devices`
  std::string fatal;
};

namespace {
template <class F>
int guarded(cuhnsw_handle* h, F f) {
  if (!h) return CUHNSW_INVALID_ARGUMENT;
  h->fatal.clear();  // the text of an earlier exception must not outlive the call that raised it
  try {
    return f(h->engine);
  } catch (const std::bad_alloc&) {
    h->fatal = "out of host memory";
    return CUHNSW_OUT_OF_MEMORY;
  } catch (const std::exception& e) {
    h->fatal = e.what();
  } catch (...) {
    h->fatal = "unknown failure";
  }
  return CUHNSW_INTERNAL_ERROR;
}
int null_argument(cuhnsw_handle* h, const char* what) {
  if (h) h->fatal = std::string("null pointer: ") + what;
  return CUHNSW_INVALID_ARGUMENT;
}
}  // namespace

extern "C" {

cuhnsw_handle* cuhnsw_create(void) {
  try {
    return new cuhnsw_handle();
  } catch (...) {
    return nullptr;
  }
}
void cuhnsw_destroy(cuhnsw_handle* h) { delete h; }
const char* cuhnsw_last_error(const cuhnsw_handle* h) {
  if (!h) return "null handle";
  return h->fatal.empty() ? h->engine.last_error() : h->fatal.c_str();
}
int cuhnsw_init(cuhnsw_handle* h, const char* opt_path) {
  return guarded(h, [&](hnsw::Engine& e) {
    int rc = e.Init(opt_path);
    if (rc == hnsw::kOk) rc = h->replicas.Configure(e, opt_path, &h->fatal);
    return rc;
  });
}
int cuhnsw_set_data(cuhnsw_handle* h, const float* data, int64_t num_data, int32_t num_dims) {
  return guarded(h, [&](hnsw::Engine& e) {
    h->replicas.Invalidate();
    return e.SetData(data, num_data, num_dims);
  });
}
int cuhnsw_set_random_levels(cuhnsw_handle* h, const int32_t* levels) {
  return guarded(h, [&](hnsw::Engine& e) {
    h->replicas.Invalidate();
    return e.SetRandomLevels(levels);
  });
}
int cuhnsw_build_graph(cuhnsw_handle* h) {
  return guarded(h, [&](hnsw::Engine& e) {
    h->replicas.Invalidate();
    int rc = e.BuildGraph();
    if (rc == hnsw::kOk && h->replicas.active()) rc = h->replicas.Sync(e, &h->fatal);
    return rc;
  });
}
int cuhnsw_save_index(cuhnsw_handle* h, const char* fpath) {
  return guarded(h, [&](hnsw::Engine& e) { return e.SaveIndex(fpath); });
}
int cuhnsw_load_index(cuhnsw_handle* h, const char* fpath) {
  return guarded(h, [&](hnsw::Engine& e) {
    h->replicas.Invalidate();
    int rc = e.LoadIndex(fpath);
    if (rc == hnsw::kOk && h->replicas.active()) rc = h->replicas.Sync(e, &h->fatal);
    return rc;
  });
}
int cuhnsw_search_knn(cuhnsw_handle* h, const float* qdata, int64_t num_queries, int32_t topk, int32_t ef_search,
                      int32_t* nns, float* distances, int32_t* found_cnt) {
  return guarded(h, [&](hnsw::Engine& e) {
    if (h->replicas.active() && e.has_graph() && num_queries > 0 && qdata && nns && distances && found_cnt)
      return h->replicas.Search(e, qdata, num_queries, topk, ef_search, nns, distances, found_cnt, &h->fatal);
    return e.SearchGraph(qdata, num_queries, topk, ef_search, nns, distances, found_cnt);
  });
}
int cuhnsw_search_knn_device(cuhnsw_handle* h, const float* d_qdata, int64_t num_queries, int32_t topk,
                             int32_t ef_search, int32_t* d_nns, float* d_distances, int32_t* d_found_cnt) {
  return guarded(h, [&](hnsw::Engine& e) {
    return e.SearchGraphDevice(d_qdata, num_queries, topk, ef_search, d_nns, d_distances, d_found_cnt);
  });
}
int cuhnsw_search_knn_async(cuhnsw_handle* h, const float* qdata, int64_t num_queries, int32_t topk, int32_t ef_search,
                            int32_t* nns, float* distances, int32_t* found_cnt) {
  return guarded(h, [&](hnsw::Engine& e) {
    return e.SearchGraphAsync(qdata, num_queries, topk, ef_search, nns, distances, found_cnt);
  });
}
namespace {
// A call on another replica makes that replica's GPU the thread's current device; the caller (who may be in the
// middle of its own CUDA work) gets its device back.
struct DeviceRestore {
  int before = -1;
  DeviceRestore() {
    if (cudaGetDevice(&before) != cudaSuccess) {
      cudaGetLastError();
      before = -1;
    }
  }
  ~DeviceRestore() {
    if (before >= 0) cudaSetDevice(before);
  }
};
}  // namespace
int cuhnsw_replica_count(const cuhnsw_handle* h) { return h ? h->replicas.count() : 0; }
int cuhnsw_stream_create_on(cuhnsw_handle* h, int32_t replica, void** out_stream) {
  return guarded(h, [&](hnsw::Engine& e) {
    int rc = hnsw::kOk;
    hnsw::Engine* r = h->replicas.Fresh(e, replica, &rc, &h->fatal);
    if (!r) return rc;
    DeviceRestore restore;
    rc = r->CreateStream(out_stream);
    if (rc != hnsw::kOk && r != &e) h->fatal = r->last_error();
    return rc;
  });
}
int cuhnsw_search_knn_async_on(cuhnsw_handle* h, int32_t replica, void* cuda_stream, const float* qdata,
                               int64_t num_queries, int32_t topk, int32_t ef_search, int32_t* nns, float* distances,
                               int32_t* found_cnt) {
  return guarded(h, [&](hnsw::Engine& e) {
    int rc = hnsw::kOk;
    hnsw::Engine* r = h->replicas.Fresh(e, replica, &rc, &h->fatal);
    if (!r) return rc;
    DeviceRestore restore;
    void* before = r->stream();
    r->SetStream(cuda_stream);
    rc = r->SearchGraphAsync(qdata, num_queries, topk, ef_search, nns, distances, found_cnt);
    r->SetStream(before);
    if (rc != hnsw::kOk && r != &e) h->fatal = r->last_error();
    return rc;
  });
}
int cuhnsw_search_knn_noalloc(cuhnsw_handle* h, const float* qdata, int64_t num_queries, int32_t topk,
                              int32_t ef_search, int32_t* nns, float* distances, int32_t* found_cnt) {
  return guarded(h, [&](hnsw::Engine& e) {
    return e.SearchGraphStatic(qdata, num_queries, topk, ef_search, nns, distances, found_cnt);
  });
}
int cuhnsw_batch_distance(cuhnsw_handle* h, const int32_t* src, const int32_t* dst, int64_t num_pairs, float* out) {
  return guarded(h, [&](hnsw::Engine& e) { return e.BatchDistance(src, dst, num_pairs, out); });
}
int cuhnsw_set_stream(cuhnsw_handle* h, void* cuda_stream) {
  return guarded(h, [&](hnsw::Engine& e) { return e.SetStream(cuda_stream); });
}
int cuhnsw_synchronize(cuhnsw_handle* h) {
  return guarded(h, [&](hnsw::Engine& e) { return e.Synchronize(); });
}
int cuhnsw_stream_create(cuhnsw_handle* h, void** out_stream) {
  return guarded(h, [&](hnsw::Engine& e) { return e.CreateStream(out_stream); });
}
int cuhnsw_stream_synchronize(cuhnsw_handle* h, void* cuda_stream) {
  return guarded(h, [&](hnsw::Engine& e) { return e.SyncStream(cuda_stream); });
}
int cuhnsw_stream_destroy(cuhnsw_handle* h, void* cuda_stream) {
  return guarded(h, [&](hnsw::Engine& e) { return e.DestroyStream(cuda_stream); });
}
void* cuhnsw_host_alloc(cuhnsw_handle* h, size_t bytes) {
  void* p = nullptr;
  guarded(h, [&](hnsw::Engine& e) {
    p = e.HostAlloc(bytes);
    return hnsw::kOk;
  });
  return p;
}
void cuhnsw_host_free(cuhnsw_handle* h, void* ptr) {
  guarded(h, [&](hnsw::Engine& e) {
    e.HostFree(ptr);
    return hnsw::kOk;
  });
}
int cuhnsw_enable_stats(cuhnsw_handle* h, int32_t on) {
  return guarded(h, [&](hnsw::Engine& e) { return e.EnableStats(on); });
}
int cuhnsw_get_stats(cuhnsw_handle* h, uint64_t* out4) {
  if (!out4) return null_argument(h, "out4");
  return guarded(h, [&](hnsw::Engine& e) { return e.GetStats(reinterpret_cast<unsigned long long*>(out4)); });
}
int cuhnsw_describe(cuhnsw_handle* h, int64_t* out8) {
  if (!out8) return null_argument(h, "out8");
  return guarded(h, [&](hnsw::Engine& e) { return e.Describe(reinterpret_cast<long long*>(out8)); });
}
int cuhnsw_get_graph(cuhnsw_handle* h, int32_t* levels, int32_t* rows0, int32_t* rows_upper) {
  return guarded(h, [&](hnsw::Engine& e) { return e.GetGraph(levels, rows0, rows_upper); });
}
double cuhnsw_last_build_seconds(const cuhnsw_handle* h) { return h ? h->engine.last_build_seconds() : 0.0; }

int cuhnsw_merge_topk_device(const int32_t* d_ids, const float* d_distances, int32_t parts, int64_t num_queries,
                             int32_t topk, int32_t* d_out_ids, float* d_out_distances, int32_t* d_out_found,
                             void* cuda_stream) {
  if (parts < 1 || topk < 1 || num_queries < 0) return CUHNSW_INVALID_ARGUMENT;
  if (num_queries > 0 && (!d_ids || !d_distances || !d_out_ids || !d_out_distances)) return CUHNSW_INVALID_ARGUMENT;
  cudaError_t e = hnsw::launch_merge_topk(d_ids, d_distances, (long long)num_queries * topk, nullptr, parts,
                                          num_queries, topk, d_out_ids, d_out_distances, d_out_found,
                                          reinterpret_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? CUHNSW_OK : CUHNSW_CUDA_ERROR;
}

int cuhnsw_merge_topk_gathered_device(const int32_t* d_gathered, const int32_t* d_id_offsets, int32_t parts,
                                      int64_t num_queries, int32_t topk, int32_t* d_out_ids, float* d_out_distances,
                                      int32_t* d_out_found, void* cuda_stream) {
  if (parts < 1 || topk < 1 || num_queries < 0) return CUHNSW_INVALID_ARGUMENT;
  if (num_queries > 0 && (!d_gathered || !d_out_ids || !d_out_distances)) return CUHNSW_INVALID_ARGUMENT;
  const long long block = (long long)num_queries * topk;
  cudaError_t e = hnsw::launch_merge_topk(d_gathered, reinterpret_cast<const float*>(d_gathered + block), 2 * block,
                                          d_id_offsets, parts, num_queries, topk, d_out_ids, d_out_distances,
                                          d_out_found, reinterpret_cast<cudaStream_t>(cuda_stream));
  return e == cudaSuccess ? CUHNSW_OK : CUHNSW_CUDA_ERROR;
}

// (no exception can come up in these: they check sizes and launch)
namespace {
int status(cudaError_t e) { return e == cudaSuccess ? CUHNSW_OK : CUHNSW_CUDA_ERROR; }
bool type_ok(int32_t type) { return type == CUHNSW_F32 || type == CUHNSW_F16 || type == CUHNSW_BF16; }
bool type_aligned(const void* p, int32_t type) { return reinterpret_cast<uintptr_t>(p) % hnsw::type_size(type) == 0; }
// rows x dims values and their bytes stay far below 2^63
bool table_ok(int64_t rows, int64_t dims) {
  return rows >= 0 && rows < 0x7fffffffll && dims >= 1 && dims <= (1 << 24);
}
bool group_ok(int64_t group) { return group == 32 || group == 64 || (group >= 128 && group % 128 == 0 && group <= (1 << 24)); }
bool packed_ok(const void* codes, const void* scales) {
  return codes && scales && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 2 == 0;
}
}  // namespace

int cuhnsw_lookup_device(const void* d_rows, int64_t row_stride, int64_t num_rows, int64_t num_dims, int32_t type,
                         const void* d_ids, int32_t ids64, int64_t num_ids, float scale, void* d_out,
                         void* cuda_stream) {
  if (!table_ok(num_rows, num_dims) || !type_ok(type) || row_stride < 0 || num_ids < 0 || num_ids >= 0x7fffffffll)
    return CUHNSW_INVALID_ARGUMENT;
  if (num_ids == 0) return CUHNSW_OK;
  if ((num_rows > 0 && !d_rows) || !d_ids || !d_out || !type_aligned(d_rows, type) || !type_aligned(d_out, type) ||
      reinterpret_cast<uintptr_t>(d_ids) % (ids64 ? 8 : 4) != 0)
    return CUHNSW_INVALID_ARGUMENT;
  hnsw::LookupParams p{d_rows, row_stride, num_rows, num_dims, type, d_ids, ids64, num_ids, scale, d_out};
  return status(hnsw::launch_lookup(p, reinterpret_cast<cudaStream_t>(cuda_stream)));
}

int64_t cuhnsw_lookup_grad_workspace(int64_t num_ids, int64_t num_rows, int64_t num_dims) {
  if (!table_ok(num_rows, num_dims) || num_ids < 0 || num_ids >= 0x7fffffffll) return CUHNSW_INVALID_ARGUMENT;
  return (int64_t)hnsw::lookup_grad_workspace(num_ids, num_rows, num_dims);
}

int cuhnsw_lookup_grad_device(const void* d_grad, int64_t grad_stride, int32_t type, const void* d_ids, int32_t ids64,
                              int64_t num_ids, int64_t num_rows, int64_t num_dims, float scale, void* d_out,
                              int32_t out_type, int32_t accumulate, void* d_workspace, void* cuda_stream) {
  if (!table_ok(num_rows, num_dims) || !type_ok(type) || (out_type != type && out_type != CUHNSW_F32) ||
      grad_stride < 0 || num_ids < 0 || num_ids >= 0x7fffffffll)
    return CUHNSW_INVALID_ARGUMENT;
  if (num_rows == 0) return CUHNSW_OK;
  if (!d_out || !type_aligned(d_out, out_type)) return CUHNSW_INVALID_ARGUMENT;
  if (num_ids > 0 && (!d_grad || !type_aligned(d_grad, type) || !d_ids || !d_workspace ||
                      reinterpret_cast<uintptr_t>(d_ids) % (ids64 ? 8 : 4) != 0 ||
                      reinterpret_cast<uintptr_t>(d_workspace) % 256 != 0))
    return CUHNSW_INVALID_ARGUMENT;
  hnsw::LookupGradParams p{d_grad, grad_stride, type, d_ids, ids64, num_ids, num_rows, num_dims, scale, d_out, out_type,
                           accumulate, d_workspace};
  return status(hnsw::launch_lookup_grad(p, reinterpret_cast<cudaStream_t>(cuda_stream)));
}

int cuhnsw_pack4_device(const void* d_rows, int64_t row_stride, int32_t type, int64_t num_rows, int64_t num_dims,
                        int64_t group, void* d_codes, void* d_scales, void* cuda_stream) {
  if (!table_ok(num_rows, num_dims) || !type_ok(type) || !group_ok(group) || row_stride < 0) return CUHNSW_INVALID_ARGUMENT;
  if (num_rows == 0) return CUHNSW_OK;
  if (!d_rows || !type_aligned(d_rows, type) || !packed_ok(d_codes, d_scales)) return CUHNSW_INVALID_ARGUMENT;
  return status(hnsw::launch_pack4(d_rows, row_stride, type, num_rows, num_dims, group, d_codes, d_scales,
                                   reinterpret_cast<cudaStream_t>(cuda_stream)));
}

int cuhnsw_unpack4_device(const void* d_codes, const void* d_scales, int64_t num_rows, int64_t num_dims, int64_t group,
                          void* d_out, int32_t type, void* cuda_stream) {
  if (!table_ok(num_rows, num_dims) || !type_ok(type) || !group_ok(group)) return CUHNSW_INVALID_ARGUMENT;
  if (num_rows == 0) return CUHNSW_OK;
  if (!packed_ok(d_codes, d_scales) || !d_out || !type_aligned(d_out, type)) return CUHNSW_INVALID_ARGUMENT;
  return status(hnsw::launch_unpack4(d_codes, d_scales, num_rows, num_dims, group, d_out, type,
                                     reinterpret_cast<cudaStream_t>(cuda_stream)));
}

int cuhnsw_scores4_device(const void* d_codes, const void* d_scales, int64_t num_rows, int64_t num_dims, int64_t group,
                          const void* d_queries, int64_t query_stride, int32_t type, int64_t num_queries,
                          const float* d_bias, float* d_out, void* cuda_stream) {
  if (!table_ok(num_rows, num_dims) || !type_ok(type) || !group_ok(group) || query_stride < 0 || num_queries < 0 ||
      num_queries > (1 << 18))
    return CUHNSW_INVALID_ARGUMENT;
  if (num_rows == 0 || num_queries == 0) return CUHNSW_OK;
  if (!packed_ok(d_codes, d_scales) || !d_queries || !type_aligned(d_queries, type) || !d_out ||
      !type_aligned(d_out, CUHNSW_F32) || !type_aligned(d_bias, CUHNSW_F32))
    return CUHNSW_INVALID_ARGUMENT;
  hnsw::Scores4Params p{d_codes, d_scales, num_rows, num_dims, group, d_queries, query_stride, type, num_queries, d_bias,
                        d_out};
  return status(hnsw::launch_scores4(p, reinterpret_cast<cudaStream_t>(cuda_stream)));
}

namespace {
bool select_ok(int64_t sequences, int64_t beams, int64_t vocabulary, int32_t keep) {
  return sequences >= 0 && sequences < 0x7fffffffll && beams >= 1 && beams <= 16384 && vocabulary >= 1 &&
         vocabulary < 0x7fffffffll && keep >= 1 && keep <= hnsw::kMaxKeep;
}
}  // namespace

int64_t cuhnsw_select_workspace(int64_t sequences, int64_t beams, int64_t vocabulary, int32_t keep) {
  if (!select_ok(sequences, beams, vocabulary, keep)) return CUHNSW_INVALID_ARGUMENT;
  return (int64_t)hnsw::select_workspace(sequences, beams, vocabulary, keep);
}

int cuhnsw_select_device(const void* d_scores, int64_t seq_stride, int64_t beam_stride, int32_t type,
                         const float* d_totals, int64_t sequences, int64_t beams, int64_t vocabulary, int32_t keep,
                         int32_t log_softmax, int32_t negate, float* d_out_totals, int32_t* d_out_beams,
                         int32_t* d_out_ids, int32_t* d_out_found, void* d_workspace, void* cuda_stream) {
  if (!select_ok(sequences, beams, vocabulary, keep) || !type_ok(type) || seq_stride < 0 || beam_stride < 0)
    return CUHNSW_INVALID_ARGUMENT;
  if (sequences == 0) return CUHNSW_OK;
  if (!d_scores || !type_aligned(d_scores, type) || !type_aligned(d_totals, CUHNSW_F32) || !d_out_totals || !d_out_ids ||
      !d_workspace || reinterpret_cast<uintptr_t>(d_workspace) % 256 != 0)
    return CUHNSW_INVALID_ARGUMENT;
  hnsw::SelectParams p{d_scores, type, seq_stride, beam_stride, d_totals, sequences, beams, vocabulary, keep, log_softmax,
                       d_out_totals, d_out_beams, d_out_ids, d_out_found, negate ? -1.0f : 1.0f, d_workspace};
  return status(hnsw::launch_select(p, reinterpret_cast<cudaStream_t>(cuda_stream)));
}

int cuhnsw_reorder_device(const cuhnsw_state* states, int32_t count, const int32_t* d_beams, int64_t sequences,
                          int64_t beams, int64_t keep, void* cuda_stream) {
  if (count < 0 || sequences < 0 || beams < 0 || keep < 0 || sequences >= 0x7fffffffll || beams >= 0x7fffffffll ||
      keep >= 0x7fffffffll || (count > 0 && !states))
    return CUHNSW_INVALID_ARGUMENT;
  if (count == 0 || sequences * keep == 0) return CUHNSW_OK;
  if (!d_beams) return CUHNSW_INVALID_ARGUMENT;
  for (int32_t i = 0; i < count; ++i) {
    const cuhnsw_state& s = states[i];
    if (s.segments < 0 || s.bytes < 0 || s.seq_stride < 0 || s.beam_stride < 0 || s.segment_stride < 0 ||
        (s.segments * s.bytes > 0 && ((beams > 0 && !s.d_src) || !s.d_dst)))
      return CUHNSW_INVALID_ARGUMENT;
  }
  for (int32_t first = 0; first < count; first += hnsw::kMaxStates) {
    hnsw::ReorderState block[hnsw::kMaxStates];
    const int32_t some = count - first < hnsw::kMaxStates ? count - first : hnsw::kMaxStates;
    for (int32_t i = 0; i < some; ++i) {
      const cuhnsw_state& s = states[first + i];
      block[i] = {s.d_src, s.d_dst, s.seq_stride, s.beam_stride, s.segment_stride, s.segments, s.bytes};
    }
    const int rc = status(hnsw::launch_reorder(block, some, d_beams, sequences, beams, keep,
                                               reinterpret_cast<cudaStream_t>(cuda_stream)));
    if (rc != CUHNSW_OK) return rc;
  }
  return CUHNSW_OK;
}

int cuhnsw_selftest_list_merge(int32_t capacity, const float* distances, const int32_t* ids,
                               const int32_t* batch_begin, int32_t num_batches, const int32_t* expand_before,
                               uint64_t* out_keys, int32_t* out_size, int32_t* out_first_position,
                               int32_t* out_cursor) {
  if (capacity < 1 || capacity > 8192 || num_batches < 0 || !batch_begin || !expand_before || !out_keys || !out_size ||
      !out_first_position || !out_cursor)
    return CUHNSW_INVALID_ARGUMENT;
  for (int b = 0; b < num_batches; ++b)
    if (batch_begin[b + 1] < batch_begin[b] || batch_begin[b + 1] - batch_begin[b] > 32) return CUHNSW_INVALID_ARGUMENT;
  if (batch_begin[num_batches] > 0 && (!distances || !ids)) return CUHNSW_INVALID_ARGUMENT;
  cudaError_t e = hnsw::selftest_list_host(capacity, distances, ids, batch_begin, num_batches, expand_before,
                                           reinterpret_cast<unsigned long long*>(out_keys), out_size,
                                           out_first_position, out_cursor);
  return e == cudaSuccess ? CUHNSW_OK : CUHNSW_CUDA_ERROR;
}

int cuhnsw_selftest_visited(int32_t entries, int64_t num_nodes, const int32_t* ids, int32_t count, int32_t* out_seen) {
  if (entries < 64 || entries > 32768 || (entries & (entries - 1)) || num_nodes < 1 || count < 0 ||
      (count > 0 && (!ids || !out_seen)))
    return CUHNSW_INVALID_ARGUMENT;
  for (int i = 0; i < count; ++i)
    if (ids[i] < 0 || ids[i] >= num_nodes) return CUHNSW_INVALID_ARGUMENT;
  cudaError_t e = hnsw::selftest_visited_host(entries, num_nodes, ids, count, out_seen);
  return e == cudaSuccess ? CUHNSW_OK : CUHNSW_CUDA_ERROR;
}

}  // extern "C"
