// Launchers of the operators over a table of embeddings (device pointers, enqueued on the given stream).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace hnsw {

// element types, as in the option row_dtype
enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

inline int type_size(int type) { return type == kF32 ? 4 : 2; }

struct LookupParams {
  const void* rows;      // n rows of d values, row_stride values apart
  long long row_stride;
  long long n;
  long long d;
  int type;
  const void* ids;       // `tokens` numbers, 32 or 64 bits
  int ids64;
  long long tokens;
  float scale;
  void* out;             // tokens x d
};
cudaError_t launch_lookup(const LookupParams& p, cudaStream_t stream);

struct LookupGradParams {
  const void* grad;      // `tokens` rows of d values, grad_stride values apart
  long long grad_stride;
  int type;
  const void* ids;
  int ids64;
  long long tokens;
  long long n;
  long long d;
  float scale;
  void* out;             // n x d, of out_type: the type of `grad` or fp32
  int out_type;
  int accumulate;        // add to what `out` holds instead of writing every row
  void* workspace;       // lookup_grad_workspace bytes, 256-byte aligned
};
size_t lookup_grad_workspace(long long tokens, long long n, long long d);
cudaError_t launch_lookup_grad(const LookupGradParams& p, cudaStream_t stream);

// Rows in 4 bits: see cuhnsw_pack4_device in include/cuhnsw_b200.h for the layout.
inline long long packed_row_bytes(long long d) { return 16 * ((d + 31) / 32); }
inline long long packed_groups(long long d, long long group) { return (d + group - 1) / group; }
cudaError_t launch_pack4(const void* rows, long long row_stride, int type, long long n, long long d, long long group,
                         void* codes, void* scales, cudaStream_t stream);
cudaError_t launch_unpack4(const void* codes, const void* scales, long long n, long long d, long long group, void* out,
                           int type, cudaStream_t stream);

struct Scores4Params {
  const void* codes;
  const void* scales;
  long long n;
  long long d;
  long long group;
  const void* queries;   // nq rows of d values, query_stride values apart
  long long query_stride;
  int type;
  long long nq;
  const float* bias;     // n values, or null
  float* out;            // nq x n
};
cudaError_t launch_scores4(const Scores4Params& p, cudaStream_t stream);

constexpr int kMaxKeep = 256;  // results per sequence of launch_select

struct SelectParams {
  const void* scores;    // sequences x beams x vocabulary; the last dimension is contiguous
  int type;
  long long seq_stride;  // in values
  long long beam_stride;
  const float* totals;   // sequences x beams, or null
  long long sequences;
  long long beams;
  long long vocabulary;
  int keep;
  int log_softmax;
  float* out_totals;     // sequences x keep
  int* out_beams;        // or null
  int* out_ids;
  int* out_found;        // sequences, or null
  float sign;            // out_totals = sign * total (-1: distances of the dot metric)
  void* workspace;       // select_workspace bytes, 256-byte aligned
};
size_t select_workspace(long long sequences, long long beams, long long vocabulary, int keep);
cudaError_t launch_select(const SelectParams& p, cudaStream_t stream);

// One state of launch_reorder: rows (sequence, beam) of `segments` pieces of `bytes` bytes each.
struct ReorderState {
  const void* src;
  void* dst;               // sequences x keep rows, dense
  long long seq_stride;    // bytes, of src
  long long beam_stride;
  long long segment_stride;
  long long segments;
  long long bytes;
};
constexpr int kMaxStates = 32;  // of one launch
cudaError_t launch_reorder(const ReorderState* states, int count, const int* beams_of, long long sequences,
                           long long beams, long long keep, cudaStream_t stream);

}  // namespace hnsw
