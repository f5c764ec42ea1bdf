// Entry points of the paged KV cache: csrc/paged_tables.cu, csrc/paged_append.cu, csrc/paged_attention.cu.
//
// A pool holds `pages` pages of `page_size` positions; a row's table says which pages it has, position p lies on page
// table[p / page_size] at p % page_size, and its slot is page * page_size + p % page_size.
// The reference has no KV cache of its own: it serves the ones of vLLM and SGLang (README.md:20-33).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace penny {

// 16-byte aligned rows of one position and head in a pool [pages, page_size, heads, dim]; strides in elements.
struct PagedPool {
  void* k;
  void* v;
  long long page_stride, pos_stride, head_stride;
  const float* k_scale;  // e4m3 pools: per head, what a stored value is multiplied by
  const float* v_scale;
  int pages, page_size, heads, dim;
};
enum PagedType { PAGED_BF16 = 0, PAGED_FP16 = 1, PAGED_E4M3 = 2 };

constexpr int kPagedMaxRows = 8192;
struct PageTables {
  int* table;  // [rows, width], rows of table_stride
  long long table_stride;
  int *lengths, *free_pages, *free_count;
  const int* news;
  long long* slots;
  int *positions, *offsets;
  bool* granted;
  int rows, width, pages, page_size, tokens;
  int max_len;  // positions that a row may be granted, at most
  int* refs;    // [pages] or null: how many rows have a page
};
cudaError_t launch_page_tables(const PageTables& a, cudaStream_t stream);

// Rows with pages in common (csrc/paged_share.cu): the state of PageTables with refs.
struct PageFork {
  int* table;
  long long table_stride;
  int *lengths, *free_pages, *free_count, *refs;
  const int *source, *target;  // [forks]
  int *copy_from, *copy_to;    // [forks]
  bool* granted;
  int rows, width, pages, page_size, forks;
};
cudaError_t launch_page_fork(const PageFork& a, cudaStream_t stream);

struct PageCompact {
  int* table;
  long long table_stride;
  const int* lengths;
  int *free_pages, *free_count, *refs;
  int *copy_from, *copy_to;  // [pages / 2]
  int rows, width, pages, page_size;
};
cudaError_t launch_page_compact(const PageCompact& a, cudaStream_t stream);

// Pages of `pools` pools of one layout: runs of run_bytes (whole 16 bytes) at outer by outer_bytes and inner by inner_bytes.
constexpr int kPageCopyPools = 128;  // of a launch
struct PageCopy {
  char* pool[kPageCopyPools];
  const int *from, *to;
  long long page_bytes, outer_bytes, inner_bytes;
  int pools, copies, pages, outer, inner, run_bytes;
};
cudaError_t launch_page_copy(const PageCopy& a, int sms, cudaStream_t stream);

struct PageGroups {
  const int* table;
  long long table_stride;
  const int* lengths;
  int *order, *starts, *shared;  // [rows], [rows + 1], [rows]
  int rows, width, page_size;
};
cudaError_t launch_page_groups(const PageGroups& a, cudaStream_t stream);

// type: of qkv and out.  out null: in place.  early: slots and positions are read before the kernels that may still run when this one
// starts end.
cudaError_t launch_paged_append(void* qkv, long long qkv_stride, void* out, long long out_stride, PagedType type, const PagedPool& pool,
                                PagedType cache, const long long* slots, const int* positions, int tokens, int heads, double theta,
                                bool early, cudaStream_t stream);

struct PagedAttention {
  const void* q;  // [rows, heads, dim]
  long long q_stride, q_head_stride;
  void* out;
  long long out_stride, out_head_stride;
  float* lse;  // [rows, heads] or null
  const int* table;
  long long table_stride;
  const int* lengths;
  int rows, heads, width, window;
  float scale;
  // Kernels that may still run when this one starts (programmatic dependent launch) write, of what it reads, q and the keys and values
  // of the rows' last positions alone: the rest is read before they end.
  bool early;
};
size_t paged_attention_workspace_bytes(int rows, int heads, int kv_heads, int dim, int max_len, int window, int sms);
cudaError_t launch_paged_attention(const PagedAttention& a, PagedType type, const PagedPool& pool, PagedType cache, void* workspace,
                                   int sms, cudaStream_t stream);

// The same for rows that share pages (csrc/paged_shared_attention.cu), groups as k_page_groups finds them; a.early is not looked at.
struct SharedGroups {
  const int *order, *starts, *shared;
};
size_t shared_attention_workspace_bytes(int rows, int heads, int dim, int sms);
cudaError_t launch_shared_attention(const PagedAttention& a, PagedType type, const PagedPool& pool, PagedType cache, const SharedGroups& groups,
                                    void* workspace, int sms, uint32_t* error_word, cudaStream_t stream);

}  // namespace penny
