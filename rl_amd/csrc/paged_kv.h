// Launch interface of the paged key-value cache kernels (paged_kv.hip):
// plain structs, no C++ exceptions across the boundary.  Every launcher
// returns the hipError_t of its launches as an int.
#pragma once

// A cache [pages][kv_heads][page_size][dim] with a dense last dim; strides in
// elements.  Page ids outside [0, pages) are never followed.
struct PagedCache {
  void* k;
  void* v;
  long k_page, k_head, k_slot;
  long v_page, v_head, v_slot;
  long pages;
  int page_shift;          // page_size = 1 << page_shift
  const int* table;        // [batch][table_stride >= table_cols]
  long table_stride;
  int table_cols;
};

struct PagedAppendArgs {
  PagedCache cache;
  const void *q, *k, *v;   // [batch][width][heads][dim]; q may be null
  long q_batch, q_token, q_head;
  long k_batch, k_token, k_head;
  long v_batch, v_token, v_head;
  void* q_out;             // [batch][width][heads][dim] dense
  const void* start;       // [batch], int32 or int64
  const void* lengths;     // [batch] or null: width
  int start_i64, lengths_i64;
  const float *cos, *sin;  // [positions][rotary / 2] dense, or null
  long positions;
  long batch;
  int width, heads, kv_heads, dim, rotary, interleaved;
  int dtype;               // RlDtype
  int vec;                 // elements per access that every address allows
};

struct PagedAttendArgs {
  PagedCache cache;
  const void* q;           // [batch][heads][dim]
  long q_batch, q_head;
  void* out;               // [batch][heads][dim] dense
  const void* lengths;     // [batch]
  int lengths_i64;
  long batch;
  int heads, kv_heads, dim;
  int dtype;
  float scale;             // of the scores, times log2(e)
  // the plan: filled in by plan_paged_attend
  int head_blocks;         // blocks of 16 query heads per key head
  int workers;             // 0: one workgroup per (sequence, key head, block)
  int waves;               // of a workgroup
  // workspace where workers > 0
  float* part;             // [2 * workers][min(16, heads / kv_heads)][dim]
  float* part_ms;          // [2 * workers][min(16, heads / kv_heads)][2]
  void* notes;             // [workers] of paged_attend_note_bytes()
};

extern "C" {
int launch_paged_append(const PagedAppendArgs* a, void* stream);
long paged_attend_note_bytes(void);
void plan_paged_attend(PagedAttendArgs* a, int cus);
int launch_paged_attend(const PagedAttendArgs* a, void* stream);
}
