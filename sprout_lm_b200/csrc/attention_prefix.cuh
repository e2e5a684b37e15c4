// What the kernels of attention over shared prefixes (attention_prefix.cu, attention_prefix_tcgen05.cu) share: a launch's parameters, the
// items of its plan, and where an item's partial results go.
#pragma once
#include "common.cuh"

namespace sprout_prefix {

// A plan takes a step's tokens in members: up to MEMBER_TOKENS tokens of a request, one behind the other.  It divides the keys that all of
// a member's tokens see into segments: a run of pages that several members hold, or a member's own keys behind those.  Tokens stand in
// the plan's order, in which the members of every segment lie side by side.  A segment's rows are its tokens times the query heads of a
// key/value head; an item is some of its rows over some of its keys, for every key/value head.  So every row of an item sees every
// key of it: there is no mask, and what a later token of the step left in the cache reaches no earlier one.  The keys that only some of
// a member's tokens see (those of the member's own later tokens, fewer than MEMBER_TOKENS) are added where the parts are put together.
constexpr int MEMBER_TOKENS = 16;

struct Item {
  int table;                           // the request whose block table gives the pages (any that holds them)
  int key_begin, key_end;
  int token_begin;                     // the segment's first token, in the plan's order
  int row_begin, rows;                 // of the segment's rows: (token - token_begin) * group + head within the group
  int part;                            // the place of this range among the token's ranges
  int open;                            // the range grows with the member: it ends with what its tokens all see (see Params::stretch)
};

struct Params {
  const void* q; long long q_stride;   // [tokens, heads * head_dim]
  const void* k_cache; const void* v_cache;            // [pages, kv_heads, page_tokens, head_dim]
  const int* block_table; int table_stride;
  const int* positions;                // [tokens]: the tokens' own, which have to be the plan's
  const Item* items;
  const int* order;                    // [tokens]: the step's token at a place of the plan's order
  const int* part_start;               // [tokens + 1]: the first of the place's partial results
  const int* seen;                     // [tokens]: keys that the items of a place's member hold
  const int* extra;                    // [tokens]: and the further ones that the place sees, fewer than MEMBER_TOKENS
  const int* table_of;                 // [tokens]: the place's request
  float* part_out;                     // [partial results, heads, head_dim], unnormalised
  float2* part_sum;                    // [partial results, heads]: the maximum (scaled, times log2(e)) and the sum
  void* out; long long out_stride;
  int tokens, heads, kv_heads, head_dim, page_tokens, num_pages;
  float scale_log2;                    // log2(e) / sqrt(head_dim)
  int* status;
  // The plan serves steps whose tokens stand up to this many positions behind those that it was made for; the member's last own range is
  // open then.
  int stretch;
  int first;                           // the call's first launch (see begin_items)
  unsigned long long* gate;            // in the scratch: holds `token` while the stream's earlier kernels are known to be done, else anything
  unsigned long long token;            // the call's own
};

// The launches of a call's items do not depend on one another.  The first waits for the stream's earlier kernels before it lets the next
// start; the others start when all of its CTAs have, so after those kernels, and wait for it only before they end: then the launch that
// puts the parts together, which waits for the last of them, starts behind all.
//
// Started after the earlier kernels is not yet told of what they wrote: only a grid's own pdl_wait makes that visible to it, and here that
// wait would be for the call's other items too (with it, 24 requests of up to 6 tokens over 2,000 keys take 36.2 us a call, 21.7 without; 32
// of up to 3,300 own keys 70.0 and 45.3).  So the first launch hands it on: a thread that has waited opens the gate (release), and every
// thread of the launches behind looks at it (acquire) before it touches what an earlier kernel may have used.  One that finds the gate
// shut waits for the launch before it, as any other kernel does.  The launch that puts the parts together shuts the gate behind itself; the
// token, whose upper half is a NaN's, is not met in memory that nothing of the call has written.
__device__ __forceinline__ void open_gate(const Params& p) {
  unsigned long long before;
  asm volatile("atom.release.gpu.global.exch.b64 %0, [%1], %2;" : "=l"(before) : "l"(p.gate), "l"(p.token) : "memory");
  if (before != p.token) pdl_launch_dependents();      // the exchange is done before anything starts
}
__device__ __forceinline__ void pass_gate(const Params& p) {
  unsigned long long seen;
  asm volatile("ld.acquire.gpu.global.b64 %0, [%1];" : "=l"(seen) : "l"(p.gate) : "memory");
  if (seen != p.token) pdl_wait();
}
__device__ __forceinline__ void begin_items(const Params& p) {
  if (!p.first) {
    pdl_launch_dependents();
    pass_gate(p);
    return;
  }
  pdl_wait();
  // a CTA lets the next launch start with the first of its threads that says so
  if (blockIdx.x != 0 || blockIdx.y != 0) pdl_launch_dependents();
  else if (threadIdx.x == 0) open_gate(p);
}
__device__ __forceinline__ void end_items(const Params& p) { if (!p.first) pdl_wait(); }

// An item as it is in this step: an open range ends with the member's first token, within the plan's bounds and never empty, whatever the
// positions say.  (The plan itself was there before the call; what a step's kernels write, positions, queries, block tables and the cache, is
// read behind begin_items.)
__device__ __forceinline__ Item in_step(const Params& p, Item item) {
  if (p.stretch > 0 && item.open) item.key_end = max(item.key_begin + 1, min(item.key_end, p.positions[p.order[item.token_begin]] + 1));
  return item;
}
// An item's row i, 0 <= i < rows: its place in the plan's order, and its query head.
__device__ __forceinline__ int place_of_row(const Item& item, int i, int group) { return item.token_begin + (item.row_begin + i) / group; }
__device__ __forceinline__ int head_of_row(const Item& item, int i, int group, int g) { return g * group + (item.row_begin + i) % group; }

// The element offset of a key's row in the cache; -1 (and a status bit) where its page lies outside the pool.
__device__ __forceinline__ long long key_row(const Params& p, const int* table, int key, int g) {
  const int page = table[key / p.page_tokens];
  if (page < 0 || page >= p.num_pages) { atomicOr(p.status, SPROUT_STATUS_BAD_PAGE); return -1; }
  return (((long long)page * p.kv_heads + g) * p.page_tokens + key % p.page_tokens) * p.head_dim;
}

// Room for `bytes` of dynamic shared memory, always the same for a kernel; asked for once a device.
template <auto KERNEL>
int reserve_shared(size_t bytes, const char* what) {
  static bool done[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return sprout_fail("%s: no current device", what);
  if (done[device]) return 0;
  const cudaError_t err = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (err != cudaSuccess) return sprout_fail("%s: cannot reserve %zu bytes of shared memory: %s", what, bytes, cudaGetErrorString(err));
  done[device] = true;
  return 0;
}

}  // namespace sprout_prefix
