/*
 * tgx.h -- C ABI of libtgx.so, the MI355X (gfx950) fused temporal data pipeline.
 *
 * Plain C: device pointers, sizes, dtype enums and a HIP stream passed as
 * `void*` (a hipStream_t; NULL means the legacy default stream).  No torch
 * types cross this boundary.  Every entry point:
 *   - launches only on the given stream and never synchronises the device;
 *   - never allocates or frees device memory: outputs, ring arrays and the
 *     workspace belong to the caller;
 *   - keeps no state between calls (safe from any host thread);
 *   - returns TGX_OK (0) or an error code; the message of the last failure on
 *     the calling thread is returned by tgx_last_error().
 *
 * Reference interfaces replaced (paths relative to the tgengine checkout):
 *   tgx_ring_append   <- TemporalGraph.advance post-freeze branch
 *                        tgengine/core/temporal_graph.py:123-129 and
 *                        _append_overflow :351-387 (pure torch there; no native op);
 *                        tgx_ring_plan / tgx_ring_commit / tgx_ring_discard split it
 *   tgx_recent        <- TemporalGraph.recent :183-349 (ring merge _merge_overflow
 *                        :307-349, CSR window :241-305) and the pybind op
 *                        temporal_recent_k (tgengine/core/csrc/temporal_sample.cu:291-329,
 *                        bound at :546-555 via tgengine/core/kernels.py:135-154), fused
 *                        with FixedCosineTimeEncoder (tgengine/nn/time_encoding.py:37-63)
 *                        and DyGFormer co-occurrence counting
 *                        (tgengine/models/dygformer.py:71-87)
 *   tgx_co_occurrence <- pybind op co_occurrence_freq (temporal_sample.cu:514-543,
 *                        kernels.py:203-221) and the (B,) pair count of
 *                        DataPipeline._co_occur_from_neighbors
 *                        (tgengine/pipeline/__init__.py:206-219)
 */
#ifndef TGX_H
#define TGX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TGX_ABI_VERSION 17

/* status codes */
#define TGX_OK 0
#define TGX_ERR_ARG 1      /* bad argument (null pointer, negative size, ...) */
#define TGX_ERR_DTYPE 2    /* unsupported dtype */
#define TGX_ERR_LIMIT 3    /* size beyond a documented limit */
#define TGX_ERR_HIP 4      /* a HIP runtime call failed (message has the HIP error) */

/* feature storage dtypes */
#define TGX_F32 0
#define TGX_BF16 1

/* dt conventions of the time encoding */
#define TGX_DT_DYGFORMER 0 /* dt = f32(q) - f32(t) in fp32; padding slots encode to 0 */
#define TGX_DT_TGN 1       /* dt = f32(q - t) (float64 subtract); padding uses t = 0.0 */

/* co-occurrence modes (pairs = queries 0 and 1 of every plan group) */
#define TGX_CO_NONE 0
#define TGX_CO_FREQ 1      /* int32 (P,K,2) counts per sequence + (P,) pair count */
#define TGX_CO_DYGFORMER 2 /* int32 (P,1+K,2): DyGFormer counts with the node at pos 0 */

/* device-side diagnostics: int32 status[TGX_STATUS_WORDS], accumulated */
#define TGX_STATUS_WORDS 8
#define TGX_ST_BAD_EVENT_NODE 0   /* append: src/dst outside [0, num_nodes) (entry skipped) */
#define TGX_ST_KEY_COLLISION 1    /* append: int(max t)+2 <= 2b-1 (reference key not lexicographic) */
#define TGX_ST_BAD_QUERY_NODE 2   /* recent: query node >= num_nodes (query returns padding) */

/* Per-node ring of `slots` entries (reference: temporal_graph.py:89-102).
 * ids int32 [N,B] (-1 empty), times float64 [N,B], feats [N,B,feat_dim] of
 * feat_dtype, write_pos int64 [N], eids int64 [N,B] (optional, may be NULL).
 * scratch: tgx_ring_scratch_size(N) bytes of device memory, zero-filled once by
 * the caller before the first append and otherwise left to the library: its
 * first N int32 are per-node counters that every tgx_ring_append restores to
 * zero, the rest is rewritten before each use.  Needed by tgx_ring_append only
 * (tgx_recent ignores it). */
typedef struct tgx_ring {
  int64_t num_nodes;
  int32_t slots;
  int32_t feat_dim;
  int32_t feat_dtype;
  int32_t reserved;
  int32_t* ids;
  double* times;
  void* feats;
  int64_t* write_pos;
  int64_t* eids;
  int32_t* scratch;
} tgx_ring;

/* Frozen CSR (reference: temporal_graph.py:133-181): offsets int64 [N+1],
 * ids int32 [E], times float64 [E] (ascending within a node), feats [E,feat_dim],
 * eids int64 [E] (optional).  max_time: the largest non-NaN time of the entries
 * (+inf when unknown).  Results never depend on it: a query at a later time is
 * after every window, and the gather then skips the search work it would issue
 * ahead for a query that may fall inside one. */
typedef struct tgx_csr {
  int64_t num_nodes;
  int64_t num_entries;
  int32_t feat_dim;
  int32_t feat_dtype;
  const int64_t* offsets;
  const int32_t* ids;
  const double* times;
  const void* feats;
  const int64_t* eids;
  double max_time;
} tgx_csr;

/* One group of queries read in place: query l of the group is node nodes[l]
 * at time times[l / times_per] (times_per = negatives per event for a (b, n)
 * row-major negative block, else 1). */
typedef struct tgx_query_group {
  const void* nodes;       /* [count] node ids: int64, or int32 with TGX_QG_NODES_I32 */
  const double* times;
  int64_t count;
  int32_t times_per;
  int32_t flags;           /* TGX_QG_* bits */
  const uint8_t* valid;    /* [count] or NULL; a 0 makes that query padding only
                              (no candidates, no status count): the 2-hop queries
                              under invalid hop-1 slots */
} tgx_query_group;
#define TGX_QG_NODES_I32 1

/* work plans of tgx_recent_args.plan_mode */
#define TGX_PLAN_TILES 0
#define TGX_PLAN_EVENTS 1
#define TGX_PLAN_LIST 2

#define TGX_MAX_QUERY_GROUPS 4

typedef struct tgx_recent_args {
  /* queries: either nodes/times, or num_query_groups > 0 groups concatenated
   * in order (query index = group offset + position in the group) */
  const int64_t* nodes;    /* [Q] node ids; < 0 = padding query */
  const double* times;     /* [Q] query times */
  int64_t num_queries;
  int32_t k;               /* neighbours per query, 1..TGX_MAX_K */
  /* work plan, by plan_mode:
   *   TGX_PLAN_TILES (plan NULL): consecutive queries; `group` queries per
   *     workgroup (a hint: when a small launch shares each query among several
   *     wavefronts, a query takes a workgroup of its own); num_groups is ignored;
   *   TGX_PLAN_EVENTS (plan NULL): event-major groups computed from the query
   *     groups: group g = event g holds, for each query group in order,
   *     its times_per queries of event g (the reference grouping [src, dst,
   *     neg row-major, neg_src], pipeline/__init__.py:40-70, read as one
   *     group per event); group = sum of times_per, num_groups = events.
   *     With event_query_groups = E > 0, only the first E query groups form
   *     the events (group = their sum of times_per); the queries of the other
   *     groups follow in workgroups of `group` consecutive queries;
   *   TGX_PLAN_LIST (plan set): group g handles queries plan[g*group + j],
   *     j < group (-1 = none).
   * Co-occurrence needs TGX_PLAN_EVENTS or TGX_PLAN_LIST (its pairs are
   * queries 0 and 1 of a group). */
  const int32_t* plan;
  int32_t group;           /* 1..8 */
  int32_t plan_mode;       /* TGX_PLAN_*; TGX_PLAN_LIST iff plan != NULL */
  int64_t num_groups;
  /* outputs (row = query index); out_feats / out_eids / out_te may be NULL */
  int32_t* out_ids;        /* [Q,K] */
  double* out_times;       /* [Q,K] */
  void* out_feats;         /* [Q,K,feat_dim] in the storage dtype */
  uint8_t* out_mask;       /* [Q,K] 0/1 */
  int64_t* out_eids;       /* [Q,K] */
  /* fused FixedCosineTimeEncoder: out_te[Q,K,d_t] = cos(fl32(dt*w) [+ b]) */
  int32_t d_t;             /* 0 = off */
  const float* te_w;       /* [d_t] */
  const float* te_b;       /* [d_t] or NULL (bias 0) */
  int32_t dt_mode;         /* TGX_DT_* */
  float* out_te;
  /* fused co-occurrence for the (query 0, query 1) pair of every group */
  int32_t co_mode;         /* TGX_CO_* */
  int32_t* co_a;           /* FREQ: [P,K,2]; DYGFORMER: [P,1+K,2] */
  int32_t* co_c;
  float* co_pair;          /* [P] float shared-neighbour count (both modes), may be NULL */
  int32_t* status;         /* [TGX_STATUS_WORDS] or NULL */
  int32_t num_query_groups;                          /* 0 = use nodes/times */
  tgx_query_group query_groups[TGX_MAX_QUERY_GROUPS];
  /* optional hipEvent_t pair recorded by the dispatches themselves: the start of the
   * gather kernel's execution and its end, or the end of the kernel that counts the
   * pairs where that is a launch of its own (some event-major launches over a CSR alone
   * with k above 64); the launches are the same as without.  Both NULL = plain launch */
  void* timing_start;
  void* timing_stop;
  /* optional ring plan run by the same launch (append_b > 0): tgx_ring_plan of
   * the batch append_src/dst/time (append_b events, append_workspace of
   * tgx_ring_append_workspace_size(append_b) bytes) that the caller appends
   * next, through tgx_ring_commit (or drops through tgx_ring_discard).  The plan
   * reads the batch and the ring's write positions and writes only the
   * workspace, so it runs beside the gather; batches above 16384 events are
   * planned by launches of their own after the gather.  append_b == 0: no plan. */
  const int64_t* append_src;
  const int64_t* append_dst;
  const double* append_time;
  int64_t append_b;
  void* append_workspace;
  size_t append_workspace_bytes;
  /* TGX_PLAN_EVENTS: the number of leading query groups that form the events
   * (0 = all of them; see plan_mode) */
  int32_t event_query_groups;
  /* d_t > 0: upper bounds of max|te_w[i]| and max|te_b[i]| (0 without bias),
   * which let the cosine skip its large-argument reduction where no argument
   * can need it.  te_bound_w <= 0 (or NaN): unknown, every element takes the
   * full-range reduction (same results, slower).  The bounds are trusted and
   * not checked on the device: a bound below the true maximum gives WRONG
   * encodings (errors far above 1e-6) wherever |fl32(dt * w) + b| reaches 2^29.
   * Pass 0 unless the bound is known on the host. */
  float te_bound_w;
  float te_bound_b;
} tgx_recent_args;

#define TGX_MAX_SLOTS 64
#define TGX_MAX_K 512
#define TGX_MAX_GROUP 8
#define TGX_MAX_DT 512

/* Ring update for one batch of b undirected events (kernel a).
 * Entries are the 2b directed edges in the order [src->dst ..., dst->src ...];
 * per node the last min(c, B) entries in that order are written to slots
 * (write_pos + m) % B, m = 0.., and write_pos grows by min(c, B).
 * feat: [b, feat_dim] in ring->feat_dtype, or NULL for zero features.
 * eids (if the ring has them) receive eid_base + event index.
 * workspace: tgx_ring_append_workspace_size(b) bytes of device memory, 16-byte
 * aligned (no initialisation needed).  Calls on one ring must be ordered (one
 * stream). */
int tgx_ring_append(const tgx_ring* ring, const int64_t* src, const int64_t* dst,
                    const double* time, const void* feat, int64_t b, int64_t eid_base,
                    void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
size_t tgx_ring_append_workspace_size(int64_t b);
size_t tgx_ring_scratch_size(int64_t num_nodes);

/* tgx_ring_append with no workspace argument and no allocation: the workspace is
 * a file-scope device array of tgx_ring_append_static_max_bytes() bytes (2 MiB;
 * each GPU the library runs on holds its own copy until the process ends),
 * enough for batches with tgx_ring_append_workspace_size(b) <= that (about
 * 100,000 events); larger batches return TGX_ERR_LIMIT.  It calls no hipMalloc
 * or hipFree.  Every call on one GPU shares that GPU's array, so calls that
 * overlap on one GPU (other streams, other threads) race; calls ordered on one
 * stream are safe.  The ring's scratch is the caller's, as for tgx_ring_append.
 * No counterpart in the reference: it is for callers that cannot allocate
 * (code under HIP graph capture, serving loops, harnesses that forbid
 * hipMalloc). */
int tgx_ring_append_static(const tgx_ring* ring, const int64_t* src, const int64_t* dst,
                           const double* time, const void* feat, int64_t b, int64_t eid_base,
                           int32_t* status, void* stream);
size_t tgx_ring_append_static_max_bytes(void);

/* tgx_ring_append in two halves, so the first can run while other work still
 * reads the ring (the same split of _append_overflow, temporal_graph.py:351-387):
 *   tgx_ring_plan   : up to 16384 events, every entry's slot (or none) and every
 *                     node's new write position, in the workspace; reads
 *                     src/dst/time and write_pos, writes no ring array and no
 *                     scratch but two diagnostic words.  Above 16384 events,
 *                     per-node counts and entry lists in the workspace and the
 *                     ring's scratch, reading src/dst/time only; needs the
 *                     scratch counters at zero (as every commit or discard
 *                     leaves them).
 *   tgx_ring_commit : the ring writes of a planned batch (same arguments and
 *                     workspace as its plan); restores the counters; reports the
 *                     plan's diagnostics into `status`.
 *   tgx_ring_discard: drops a planned batch without touching the ring arrays and
 *                     restores the counters.
 * Plan, then exactly one of commit / discard, ordered on streams by the caller,
 * with no other write to the ring between them (the plan reads write_pos). */
int tgx_ring_plan(const tgx_ring* ring, const int64_t* src, const int64_t* dst,
                  const double* time, int64_t b, void* workspace, size_t workspace_bytes,
                  void* stream);
int tgx_ring_commit(const tgx_ring* ring, const int64_t* src, const int64_t* dst,
                    const double* time, const void* feat, int64_t b, int64_t eid_base,
                    void* workspace, size_t workspace_bytes, int32_t* status, void* stream);
int tgx_ring_discard(const tgx_ring* ring, const int64_t* src, const int64_t* dst, int64_t b,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Frozen-CSR build (TemporalGraph.freeze_csr, temporal_graph.py:133-181).
 * The n directed entries of the pre-freeze advance() calls, in build order
 * (per call: [src->dst for every event, dst->src for every event]), are sorted
 * stably by time, then stably by node: a node's entries end up time-ascending
 * with ties in build order.  Outputs (the tgx_csr arrays): out_offsets [N+1],
 * out_ids int32 [n] (= to), out_times [n], out_feats [n, feat_dim] (row of the
 * entry's event in feats, zero when feats is NULL), out_eids [n] (= event, may
 * be NULL).  Entries whose node is outside [0, N), or whose event is outside
 * [0, num_events) while feats is set, are counted in
 * status[TGX_ST_BAD_EVENT_NODE] (out-of-range nodes sort after every node).
 * workspace: tgx_csr_build_workspace_size(n) bytes, no initialisation needed.
 *
 * flags & TGX_CSR_EVENT_PAIRS: from/to/time hold the n/2 EVENTS (src, dst,
 * time) instead of the n entries, in an order where the stable sort by time
 * is the identity on the entries 2k = from[k]->to[k], 2k+1 = to[k]->from[k]
 * (both at time[k]; event index k, or event[k] when event is set): times
 * strictly increasing within every advance() call and non-decreasing across
 * calls, which makes this order the stable time order of the build order.  The
 * time passes are skipped; the caller checks the condition.
 *
 * flags & TGX_CSR_EVENTS_BY_CALL: from/to/time (and event) hold the n/2
 * events in stream order, and call_starts [num_calls] the first event of each
 * advance() call (ascending, starting at 0); the build forms the build order
 * itself (per call: from->to of each event, then to->from of each) and sorts
 * it by time.  With TGX_CSR_NONDECREASING as well, the caller asserts that
 * time never decreases along the events (no NaN): the stable time order is
 * then, run by run of equal times within a call, the run's from->to entries
 * followed by its to->from entries, and the time passes are skipped.  Call
 * starts outside [1, n/2) are ignored; a wrong order assertion gives a wrong
 * order, never an access outside the arrays. */
typedef struct tgx_csr_build_args {
  int64_t num_nodes;
  int64_t num_entries;
  const int64_t* from;     /* [n] node of each entry */
  const int64_t* to;       /* [n] neighbour id */
  const double* time;      /* [n] */
  const int64_t* event;    /* [n] event of each entry: edge id and feature row (NULL when unused) */
  const void* feats;       /* [num_events, feat_dim] in feat_dtype, or NULL */
  int64_t num_events;
  int32_t feat_dim;
  int32_t feat_dtype;
  int64_t* out_offsets;
  int32_t* out_ids;
  double* out_times;
  void* out_feats;
  int64_t* out_eids;
  void* workspace;
  size_t workspace_bytes;
  int32_t* status;         /* [TGX_STATUS_WORDS] or NULL */
  uint32_t flags;          /* TGX_CSR_* */
  const int64_t* call_starts;  /* [num_calls], TGX_CSR_EVENTS_BY_CALL only */
  int64_t num_calls;
} tgx_csr_build_args;

#define TGX_CSR_EVENT_PAIRS 1u
#define TGX_CSR_EVENTS_BY_CALL 2u
#define TGX_CSR_NONDECREASING 4u

size_t tgx_csr_build_workspace_size(int64_t num_entries);
int tgx_csr_build(const tgx_csr_build_args* args, void* stream);

/* Pre-freeze scan.  No counterpart in the reference, whose freeze_csr
 * (temporal_graph.py:133-181) sorts host lists; here freeze_csr learns from it,
 * in one round trip, the node range it checks, which build to run (event pairs
 * or general) and the largest time.  Over the num_events > 0 events src/dst/time of the pre-freeze
 * advance() calls, whose first events are call_starts [num_calls] (ascending,
 * a repeated value counts once; may be NULL when num_calls is 0), writes out
 * int64 [4]:
 *   out[0], out[1]  min and max node id over src and dst,
 *   out[2]          2 when the stream is time-ordered in the sense of
 *                   TGX_CSR_EVENT_PAIRS: for every k >= 1 the float64
 *                   difference time[k] - time[k-1] is > 0, or == 0 with k in
 *                   call_starts (NaN and inf - inf differences break it);
 *                   else 1 when time[k] >= time[k-1] for every k >= 1 (the
 *                   TGX_CSR_NONDECREASING condition), else 0,
 *   out[3]          the bits of the largest non-NaN time (-inf when all are NaN).
 * workspace: tgx_csr_scan_workspace_size() bytes, no initialisation needed.
 * Two launches; the caller reads out after the stream. */
size_t tgx_csr_scan_workspace_size(void);
int tgx_csr_scan(const int64_t* src, const int64_t* dst, const double* time, int64_t num_events,
                 const int64_t* call_starts, int64_t num_calls, int64_t* out, void* workspace,
                 size_t workspace_bytes, void* stream);

/* Historical negative pool (HistoricalNegPool, pipeline/negatives.py:14-126).
 * pool int32 [num_nodes, pool_size] (-1 = empty), count int64 [num_nodes]
 * (edges seen per source), both zero-/minus-one-filled by the caller once.
 * update: edge j of the batch, the r-th from its source u in batch order, is
 * u's e-th edge (e = count[u] + r + 1): e <= pool_size fills slot e-1, else it
 * replaces slot rand % pool_size with probability pool_size/e (float32); the
 * later edge of the batch wins a slot two edges take; count[u] grows by u's
 * edges.  sample: out[q] = pool[u][int(U * min(count[u], pool_size))] (slot
 * clamped to pool_size-1), or a random node in [0, num_nodes) for a node with
 * no history.  Random numbers: rand64(seed, call, i, stream) =
 * mix(mix(mix(seed ^ 0x9e3779b97f4a7c15) ^ call) ^ (4i + stream)), mix the
 * splitmix64 finalizer, U = (rand64 >> 40) * 2^-24; streams 0/1 (update accept /
 * slot), 2/3 (sample slot / fallback node).  Out-of-range ids are skipped
 * (update) or sampled as nodes without history (sample) and counted in status.
 * workspace: tgx_negpool_update_workspace_size(n) bytes (no initialisation
 * needed).  scratch: NULL, or tgx_negpool_scratch_size() bytes of device memory,
 * 256-byte aligned, zero-filled once by the caller and otherwise left to the
 * library (a table that every update leaves zeroed again); with it, batches of
 * up to 32,768 edges update in two launches over the whole device, without it in
 * one workgroup (up to 8,192 edges) or by sorting.  Same results either way.
 * Updates that share a scratch must be ordered (one stream). */
size_t tgx_negpool_update_workspace_size(int64_t n);
size_t tgx_negpool_scratch_size(void);
int tgx_negpool_update(int32_t* pool, int64_t* count, int64_t num_nodes, int32_t pool_size,
                       const int64_t* src, const int64_t* dst, int64_t n, uint64_t seed,
                       uint64_t call, void* workspace, size_t workspace_bytes, void* scratch,
                       size_t scratch_bytes, int32_t* status, void* stream);
int tgx_negpool_sample(const int32_t* pool, const int64_t* count, int64_t num_nodes,
                       int32_t pool_size, const int64_t* src, int64_t n, uint64_t seed,
                       uint64_t call, int64_t* out, int32_t* status, void* stream);

/* The same two operations with the caller's random draws, indexed as the
 * reference indexes its torch.rand / torch.randint draws
 * (pipeline/negatives.py:78-86, :116-124), so that draws taken from torch's
 * generator in the reference's call order give the reference's pool and
 * samples.  update: u_accept[p] (float32 in [0, 1)) and slot_draw[p] (in
 * [0, pool_size); other values skip the edge) of the edge at position p of
 * the batch's stable sort by source; sample: u_slot[q] (float32 in [0, 1)) of
 * query q, and out[q] = -1 for a node without history (the reference then
 * draws those nodes with torch.randint(0, num_nodes, (#such queries,)) in
 * query order; the caller does that).  The later edge of a batch still wins a
 * slot two accepted edges take, where the reference leaves it to the last
 * index_put_ write. */
int tgx_negpool_update_draws(int32_t* pool, int64_t* count, int64_t num_nodes, int32_t pool_size,
                             const int64_t* src, const int64_t* dst, int64_t n,
                             const float* u_accept, const int64_t* slot_draw, void* workspace,
                             size_t workspace_bytes, int32_t* status, void* stream);
int tgx_negpool_sample_draws(const int32_t* pool, const int64_t* count, int64_t num_nodes,
                             int32_t pool_size, const int64_t* src, int64_t n, const float* u_slot,
                             int64_t* out, int32_t* status, void* stream);

/* Fused most-recent-K gather (+ time encoding, + co-occurrence) (kernels b, c).
 * ring and/or csr may be NULL (no candidates from that store); with both NULL
 * every query is padding and out_feats must be NULL (the row width comes from
 * them). */
int tgx_recent(const tgx_ring* ring, const tgx_csr* csr, const tgx_recent_args* args,
               void* stream);

/* Launch shape tgx_recent would use for these arguments, without launching:
 * shape[0] workgroups, [1] threads per workgroup, [2] dynamic LDS bytes,
 * [3] queries per wavefront, [4] wavefronts per query in one workgroup (a
 * query split over more than 4 wavefronts without a ring spreads them over
 * several workgroups), [5] queries per workgroup (1 also for those),
 * [6] plan workgroups, [7] feature copy width in bytes.  Same
 * argument checks and return codes as tgx_recent. */
int tgx_recent_launch_shape(const tgx_ring* ring, const tgx_csr* csr, const tgx_recent_args* args,
                            int64_t shape[8]);

/* Stand-alone co-occurrence over neighbour-id rows a, c int32 [P,K]:
 * a_cnt/c_cnt int32 [P,K,2] (mode FREQ) and pair_count float [P] (may be NULL).
 * a_mask / c_mask uint8 [P,K] (0/1) mark the valid positions; with a NULL mask
 * a position is valid iff its id is not -1.  A count covers valid positions
 * only, and an invalid position's counts are 0 (reference
 * temporal_sample.cu:453-511, and the masked pair count of
 * pipeline/__init__.py:206-219). */
int tgx_co_occurrence(const int32_t* a_ids, const int32_t* c_ids, const uint8_t* a_mask,
                      const uint8_t* c_mask, int64_t pairs, int32_t k, int32_t* a_cnt,
                      int32_t* c_cnt, float* pair_count, void* stream);

/* ---- Operators of a temporal attention model on prepared batches ----
 * No counterpart in the reference, whose models (tgengine/models, tgengine/nn) take
 * these steps in torch.  Values are TGX_F32 or TGX_BF16; sums, statistics and softmax
 * are held in 32 bits or more and each output is rounded once.  No floating-point
 * atomics: the same inputs give the same bits. */
#define TGX_MAX_EMBED_DIM 65536
#define TGX_MAX_NORM_DIM 16384
#define TGX_MAX_HEAD_DIM 256

/* out[i] = scale * table[ids[i]] for i < n, rows of dim values; an id outside
 * [0, rows) (the -1 of a padded neighbour) gives a row of zeros.  table: rows
 * `stride` values apart (at least dim, or 0: one row for all); ids int32 (ids_i32 != 0) or int64; out [n, dim]. */
int tgx_embed(const void* table, int64_t rows, int64_t dim, int64_t stride, int32_t dtype,
              const void* ids, int32_t ids_i32, int64_t n, float scale, void* out, void* stream);
/* Its gradient (n <= 2^29 - 64): grad [rows, dim], every row written: scale * the sum of dout[i] over
 * the i with that id, in an order that the ids alone decide.  workspace:
 * tgx_embed_grad_workspace_size(n, dim) bytes, 16-byte aligned, no initialisation. */
size_t tgx_embed_grad_workspace_size(int64_t n, int64_t dim);
int tgx_embed_grad(const void* dout, const void* ids, int32_t ids_i32, int64_t n, int64_t rows,
                   int64_t dim, int32_t dtype, float scale, void* grad, void* workspace,
                   size_t workspace_bytes, void* stream);

/* Layer norm of `rows` rows of dim values (x: `stride` values apart; out [rows, dim]):
 * (x - mean) * rstd * weight + bias with rstd = 1 / sqrt(var + eps), var the mean of
 * squares about the mean.  weight and bias [dim] of wdtype, either may be NULL.  mean
 * and rstd [rows]: both set (the gradient reads them) or both NULL. */
int tgx_layer_norm(const void* x, int64_t rows, int64_t dim, int64_t stride, int32_t dtype,
                   const void* weight, const void* bias, int32_t wdtype, float eps, void* out,
                   float* mean, float* rstd, void* stream);
/* Its gradient: dx [rows, dim], dw and db [dim] of wdtype; each may be NULL.  dy
 * [rows, dim].  workspace (needed with dw or db):
 * tgx_layer_norm_grad_workspace_size(rows, dim) bytes, 16-byte aligned. */
size_t tgx_layer_norm_grad_workspace_size(int64_t rows, int64_t dim);
int tgx_layer_norm_grad(const void* x, const void* dy, int64_t rows, int64_t dim, int64_t stride,
                        int32_t dtype, const void* weight, int32_t wdtype, const float* mean,
                        const float* rstd, void* dx, void* dw, void* db, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Attention of lq query tokens to lk states of another sequence, per batch row and
 * head; query head h reads key/value head h / (heads / kv_heads).  Element (b, i, h, c)
 * of q is q[b * q_stride[0] + i * q_stride[1] + h * q_stride[2] + c], k and v alike
 * with kv_heads; a stride may be 0 (a broadcast input).  mask: NULL, or bytes at
 * mask[b * mask_stride + j], 0 = key j takes no part (its k and v are not used,
 * whatever they hold).  A row that keeps no key gives zeros and takes no gradient.
 * out [batch, lq, heads, dim]; lse float [batch, lq, heads], the log of each row's sum
 * of exp(scale q.k) (-inf without a key): NULL, or kept for the gradient. */
typedef struct tgx_attention_args {
  const void* q;
  const void* k;
  const void* v;
  const uint8_t* mask;
  int64_t batch;
  int64_t lq;
  int64_t lk;
  int32_t heads;
  int32_t kv_heads;
  int32_t dim;             /* 1 .. TGX_MAX_HEAD_DIM */
  int32_t dtype;
  int64_t q_stride[3];     /* batch, token, head */
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t mask_stride;
  float scale;
  int32_t reserved;
  void* out;
  float* lse;
  void* out_rest;          /* TGX_BF16: NULL, or [batch, lq, heads, dim] for what rounding took
                              from out, which the gradient's inner products then add again */
  /* tgx_attention_grad: out, lse and out_rest as tgx_attention wrote them, grad_out
   * [batch, lq, heads, dim]; grad_q of q's shape, grad_k and grad_v
   * [batch, lk, kv_heads, dim], each may be NULL */
  const void* grad_out;
  void* grad_q;
  void* grad_k;
  void* grad_v;
  void* workspace;         /* 16-byte aligned, no initialisation; NULL when 0 bytes are needed */
  size_t workspace_bytes;
} tgx_attention_args;

/* bytes of workspace that the call of the same arguments needs (0 for arguments that
 * it refuses) */
size_t tgx_attention_workspace_size(const tgx_attention_args* args);
size_t tgx_attention_grad_workspace_size(const tgx_attention_args* args);
int tgx_attention(const tgx_attention_args* args, void* stream);
int tgx_attention_grad(const tgx_attention_args* args, void* stream);

/* Clipping by the global norm: norm[0] = sqrt(sum of squares over all `count` tensors),
 * outs[t] = grads[t] * min(1, max_norm / (norm + 1e-6)).  The arrays are host arrays,
 * read during the call; tensor t is sizes[t] contiguous values of dtypes[t], its output
 * of out_dtypes[t] may be the tensor itself (same dtype); outputs that overlap otherwise,
 * each other or a tensor, are refused (TGX_ERR_ARG).
 * A NaN or infinite norm scales as the formula says.  workspace:
 * tgx_clip_grad_norm_workspace_size(sizes, count) bytes. */
size_t tgx_clip_grad_norm_workspace_size(const int64_t* sizes, int64_t count);
int tgx_clip_grad_norm(const void* const* grads, const int32_t* dtypes, void* const* outs,
                       const int32_t* out_dtypes, const int64_t* sizes, int64_t count,
                       float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                       void* stream);

/* A gated recurrence along the tokens of every batch row, over dim channels:
 *   h_t = a_t h_{t-1} + (1 - a_t) x_t,  a_t = sigmoid(gate_t);  a masked token: h_t = h_{t-1}
 * from h_0 = state (zeros without one).  Element (b, t, c) of x is x[b * x_stride[0] + t *
 * x_stride[1] + c], gate alike; a stride may be 0, but not below.  mask: NULL, or bytes at mask[b *
 * mask_stride + t], 0 = token t takes no part (its x and gate are not used, whatever they
 * hold).  out [batch, length, dim] holds every h_t rounded, last [batch, dim] the last one.  What is
 * written may share no memory with what is read. */
typedef struct tgx_scan_args {
  const void* x;
  const void* gate;
  const uint8_t* mask;
  const float* state;      /* NULL or [batch, dim] */
  int64_t batch;
  int64_t length;
  int64_t dim;
  int64_t x_stride[2];     /* batch, token */
  int64_t gate_stride[2];
  int64_t mask_stride;
  int32_t dtype;
  int32_t reserved;
  void* out;
  float* last;
  float* starts;           /* NULL, or [batch, tgx_scan_starts(length), dim]: states within the rows,
                              which the gradient reads */
  /* tgx_scan_grad: starts as tgx_scan wrote them (out and last are not read); grad_out
   * [batch, length, dim] and grad_last [batch, dim], each NULL for zeros; grad_x and
   * grad_gate [batch, length, dim]; grad_state NULL or [batch, dim] */
  const void* grad_out;
  const float* grad_last;
  void* grad_x;
  void* grad_gate;
  float* grad_state;
  void* workspace;         /* 16-byte aligned, no initialisation; NULL when 0 bytes are needed */
  size_t workspace_bytes;
} tgx_scan_args;

int64_t tgx_scan_starts(int64_t length);
/* bytes of workspace that tgx_scan or tgx_scan_grad of these arguments needs (0 for
 * arguments that they refuse) */
size_t tgx_scan_workspace_size(const tgx_scan_args* args);
int tgx_scan(const tgx_scan_args* args, void* stream);
int tgx_scan_grad(const tgx_scan_args* args, void* stream);

/* The residual sum after a block and the norm before the next one, over `rows` rows of dim
 * values:
 *   sum = residual + scale sigmoid(gate) n,  n = x or norm(x) post_weight
 *   out = norm(sum) weight + bias,  norm(v) = (v - mean v) / sqrt(var v + eps)
 * scale, weight, bias and post_weight [dim] of wdtype; gate, scale, post_weight (then n = x),
 * weight and bias may be NULL.  center = 0: norm(v) = v / sqrt(mean v^2 + eps).  Rows of x,
 * residual and gate are their strides apart; out and sum [rows, dim].  What is written may share
 * no memory with what is read. */
typedef struct tgx_residual_norm_args {
  const void* x;
  const void* residual;
  const void* gate;
  const void* weight;
  const void* bias;
  const void* scale;
  const void* post_weight;
  int64_t rows;
  int64_t dim;             /* 1 .. TGX_MAX_NORM_DIM */
  int64_t x_stride;
  int64_t residual_stride;
  int64_t gate_stride;
  int32_t dtype;
  int32_t wdtype;
  int32_t center;
  float eps;
  void* out;
  void* sum;
  float* stats;            /* NULL, or kept for the gradient: [2, rows], with post_weight [4, rows] */
  /* tgx_residual_norm_grad: stats as tgx_residual_norm wrote them (out and sum are not read);
   * grad_out and grad_sum [rows, dim], each NULL for zeros; every other may be NULL.  Without
   * gate, scale and post_weight the gradient of x is grad_residual (grad_x has to be NULL), and
   * x may hold the sum instead, with residual NULL. */
  const void* grad_out;
  const void* grad_sum;
  void* grad_x;
  void* grad_residual;
  void* grad_gate;
  void* grad_weight;
  void* grad_bias;
  void* grad_scale;
  void* grad_post_weight;
  void* workspace;         /* 16-byte aligned, no initialisation; needed with a gradient of wdtype */
  size_t workspace_bytes;
} tgx_residual_norm_args;

int tgx_residual_norm(const tgx_residual_norm_args* args, void* stream);
size_t tgx_residual_norm_grad_workspace_size(const tgx_residual_norm_args* args);
int tgx_residual_norm_grad(const tgx_residual_norm_args* args, void* stream);

/* One AdamW step over `count` tensors: t = *step + 1 is written back,
 *   g = grad * min(1, max_norm / (*grad_norm + 1e-6))      (grad_norm NULL: grad)
 *   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
 *   param = param (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
 * The table is a host array, read during the call; step, lr_device (in place of lr) and
 * grad_norm are on the device, so that a captured step counts, and takes a new rate and norm,
 * at every replay.  bits = 32: exp_avg and exp_avg_sq hold m and v in f32.  bits = 8: m and
 * sqrt(v) as e4m3 (OCP, with NaN, without infinities) times scales [2][blocks], a power of two
 * for each TGX_ADAMW_BLOCK values, the last block with what is left; all zeros before the first step.  They are
 * rounded down or up by a dither of the value's place and t, and a second average above zero stays
 * so.  Memory that is written may overlap nothing else (TGX_ERR_ARG). */
#define TGX_ADAMW_BLOCK 256
typedef struct tgx_adamw_tensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* scales;           /* NULL with 32 bits */
  int64_t* step;           /* one value */
  int64_t size;            /* values, one after the other */
  int32_t dtype;
  int32_t grad_dtype;
  int32_t bits;
  int32_t reserved;
} tgx_adamw_tensor;

typedef struct tgx_adamw_args {
  const tgx_adamw_tensor* tensors;
  int64_t count;           /* at most 65535 */
  double lr;
  double beta1;
  double beta2;
  double eps;
  double weight_decay;
  double max_norm;
  const float* lr_device;  /* NULL: lr */
  const float* grad_norm;  /* NULL: gradients as they are */
  void* workspace;         /* tgx_adamw_workspace_size(count) bytes, 16-byte aligned, no initialisation */
  size_t workspace_bytes;
} tgx_adamw_args;

size_t tgx_adamw_workspace_size(int64_t count);
int tgx_adamw(const tgx_adamw_args* args, void* stream);

const char* tgx_last_error(void);
int tgx_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* TGX_H */
