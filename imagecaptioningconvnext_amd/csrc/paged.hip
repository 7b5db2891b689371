// Paged key/value cache of incremental decoding: page planning from the requests' lengths, the
// writer of new tokens' keys and values, and attention of one new token per request.
//
// A cache is [pages][page][kv heads][dh] (any strides, unit inner one); a request owns the pages
// that its row of the table names, position p of it sits in slot table[p / page] * page + p % page.
#include "common.h"

namespace imgcap {

// ---- page planning ------------------------------------------------------------------------
// Integer prefix sums give each request its place on the stack of free pages and its first token;
// every token then finds its request by bisection of the starts.  A step of up to PLAN_ROWS requests
// is one pass of one workgroup with 32-bit sums in the lanes; up to PLAN_TOKENS tokens it also lays
// out the tokens itself, from LDS.  It is latency that counts there, so loads come in two rounds: the
// lengths and the stack's height; then the pages that requests have open, the top of the stack and the
// pages of ended requests, all of which the tokens find in LDS.  Barriers wait for LDS alone, not for
// the global stores and loads on their way (64 requests, five of them ended: 3.2 us; with a pass over
// the requests' pages and loads one after another 8.2).  More tokens go to a second launch over the
// whole chip; more requests (or sums that might pass 32 bits) to a pass in chunks with 64-bit sums.
constexpr int PLAN_ROWS = 1024, PLAN_TOKENS = 4096, PLAN_CAP = 1 << 20, PLAN_BACK = 2048;

struct PlanArgs : imgcap_paged_plan_desc { int lp; };  // lp: log2 of the page size

DEV int wave_scan_incl(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15: row 0 -> 1, 2 -> 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31: rows 0, 1 -> 2, 3
  return v;
}
DEV long wave_scan_incl(long v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long u = __shfl_up(v, o, 64);
    if ((int)(threadIdx.x & 63) >= o) v += u;
  }
  return v;
}
// inclusive prefix over the block; `total` gets the block's sum.  red: blockDim / 64 values.
DEV long block_scan_incl(long v, long* red, long& total) {
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  v = wave_scan_incl(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[w] = v;
  __syncthreads();
  long before = 0, all = 0;
  for (int i = 0; i < nw; ++i) {
    if (i < w) before += red[i];
    all += red[i];
  }
  total = all;
  return v + before;
}
// a barrier of what lies in LDS
DEV void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// inclusive prefixes of two values over the block and their sums; red: 16 pairs
DEV void block_scan2(int& a, int& b, int2* red, int& sum_a, int& sum_b) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, nw = blockDim.x >> 6;
  a = wave_scan_incl(a);
  b = wave_scan_incl(b);
  if (nw == 1) {
    sum_a = __builtin_amdgcn_readlane(a, 63);
    sum_b = __builtin_amdgcn_readlane(b, 63);
    return;
  }
  lds_barrier();
  if (lane == 63) red[w] = make_int2(a, b);
  lds_barrier();
  const int2 mine = lane < nw ? red[lane] : make_int2(0, 0);
  const int ia = wave_scan_incl(mine.x), ib = wave_scan_incl(mine.y);
  sum_a = __builtin_amdgcn_readlane(ia, 63);
  sum_b = __builtin_amdgcn_readlane(ib, 63);
  const int uw = __builtin_amdgcn_readfirstlane(w);
  if (uw > 0) {
    a += __builtin_amdgcn_readlane(ia, uw - 1);
    b += __builtin_amdgcn_readlane(ib, uw - 1);
  }
}

// the request of token i: starts[r] <= i < starts[r + 1] (n requests; the last of those that start alike)
DEV int plan_row(const int32_t* starts, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}
DEV void plan_put(const PlanArgs& a, int i, int row, long pos, int id) {
  const int off = (int)pos & ((1 << a.lp) - 1);
  a.slots[i] = (unsigned)id < (unsigned)a.pool ? ((int64_t)id << a.lp) + off : -1;
  a.rows[i] = row;
  a.positions[i] = pos;
}
DEV void plan_none(const PlanArgs& a, int i) {
  a.slots[i] = -1;
  a.rows[i] = -1;
  a.positions[i] = 0;
}
// the token that opens a page enters it into the table
DEV void plan_enter(const PlanArgs& a, int row, int pi, long pos, int id) {
  if (((int)pos & ((1 << a.lp) - 1)) == 0) a.table[(long)row * a.table_row + pi] = id;
}

__global__ __launch_bounds__(PLAN_ROWS) void paged_plan_kernel(PlanArgs a, int expand) {
  __shared__ int2 red[16];
  __shared__ int starts_s[PLAN_ROWS], at_s[PLAN_ROWS], past_s[PLAN_ROWS], open_s[PLAN_ROWS];
  __shared__ int before_s[PLAN_ROWS], stack_s[PLAN_ROWS], push_s[PLAN_BACK];
  // the arguments in one go: the compiler would fetch each where it is first used, one wait after another
  asm volatile("" ::"s"(a.B), "s"(a.past), "s"(a.add), "s"(a.count), "s"(a.table), "s"(a.free_ids), "s"(a.lp), "s"(a.pool),
               "s"(a.width), "s"(a.tokens));
  const int T = blockDim.x, b = threadIdx.x, page = 1 << a.lp;
  const bool in = b < a.B;
  const int past = in ? a.past[b] : 0, add = in ? a.add[b] : -1;
  const int height = min(max(*a.count, 0), a.pool);
  const long lp = past, la = add, room = (long)a.width << a.lp;
  const bool live = add >= 0;
  const int have = (int)((max(lp, 0l) + page - 1) >> a.lp);
  int open = -1, under = -1;  // the page that the request's next token goes to; the b-th page from the stack's top
  if (live && past > 0 && (past & (page - 1)) && (past >> a.lp) < a.width) open = a.table[b * a.table_row + (past >> a.lp)];
  if (expand && b < height) under = a.free_ids[height - 1 - b];
  const int back = in && !live ? min(have, a.width) : 0;
  bool fits = live && past >= 0 && lp + la <= room;
  const int asked = fits ? min(add, a.tokens + 1) : 0;  // one past the capacity is as far as it counts
  int tok = asked, given = back, asked_all, back_all, need_all, none;
  block_scan2(tok, given, red, asked_all, back_all);
  fits = fits && tok <= a.tokens;
  const int need = fits ? (int)((lp + la + page - 1) >> a.lp) - have : 0;
  int upto = need, zero = 0;
  block_scan2(upto, zero, red, need_all, none);
  const int top = (int)min((long)height + back_all, (long)a.pool);
  if (back_all > 0) {  // pages of ended requests go back on the stack, in the requests' order
    before_s[b] = given - back;
    lds_barrier();
    for (int at = b; at < back_all; at += T) {
      const int r = plan_row(before_s, a.B, at), id = a.table[r * a.table_row + (at - before_s[r])];
      if ((long)height + at < a.pool) a.free_ids[height + at] = id;
      if (at < PLAN_BACK) push_s[at] = id;
    }
  }
  const bool granted = fits && (need == 0 || upto <= top);
  int start = tok - asked, total = asked_all, used = need_all;
  if (asked_all > a.tokens || need_all > top) {  // some request waits: what the others get, again
    int got = granted ? add : 0, took = granted ? need : 0;
    block_scan2(got, took, red, total, used);
    start = got - (granted ? add : 0);
  }
  if (in) {
    a.lens[b] = live ? past + (granted ? add : 0) : 0;
    a.starts[b] = start;
    a.waits[b] = live && !granted ? 1 : 0;
  }
  if (b == 0) {
    a.starts[a.B] = total;
    *a.count_out = top - used;
  }
  if (!expand) {
    if (in) a.ws[b] = upto - need;
    if (b == 0) a.ws[a.B] = top;
    return;
  }
  starts_s[b] = start;
  at_s[b] = top - 1 - (upto - need);
  past_s[b] = past;
  open_s[b] = open;
  stack_s[b] = under;
  if (back_all > PLAN_BACK) __syncthreads();  // some of the pages put back are read from the stack
  else lds_barrier();
  for (int i = b; i < a.tokens; i += T) {
    if (i >= total) {
      plan_none(a, i);
      continue;
    }
    const int r = plan_row(starts_s, a.B, i), p0 = past_s[r];
    const long pos = (long)p0 + (i - starts_s[r]);
    const int pi = (int)(pos >> a.lp), h = (int)(((long)p0 + page - 1) >> a.lp);
    int id = open_s[r];
    if (pi >= h) {  // a page of the stack: place `at`, counted from its bottom
      const int at = at_s[r] - (pi - h), pushed = at - height, deep = height - 1 - at;
      id = pushed >= 0 && pushed < PLAN_BACK ? push_s[pushed] : deep >= 0 && deep < T ? stack_s[deep] : a.free_ids[at];
      plan_enter(a, r, pi, pos, id);
    }
    plan_put(a, i, r, pos, id);
  }
}

// any number of requests: chunks of the workgroup's width, 64-bit sums
__global__ __launch_bounds__(1024) void paged_plan_long_kernel(PlanArgs a) {
  __shared__ long red[16];
  __shared__ long base_s[1024];
  __shared__ int back_s[1024];
  const int T = blockDim.x, tid = threadIdx.x;
  const int page = 1 << a.lp;
  const long room = (long)a.width << a.lp;
  long top = min(max(*a.count, 0), a.pool);
  for (int b0 = 0; b0 < a.B; b0 += T) {
    const int b = b0 + tid;
    long back = 0;
    if (b < a.B && a.add[b] < 0) back = min(((long)max(a.past[b], 0) + page - 1) >> a.lp, (long)a.width);
    if (!__syncthreads_or(back > 0)) continue;
    long total;
    const long upto = block_scan_incl(back, red, total);
    base_s[tid] = top + upto - back;
    back_s[tid] = (int)back;
    __syncthreads();
    const int n = min(T, a.B - b0);
    for (int r = tid >> 6; r < n; r += T >> 6)
      for (int j = tid & 63; j < back_s[r]; j += 64)
        if (base_s[r] + j < a.pool) a.free_ids[base_s[r] + j] = a.table[(long)(b0 + r) * a.table_row + j];
    top = min(top + total, (long)a.pool);
    __syncthreads();
  }
  long tok0 = 0, page0 = 0, out0 = 0, used = 0;
  for (int b0 = 0; b0 < a.B; b0 += T) {
    const int b = b0 + tid;
    const bool in = b < a.B;
    const long past = in ? a.past[b] : 0, add = in ? a.add[b] : -1;
    const bool live = add >= 0;
    bool fits = live && past >= 0 && past + add <= room;
    long total;
    const long tok = tok0 + block_scan_incl(fits ? add : 0l, red, total);
    tok0 += total;
    fits = fits && tok <= a.tokens;
    const long have = (max(past, 0l) + page - 1) >> a.lp;
    const long need = fits ? ((past + add + page - 1) >> a.lp) - have : 0;
    const long upto = page0 + block_scan_incl(need, red, total);
    page0 += total;
    const bool granted = fits && (need == 0 || upto <= top);
    const long out = out0 + block_scan_incl(granted ? add : 0l, red, total);
    out0 += total;
    block_scan_incl(granted ? need : 0l, red, total);
    used += total;
    if (in) {
      a.lens[b] = live ? (int)(past + (granted ? add : 0)) : 0;
      a.starts[b] = (int)(out - (granted ? add : 0));
      a.waits[b] = live && !granted ? 1 : 0;
      a.ws[b] = (int)(upto - need);
    }
  }
  if (tid == 0) {
    a.starts[a.B] = (int)out0;
    a.ws[a.B] = (int)top;
    *a.count_out = (int)(top - used);
  }
}

// lays out the tokens after either planner: four consecutive ones a thread (one search for them, 16-byte
// stores where the outputs are so aligned), the starts in LDS if they fit.  Bound by latency and the
// 20 bytes a token that it writes (500,250 tokens of 500 requests 7.4 us; a token a thread 9.4).  A
// request's old length is its new one less its tokens (past itself may be the array that the new ones
// went to).
constexpr int SLOT_TOKENS = 1024, SLOT_ROWS = 4096;
__global__ __launch_bounds__(256) void paged_slots_kernel(PlanArgs a, int aligned) {
  __shared__ int32_t starts_s[SLOT_ROWS];
  asm volatile("" ::"s"(a.B), "s"(a.lens), "s"(a.starts), "s"(a.ws), "s"(a.table), "s"(a.free_ids), "s"(a.lp), "s"(a.pool),
               "s"(a.slots), "s"(a.rows), "s"(a.positions), "s"(a.tokens));  // in one go
  const int32_t* starts = a.starts;
  const int total = a.starts[a.B], top = a.ws[a.B], page = 1 << a.lp;
  const long i0 = (long)blockIdx.x * SLOT_TOKENS + 4 * threadIdx.x;
  if (a.B <= SLOT_ROWS) {
    for (int i = threadIdx.x; i < a.B; i += 256) starts_s[i] = a.starts[i];
    __syncthreads();
    starts = starts_s;
  }
  if (i0 >= a.tokens) return;
  int r = plan_row(starts, a.B, (int)min(i0, (long)total)), begin = starts[r];
  int end = r + 1 < a.B ? starts[r + 1] : total, p0 = a.lens[r] - (end - begin), at = top - 1 - a.ws[r], known = -1, id = -1;
  int64_t slot[4], position[4];
  int32_t row[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long i = i0 + j;
    slot[j] = -1;
    position[j] = 0;
    row[j] = -1;
    if (i >= total || i >= a.tokens) continue;
    if (i >= end) {  // the next request that has a token here
      do {
        begin = end;
        ++r;
        end = r + 1 < a.B ? starts[r + 1] : total;
      } while (i >= end);
      p0 = a.lens[r] - (end - begin);
      at = top - 1 - a.ws[r];
      known = -1;
    }
    const long pos = (long)p0 + (i - begin);
    const int pi = (int)(pos >> a.lp), h = (int)(((long)p0 + page - 1) >> a.lp), off = (int)pos & (page - 1);
    if (pi != known) id = pi < h ? a.table[(long)r * a.table_row + pi] : a.free_ids[at - (pi - h)];
    known = pi;
    if (pi >= h && off == 0) a.table[(long)r * a.table_row + pi] = id;
    slot[j] = (unsigned)id < (unsigned)a.pool ? ((int64_t)id << a.lp) + off : -1;
    position[j] = pos;
    row[j] = r;
  }
  if (aligned && i0 + 4 <= a.tokens) {
    *(longlong2*)(a.slots + i0) = make_longlong2(slot[0], slot[1]);
    *(longlong2*)(a.slots + i0 + 2) = make_longlong2(slot[2], slot[3]);
    *(longlong2*)(a.positions + i0) = make_longlong2(position[0], position[1]);
    *(longlong2*)(a.positions + i0 + 2) = make_longlong2(position[2], position[3]);
    *(int4*)(a.rows + i0) = make_int4(row[0], row[1], row[2], row[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < a.tokens) {
        a.slots[i0 + j] = slot[j];
        a.positions[i0 + j] = position[j];
        a.rows[i0 + j] = row[j];
      }
  }
}

// ---- cache writer -------------------------------------------------------------------------
// 16 bytes a thread: token, head and vector of a unit; slots outside the cache are skipped.  Bound by
// HBM: 20,001 tokens of 8 x 128 bf16 (164 MB read and written) 31.8 us, 5.2 TB/s; 64 of 8 x 64 2.6 us.
__global__ __launch_bounds__(256) void paged_write_kernel(imgcap_paged_write_desc d, int vecs, int lp, int esz) {
  const unsigned per = (unsigned)d.heads * vecs;
  const unsigned u = blockIdx.x * 256u + threadIdx.x;
  if (u >= per * (unsigned)d.n) return;
  const unsigned tok = u / per, rest = u - tok * per, head = rest / vecs, vec = rest - head * vecs;
  const long slot = d.slots[tok];
  if (slot < 0 || (slot >> lp) >= d.pages) return;
  const long pg = slot >> lp, off = slot & (d.page - 1);
  const bool second = blockIdx.y != 0;
  const char* src = (const char*)(second ? d.v : d.k);
  char* dst = (char*)(second ? d.vc : d.kc);
  src += ((long)tok * (second ? d.v_row : d.k_row) + (long)head * (second ? d.v_head : d.k_head)) * esz + vec * 16;
  dst += (pg * (second ? d.vc_page : d.kc_page) + off * (second ? d.vc_tok : d.kc_tok) +
          (long)head * (second ? d.vc_head : d.kc_head)) * esz + vec * 16;
  *(uint4*)dst = *(const uint4*)src;
}

// ---- attention of one new token per request --------------------------------------------------
// Row = (request, kv head, 16 of the query heads that share it).  A wave takes 32 tokens a step:
//   S^T[token][head] = K Q^T   (A = 16 tokens of K, B = the queries; the accumulator's column is a
//                               head, its rows 4 tokens per lane group)
//   O^T[dh][head]  += V^T P^T  (B = those very registers: lane group g holds tokens 4g..4g+3 of each
//                               16, so the product's k order is taken to be that, and V's rows are
//                               read in it: no exchange between lanes, nothing through LDS)
// with a running maximum and sum per head (base 2).  A lane of V holds DH / 16 consecutive columns
// of its 4 + 4 tokens; the transposed operand is byte permutes of those words.  fp32 does the same
// on the exact fp32 instruction, whose k is one token per lane group.
// Positions past the length, or on a page outside the cache, are not there: score -inf, V zeroed.
template <int BYTES> struct Words { uint32_t w[BYTES / 4]; };
template <int BYTES> DEV Words<BYTES> load_words(const void* p) {
  Words<BYTES> r;
  if constexpr (BYTES == 8) {
    const uint2 u = *(const uint2*)p;
    r.w[0] = u.x; r.w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 u = ((const uint4*)p)[i];
      r.w[4 * i] = u.x; r.w[4 * i + 1] = u.y; r.w[4 * i + 2] = u.z; r.w[4 * i + 3] = u.w;
    }
  }
  return r;
}

// The pages of a wave's steps (32 tokens each), looked up a step before their use; -1 for an id outside
// the cache.  Pages of 16 tokens and more: 16 tokens share a page, lanes 0 and 1 hold those of the two
// halves.  TINY: a lane holds the page of its own token r of either half.
template <bool TINY> struct Pages {
  static constexpr int N = TINY ? 2 : 1;
  const int32_t* table;
  int now[N], then[N];
  int lp, last, pages;
  DEV void look(int (&to)[N], int tok) const {
    const int lane = threadIdx.x & 63, own = TINY ? lane & 15 : 16 * (lane & 1);
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = table[min((tok + 16 * i + own) >> lp, last)];
  }
  // nothing here waits for the request's length: entries past it are as good as any
  DEV Pages(const imgcap_paged_attn_desc& d, const int32_t* row, int tok, int step, int lp_)
      : table(row), lp(lp_), last(d.width - 1), pages(d.pages) {
    look(now, tok);
    look(then, tok + step);
  }
  // the pages of the step at tok, if there is one; steps are taken in order.  No branch: a load under
  // one would be waited for, and all before it, where the paths meet.
  DEV void take(int (&id)[2], int tok, int step, bool more) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = TINY ? now[h % N] : __builtin_amdgcn_readlane(now[0], h);
      id[h] = !more ? id[h] : (unsigned)e < (unsigned)pages ? e : -1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) now[i] = then[i];
    look(then, tok + 2 * step);
  }
};

// 32 tokens of one kv head as a wave's operands.  A page outside the cache reads page 0, and its
// tokens are masked.
template <typename T, int DH, bool TINY> struct KvTile {
  static constexpr int NS = DH * sizeof(T) / 64;   // 16-byte pieces of a key row per lane
  static constexpr int VB = DH / 16 * sizeof(T);   // bytes of a value row per lane
  uint4 k[2][NS];
  Words<VB> v[2][4];
  int id[2];  // page of each half (TINY: of token r of it), -1 if outside the cache
  DEV void load_k(const imgcap_paged_attn_desc& d, const T* kb, int tok, int r, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* kp = kb + (long)max(id[h], 0) * d.k_page + ((tok + 16 * h + r) & (d.page - 1)) * d.k_tok + g * (16 / sizeof(T));
#pragma unroll
      for (int s = 0; s < NS; ++s) k[h][s] = *(const uint4*)(kp + s * (64 / sizeof(T)));
    }
  }
  DEV void load_v(const imgcap_paged_attn_desc& d, const T* vb, int tok, int r, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* vp = vb + r * (DH / 16);
      if (!TINY) vp += (long)max(id[h], 0) * d.v_page + ((tok + 16 * h + 4 * g) & (d.page - 1)) * d.v_tok;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* at = vp + i * d.v_tok;
        if (TINY)
          at = vp + (long)max(__shfl(id[h], 4 * g + i, 64), 0) * d.v_page + ((tok + 16 * h + 4 * g + i) & (d.page - 1)) * d.v_tok;
        v[h][i] = load_words<VB>(at);
      }
    }
  }
  // whether lane-group token i of half h is a live position
  DEV bool live(int h, int i, int tok, int t1, int g) const {
    return (TINY ? __shfl(id[h], 4 * g + i, 64) : id[h]) >= 0 && tok + 16 * h + 4 * g + i < t1;
  }
  DEV bool all_live(int tok, int t1) const {
    return tok + 32 <= t1 && !__any(id[0] < 0 || id[1] < 0);
  }
};

// over the four lane groups (lane ^ 16, lane ^ 32), on swaps of 16 and of 32 lanes: after either, a
// lane holds its own group's value and its partner's
template <typename F> DEV float groups_fold(float v, F f) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t x0 = x[0], x1 = x[1];
  v = f(__builtin_bit_cast(float, x0), __builtin_bit_cast(float, x1));
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t y0 = y[0], y1 = y[1];
  return f(__builtin_bit_cast(float, y0), __builtin_bit_cast(float, y1));
}

DEV uint32_t pack_bf16(float a, float b) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (bf16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (bf16)b) << 16);
}

// what is left of weight a beside its top bits, but at least the smallest normal number; a itself where that
// is less, so that the value of a weight of 0 adds nothing, however large (the rest is at most a: one
// median says all of it)
DEV float weight_rest(float a, float top) { return __builtin_amdgcn_fmed3f(a, a - top, 0x1p-126f); }

// JOIN: the workgroup's waves share a chunk (blockIdx.x the row, blockIdx.y the chunk), 32 tokens each
// in turn, and put their parts together in LDS.  Else each wave has a short row to itself, the waves of
// a group consecutive rows (kv heads of the same tokens, which lie side by side in memory), and
// nothing is exchanged.  Bound by HBM where the caches are large, and more waves than two a SIMD
// only lengthen the queues there (first scores of a wave after 16 us at 12 waves a CU): 48 requests of
// up to 20011 tokens 393 us at two, 401 at three.
constexpr int JOIN_WAVES = 4, MAX_SPLIT = 1024;
static_assert(JOIN_WAVES % 2 == 0, "half of the waves hand over to the other half");
template <typename T, int DH, bool TINY, bool JOIN>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_attn_kernel(
    imgcap_paged_attn_desc d, int chunk, int nsplit, int gtiles, int lp, float* ws_o, float* ws_ml) {
  using Tile = KvTile<T, DH, TINY>;
  constexpr int VPL = DH / 16, LDO = DH + 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int row = JOIN ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + w;
  if (!JOIN && row >= d.B * d.Hkv * gtiles) return;
  const int gt = row % gtiles, kvh = (row / gtiles) % d.Hkv, b = row / gtiles / d.Hkv;
  const int split = blockIdx.y, G = d.H / d.Hkv, heads = min(16, G - 16 * gt), h0 = kvh * G + 16 * gt;
  const int t0 = split * chunk, step = JOIN ? 32 * JOIN_WAVES : 32;
  const int32_t* table = d.table + (long)b * d.table_row;
  int tok = t0 + (JOIN ? 32 * w : 0);
  Tile t;
  Pages<TINY> pages(d, table, tok, step, lp);
  int len = __builtin_amdgcn_readfirstlane(d.lens[b]);
  asm volatile("" : "+v"(pages.now[0]), "+s"(len));  // loaded side by side, not one after the other
  const int n = min(max(len, 0), d.max_len);
  if (split > 0 && t0 >= n) return;
  const int t1 = t0 + min(chunk, n - t0);  // t0 + chunk may pass 32 bits
  const T* kb = (const T*)d.k + (long)kvh * d.k_head;
  const T* vb = (const T*)d.v + (long)kvh * d.v_head;
  const float c = d.scale * 1.44269504088896341f;
  uint4 q[Tile::NS];
#pragma unroll
  for (int s = 0; s < Tile::NS; ++s) {
    q[s] = make_uint4(0u, 0u, 0u, 0u);
    if (r < heads)
      q[s] = *(const uint4*)((const T*)d.q + (long)b * d.q_row + (long)(h0 + r) * d.q_head + s * (64 / sizeof(T)) +
                             g * (16 / sizeof(T)));
  }
  f32x4 acc[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  if (tok < t1) {
    pages.take(t.id, tok, step, true);
    t.load_k(d, kb, tok, r, g);
    t.load_v(d, vb, tok, r, g);
    while (true) {
      const bool full = t.all_live(tok, t1), more = tok + step < t1;
      float p[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 s4 = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < Tile::NS; ++s) {
          if constexpr (sizeof(T) == 2) {
            s4 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, t.k[h][s]),
                                                         __builtin_bit_cast(bf16x8, q[s]), s4, 0, 0, 0);
          } else {
            const f32x4 kk = __builtin_bit_cast(f32x4, t.k[h][s]), qq = __builtin_bit_cast(f32x4, q[s]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], qq[e], s4, 0, 0, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) p[h][i] = s4[i] * c;
      }
      if (!full) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!t.live(h, i, tok, t1, g)) {
              p[h][i] = -INFINITY;
#pragma unroll
              for (int e = 0; e < Tile::VB / 4; ++e) t.v[h][i].w[e] = 0u;
            }
      }
      // the keys' registers are free: the next step's go out now, its values' after the product below
      // (after the last step this one's again, from the cache)
      pages.take(t.id, tok + step, step, more);
      const int ahead = more ? tok + step : tok;
      t.load_k(d, kb, ahead, r, g);
      float mx = fmaxf(fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[0][2], p[0][3])),
                       fmaxf(fmaxf(p[1][0], p[1][1]), fmaxf(p[1][2], p[1][3])));
      mx = groups_fold(mx, [](float x, float y) { return fmaxf(x, y); });
      if (__any(mx > m)) {  // seldom after the first steps of a long row
        const float mn = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        l *= alpha;
#pragma unroll
        for (int j = 0; j < VPL; ++j) acc[j] *= alpha;
      }
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[h][i] = __builtin_amdgcn_exp2f(p[h][i] - ms);
          l += p[h][i];
        }
      if constexpr (sizeof(T) == 2) {
        // the weights go in as their top bf16 bits and the remainder in bf16: 15 bits and more of them,
        // so the output carries little but its own rounding.  Both pieces of a weight above 0 are kept
        // positive (weight_rest): an infinite value times a zero or negative remainder would turn the
        // infinity into NaN.
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = p[e >> 1][2 * (e & 1)], bb = p[e >> 1][2 * (e & 1) + 1];
          hi[e] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, bb), __builtin_bit_cast(uint32_t, a), 0x07060302u);
          lo[e] = pack_bf16(weight_rest(a, __builtin_bit_cast(float, hi[e] << 16)),
                            weight_rest(bb, __builtin_bit_cast(float, hi[e] & 0xffff0000u)));
        }
        const bf16x8 ph = __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        const bf16x8 pl = __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
          const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[e] = __builtin_amdgcn_perm(t.v[e >> 1][2 * (e & 1) + 1].w[j >> 1], t.v[e >> 1][2 * (e & 1)].w[j >> 1], sel);
          const bf16x8 vf = __builtin_bit_cast(bf16x8, make_uint4(x[0], x[1], x[2], x[3]));
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph, acc[j], 0, 0, 0);
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl, acc[j], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < VPL; ++j)
              acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.v[h][i].w[j]), p[h][i], acc[j],
                                                            0, 0, 0);
      }
      if (!more) break;
      tok += step;
      t.load_v(d, vb, tok, r, g);
    }
  }
  l = groups_fold(l, [](float x, float y) { return x + y; });
  // lane (r, g) holds head r, columns VPL * (4 g + i) + j: DH / 4 consecutive ones
  if constexpr (!JOIN) {  // rows that are not split
    if (r >= heads) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    T* o = (T*)d.o + (long)b * d.o_row + (long)(h0 + r) * d.o_head + VPL * 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VPL; ++j) o[VPL * i + j] = from_f<T>(l == 0.f ? 0.f : acc[j][i] * f);
    if (d.lse && g == 0) d.lse[(long)b * d.H + h0 + r] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
  } else {
    const bool whole = n <= chunk;
    __shared__ float ml[JOIN_WAVES][2][16];
    __shared__ float sm[JOIN_WAVES / 2 * 16 * LDO];  // parts, to the common maximum
    if (g == 0) {
      ml[w][0][r] = m;
      ml[w][1][r] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < JOIN_WAVES; ++i) M = fmaxf(M, ml[i][0][r]);
    const float ms = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < JOIN_WAVES; ++i) L += __builtin_amdgcn_exp2f(ml[i][0][r] - ms) * ml[i][1][r];
    const float f = __builtin_amdgcn_exp2f(m - ms) * (!whole ? 1.f : L == 0.f ? 0.f : 1.f / L);
    // half of the waves hand their parts to the other half, lane to lane: that many parts lie in LDS
    constexpr int HALF = JOIN_WAVES / 2;
    float* so = sm + (w % HALF * 16 + r) * LDO + VPL * 4 * g;
    if (w >= HALF) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VPL; j += 4)
          *(f32x4*)(so + VPL * i + j) = f * f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
    }
    __syncthreads();
    if (w < HALF) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VPL; j += 4)
          *(f32x4*)(so + VPL * i + j) += f * f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
    }
    __syncthreads();
    for (int e = threadIdx.x; e < heads * (DH / 4); e += 64 * JOIN_WAVES) {
      const int hd = e / (DH / 4), col = 4 * (e % (DH / 4));
      const long bh = (long)b * d.H + h0 + hd;
      f32x4 o = *(const f32x4*)(sm + hd * LDO + col);
#pragma unroll
      for (int i = 1; i < HALF; ++i) o += *(const f32x4*)(sm + (i * 16 + hd) * LDO + col);
      if (whole) {
        T* out = (T*)d.o + (long)b * d.o_row + (long)(h0 + hd) * d.o_head + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = from_f<T>(o[i]);
      } else {
        *(f32x4*)(ws_o + (bh * nsplit + split) * DH + col) = o;
      }
    }
    if (w == 0 && g == 0 && r < heads) {
      const long bh = (long)b * d.H + h0 + r;
      if (!whole) *(f32x2*)(ws_ml + (bh * nsplit + split) * 2) = f32x2{M, L};
      else if (d.lse) d.lse[bh] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
    }
  }
}

// joins the chunks of a row: out = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s.  A workgroup takes COLS
// columns of one (request, head): all of them where there are rows enough to fill the chip, 32 where
// there are few (a single long request of 16 heads over 391 chunks: 15.6 us by whole rows, one
// workgroup a head; 241 chunks 3.9 us by 32 columns).  The chunks' factors are worked out once, in
// LDS, while the first outputs are on their way.
template <typename T, int DH, int COLS>
__global__ __launch_bounds__(256) void paged_join_kernel(imgcap_paged_attn_desc d, int chunk, int nsplit,
                                                         const float* __restrict__ ws_o, const float* __restrict__ ws_ml) {
  constexpr int C4 = COLS / 4, PARTS = 256 / C4;
  __shared__ float red[8];
  __shared__ float factor[MAX_SPLIT];
  __shared__ f32x4 part[PARTS][C4];
  const int row = blockIdx.x / (DH / COLS), c0 = blockIdx.x % (DH / COLS) * COLS, b = row / d.H, h = row % d.H;
  const int n = min(max(d.lens[b], 0), d.max_len);
  if (n <= chunk) return;
  const int ns = (n - 1) / chunk + 1, w = threadIdx.x >> 6;  // n + chunk may pass 32 bits
  const float* ml = ws_ml + (long)row * nsplit * 2;
  const int c4 = threadIdx.x % C4, pt = threadIdx.x / C4;
  const float* oo = ws_o + (long)row * nsplit * DH + c0 + 4 * c4;
  constexpr int AHEAD = 8;  // outputs on their way while the factors are worked out
  f32x4 early[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) early[i] = *(const f32x4*)(oo + (long)min(pt + i * PARTS, ns - 1) * DH);
  float M = -INFINITY, L = 0.f;
  for (int s = threadIdx.x; s < ns; s += 256) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  if ((threadIdx.x & 63) == 0) red[w] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ms = M == -INFINITY ? 0.f : M;
  for (int s = threadIdx.x; s < ns; s += 256) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - ms);
    factor[s] = f;
    L += f * ml[2 * s + 1];
  }
  L = wave_sum(L);
  if ((threadIdx.x & 63) == 0) red[4 + w] = L;
  __syncthreads();
  L = (red[4] + red[5]) + (red[6] + red[7]);
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (pt + i * PARTS < ns) o += factor[pt + i * PARTS] * early[i];
#pragma unroll 4
  for (int s = pt + AHEAD * PARTS; s < ns; s += PARTS) o += factor[s] * *(const f32x4*)(oo + (long)s * DH);
  part[pt][c4] = o;
  __syncthreads();
  if (threadIdx.x < COLS) {
    const float* p = (const float*)part + threadIdx.x;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) v += p[i * COLS];
    const int col = c0 + threadIdx.x;
    ((T*)d.o)[(long)b * d.o_row + (long)h * d.o_head + col] = from_f<T>(L == 0.f ? 0.f : v / L);
    if (d.lse && col == 0) d.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.69314718055994531f;
  }
}

static int log2_of(int v) { return __builtin_ctz((unsigned)v); }
static bool is_pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }

static int attn_check(const imgcap_paged_attn_desc* d) {
  IMGCAP_REQUIRE(d != nullptr, "paged attention: desc NULL");
  IMGCAP_REQUIRE(d->dtype == IMGCAP_F32 || d->dtype == IMGCAP_BF16, "paged attention: dtype must be fp32 or bf16");
  IMGCAP_REQUIRE(d->dh == 64 || d->dh == 128, "paged attention: head dim must be 64 or 128");
  IMGCAP_REQUIRE(d->B >= 0 && d->Hkv > 0 && d->H > 0 && d->H % d->Hkv == 0,
                 "paged attention: query heads must be a multiple of the key/value heads");
  IMGCAP_REQUIRE(is_pow2(d->page) && d->page <= 1024, "paged attention: page must be a power of two, at most 1024");
  IMGCAP_REQUIRE(d->pages > 0 && d->width > 0 && d->max_len > 0, "paged attention: empty cache, table or max_len");
  IMGCAP_REQUIRE((int64_t)d->width * d->page <= (1ll << 31) - 65536 && d->max_len <= (int64_t)d->width * d->page,
                 "paged attention: max_len must be within the table's width, and that at most 2^31 - 65536 tokens");
  IMGCAP_REQUIRE(d->q && d->k && d->v && d->o && d->table && d->lens, "paged attention: NULL operand");
  const int64_t vec = d->dtype == IMGCAP_F32 ? 4 : 8;
  const struct { int size; int64_t stride; } dims[] = {{d->B, d->q_row},      {d->H, d->q_head},  {d->pages, d->k_page},
                                                       {d->page, d->k_tok},   {d->Hkv, d->k_head}, {d->pages, d->v_page},
                                                       {d->page, d->v_tok},   {d->Hkv, d->v_head}};
  bool whole = aligned16(d->q) && aligned16(d->k) && aligned16(d->v);
  for (const auto& m : dims) whole = whole && (m.size <= 1 || m.stride % vec == 0);  // no stride where there is one of it
  IMGCAP_REQUIRE(whole, "paged attention: q, k and v must be 16-byte aligned with strides of whole 16 bytes");
  // below this, rows times max_len stay within 63 bits; a launch takes fewer still (attn_fits)
  IMGCAP_REQUIRE((int64_t)d->B * d->Hkv * ((d->H / d->Hkv + 15) / 16) < (1ll << 26), "paged attention: too many rows");
  return 0;
}

// How the length is cut (times of bf16 and pages of 16 tokens unless said, MI355X, calls replayed from a
// graph; pages of one token take 0.1 to 0.7 us more at 64 rows of 49 to 200 tokens, and 395 us against 383 at
// 48 rows of up to 20000, so one rule cuts both).
//  - Up to 64 tokens, two steps, a wave has the row to itself: 512 rows of up to 52 tokens 4.5 us
//    against 4.9 by workgroups of 4 waves; fp32, whose step is longer, up to 32 (40 rows of 49 tokens
//    5.5 by workgroups, 6.5 by waves).
//  - Longer ones go to workgroups of 4 waves (8: 32 requests of up to 2048 tokens with 8 kv heads 44 us,
//    4: 40, a wave each: 51), whole up to 512 tokens, up to 1024 where the rows alone are a
//    workgroup to each CU: the second launch that joins parts costs 4 us (512 rows of up to 600
//    tokens 12.2 whole, 15.9 in chunks of 512).
//  - Else chunks of 512 tokens, shorter (to 128) where that leaves CUs without one, longer where it
//    leaves more than 4096 (48 requests of up to 20011 tokens, 8 kv heads of 128: 402 us with 2048
//    workgroups, 393 with 4096; 432 with 1024).
struct AttnPlan { int gtiles, chunk, nsplit; bool join; };  // nsplit: 1 .. MAX_SPLIT
static AttnPlan attn_plan(const imgcap_paged_attn_desc* d) {
  AttnPlan p;
  p.gtiles = (d->H / d->Hkv + 15) / 16;
  p.join = d->max_len > (d->dtype == IMGCAP_F32 ? 32 : 64);
  const int64_t rows = (int64_t)d->B * d->Hkv * p.gtiles, tokens = rows * d->max_len;
  int64_t chunk = tokens / 256 < 512 ? tokens / 256 : 512;
  if (chunk < tokens / 4096) chunk = tokens / 4096;
  if (chunk < 128) chunk = 128;
  if (chunk < (d->max_len + MAX_SPLIT - 1) / MAX_SPLIT) chunk = (d->max_len + MAX_SPLIT - 1) / MAX_SPLIT;
  if (chunk > d->max_len || d->max_len <= (rows >= 256 ? 1024 : 512)) chunk = d->max_len;
  p.chunk = (int)((chunk + 31) / 32 * 32);
  p.nsplit = (d->max_len - 1) / p.chunk + 1;  // max_len + chunk may pass 32 bits
  return p;
}
// A launch has fewer than 2^32 threads: 256 a row of workgroups, 64 a row that a wave has to itself
// (attn_check).  The join has no more of them: a length is split for fewer than 4096 rows only.
static int attn_fits(const imgcap_paged_attn_desc* d, const AttnPlan& p) {
  IMGCAP_REQUIRE(!p.join || (int64_t)d->B * d->Hkv * p.gtiles < (1ll << 24), "paged attention: too many rows");
  return 0;
}
static int64_t attn_ws(const imgcap_paged_attn_desc* d, const AttnPlan& p) {
  return p.nsplit > 1 ? (int64_t)d->B * d->H * p.nsplit * (d->dh + 2) * 4 : 0;
}

template <typename T, int DH>
static void attn_launch(const imgcap_paged_attn_desc* d, const AttnPlan& p, hipStream_t st) {
  float* ws_o = (float*)d->ws;
  float* ws_ml = ws_o ? ws_o + (int64_t)d->B * d->H * p.nsplit * DH : nullptr;
  const int rows_kv = d->B * d->Hkv * p.gtiles, lp = log2_of(d->page);
  const int waves = rows_kv >= 1024 ? 4 : 1;  // few short rows: a wave to a workgroup, so that they spread over the CUs
#define PA_(TINY, JOIN)                                                                                          \
  hipLaunchKernelGGL((paged_attn_kernel<T, DH, TINY, JOIN>),                                                     \
                     dim3(JOIN ? rows_kv : (rows_kv + waves - 1) / waves, p.nsplit),                             \
                     dim3(64 * (JOIN ? JOIN_WAVES : waves)), 0, st, *d, p.chunk, p.nsplit, p.gtiles, lp, ws_o, ws_ml)
  if (d->page >= 16) {
    if (p.join) PA_(false, true);
    else PA_(false, false);
  } else {
    if (p.join) PA_(true, true);
    else PA_(true, false);
  }
#undef PA_
  if (p.nsplit > 1) {
    const int rows = d->B * d->H;
    if (rows >= 256)
      hipLaunchKernelGGL((paged_join_kernel<T, DH, DH>), dim3(rows), dim3(256), 0, st, *d, p.chunk, p.nsplit, ws_o, ws_ml);
    else
      hipLaunchKernelGGL((paged_join_kernel<T, DH, 32>), dim3(rows * (DH / 32)), dim3(256), 0, st, *d, p.chunk, p.nsplit,
                         ws_o, ws_ml);
  }
}

}  // namespace imgcap

using namespace imgcap;

extern "C" int imgcap_paged_plan(const imgcap_paged_plan_desc* d, void* stream) {
  IMGCAP_REQUIRE(d != nullptr, "imgcap_paged_plan: desc NULL");
  const int B = d->B, width = d->width, tokens = d->tokens;
  IMGCAP_REQUIRE(B > 0 && width > 0 && d->pool > 0 && tokens >= 0,
                 "imgcap_paged_plan: B, width and pool must be positive, tokens not negative");
  IMGCAP_REQUIRE(is_pow2(d->page) && d->page <= 1024, "imgcap_paged_plan: page must be a power of two, at most 1024");
  IMGCAP_REQUIRE((int64_t)width * d->page < (1ll << 31), "imgcap_paged_plan: width * page must be below 2^31");
  IMGCAP_REQUIRE(d->table_row >= width, "imgcap_paged_plan: table rows overlap");
  IMGCAP_REQUIRE(d->past && d->add && d->table && d->free_ids && d->count && d->count_out && d->lens && d->starts &&
                     d->waits && (tokens == 0 || (d->slots && d->rows && d->positions)),
                 "imgcap_paged_plan: NULL operand");
  PlanArgs a;
  (imgcap_paged_plan_desc&)a = *d;
  a.lp = log2_of(d->page);
  const bool fast = B <= PLAN_ROWS && tokens <= PLAN_CAP && width <= PLAN_CAP;
  const bool one = fast && tokens <= PLAN_TOKENS;
  IMGCAP_REQUIRE(one || d->ws, "imgcap_paged_plan: NULL workspace");
  hipStream_t st = (hipStream_t)stream;
  if (fast) {
    const int most = one && tokens > B ? (tokens < PLAN_ROWS ? tokens : PLAN_ROWS) : B;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3((most + 63) / 64 * 64), 0, st, a, one ? 1 : 0);
  } else {
    hipLaunchKernelGGL(paged_plan_long_kernel, dim3(1), dim3(1024), 0, st, a);
  }
  if (!one && tokens > 0)
    hipLaunchKernelGGL(paged_slots_kernel, dim3((unsigned)(((int64_t)tokens + SLOT_TOKENS - 1) / SLOT_TOKENS)), dim3(256),
                       0, st, a, aligned16(d->slots) && aligned16(d->rows) && aligned16(d->positions) ? 1 : 0);
  IMGCAP_CHECK_LAUNCH("imgcap_paged_plan");
  return 0;
}

extern "C" int imgcap_paged_write(const imgcap_paged_write_desc* d, void* stream) {
  IMGCAP_REQUIRE(d != nullptr, "imgcap_paged_write: desc NULL");
  IMGCAP_REQUIRE(d->dtype == IMGCAP_F32 || d->dtype == IMGCAP_BF16, "imgcap_paged_write: dtype must be fp32 or bf16");
  const int esz = d->dtype == IMGCAP_F32 ? 4 : 2, vec = 16 / esz;
  IMGCAP_REQUIRE(d->n >= 0 && d->heads > 0 && d->dh > 0 && d->dh % vec == 0,
                 "imgcap_paged_write: head dim must be whole 16-byte pieces");
  IMGCAP_REQUIRE(is_pow2(d->page) && d->page <= 1024 && d->pages > 0,
                 "imgcap_paged_write: page must be a power of two, at most 1024");
  if (d->n == 0) return 0;
  IMGCAP_REQUIRE(d->k && d->v && d->kc && d->vc && d->slots, "imgcap_paged_write: NULL operand");
  const struct { int size; int64_t stride; } dims[] = {
      {d->n, d->k_row},      {d->heads, d->k_head},  {d->n, d->v_row},      {d->heads, d->v_head},  {d->pages, d->kc_page},
      {d->page, d->kc_tok},  {d->heads, d->kc_head}, {d->pages, d->vc_page}, {d->page, d->vc_tok},  {d->heads, d->vc_head}};
  for (const auto& m : dims)
    IMGCAP_REQUIRE(m.size <= 1 || m.stride % vec == 0, "imgcap_paged_write: strides must be whole 16-byte pieces");
  IMGCAP_REQUIRE(aligned16(d->k) && aligned16(d->v) && aligned16(d->kc) && aligned16(d->vc),
                 "imgcap_paged_write: operands must be 16-byte aligned");
  const int vecs = d->dh / vec;
  const int64_t units = (int64_t)d->n * d->heads * vecs;
  IMGCAP_REQUIRE(units < (1ll << 31), "imgcap_paged_write: at most 2^31 16-byte pieces a call");
  hipLaunchKernelGGL(paged_write_kernel, dim3((unsigned)((units + 255) / 256), 2), dim3(256), 0, (hipStream_t)stream,
                     *d, vecs, log2_of(d->page), esz);
  IMGCAP_CHECK_LAUNCH("imgcap_paged_write");
  return 0;
}

extern "C" int imgcap_paged_attention_ws(const imgcap_paged_attn_desc* d, int64_t* bytes) {
  if (int rc = attn_check(d)) return rc;
  IMGCAP_REQUIRE(bytes != nullptr, "imgcap_paged_attention_ws: bytes NULL");
  const AttnPlan p = attn_plan(d);
  if (int rc = attn_fits(d, p)) return rc;
  *bytes = attn_ws(d, p);
  return 0;
}

extern "C" int imgcap_paged_attention(const imgcap_paged_attn_desc* d, void* stream) {
  if (int rc = attn_check(d)) return rc;
  if (d->B == 0) return 0;
  const AttnPlan p = attn_plan(d);
  if (int rc = attn_fits(d, p)) return rc;
  const int64_t need = attn_ws(d, p);
  if (need > 0 && !(d->ws && aligned16(d->ws) && d->ws_bytes >= need))
    return fail(IMGCAP_EWORKSPACE, "imgcap_paged_attention: " + std::to_string(need) +
                                       " bytes of 16-byte aligned workspace needed (imgcap_paged_attention_ws)");
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == IMGCAP_BF16) {
    if (d->dh == 64) attn_launch<bf16, 64>(d, p, st);
    else attn_launch<bf16, 128>(d, p, st);
  } else {
    if (d->dh == 64) attn_launch<float, 64>(d, p, st);
    else attn_launch<float, 128>(d, p, st);
  }
  IMGCAP_CHECK_LAUNCH("imgcap_paged_attention");
  return 0;
}
