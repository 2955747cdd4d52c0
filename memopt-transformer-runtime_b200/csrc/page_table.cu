// page_table.cu — page tables and slot maps built on the GPU from request
// lengths.
//
// The device counterpart of the host page tables (memopt.PageTable over the
// FIFO free-list, reference src/csrc/kv_cache.cu:146-201): the free pages form
// a ring in device memory, sequences own rows of one block table, and a call
// takes a batch of rows with their numbers of new (or kept) tokens.
//
//   reserve:  o_b = lens[row_b], n_b new tokens; cu = exclusive scan of n;
//             need_b = ceil((o_b + n_b) / BS) - ceil(o_b / BS), g = its
//             exclusive scan; page i of row b is its table entry for
//             i < ceil(o_b / BS), else ring[(head + g_b + i - ceil(o_b/BS)) mod NB];
//             token cu_b + r has index p = o_b + r in its row, slot
//             page(p / BS) * BS + p mod BS and position p + offset_b, the
//             offset being what an eviction took out of the row before it.
//   truncate: the pages past ceil(k_b / BS) go to the ring's tail in row and
//             page order.
//   replace:  truncate to nothing, then reserve, both or neither: the first
//             launch checks the second one's batch too and does nothing if that
//             will not fit, and the second refuses rows that were not cut.
//
// One launch each (two for replace): every CTA reads the old lengths and the old ring state and
// repeats the scan over the batch in shared memory (no CTA waits for another),
// then expands its share of the tokens and of the table rows.  The CTA that
// arrives last at a ticket in the pool state commits the new lengths, head and
// count, so nothing reads a value that the same call wrote.  Whole numbers only;
// bound by latency: the launch, the dependent loads row -> length -> page, the
// fence and the ticket.  Hence a warp per table row with its entries in flight at
// once, and CTAs of 256 threads, or of 1024 where the batch is larger than 256
// rows (the scan is then still one round of loads).
#include <algorithm>

#include "common.cuh"

namespace memopt {
namespace {

constexpr int kTokensPerThread = 4;
constexpr int kInFlight = 8;  // table entries that a lane loads before it stores them
constexpr int kMaxBatch = 8192;
constexpr int kMaxRows = 1 << 18;

struct PageArgs {
  int32_t* tables;      // [R, MB]
  int32_t* lens;        // [R]
  int32_t* ring;        // [NB]
  int32_t* state;       // head, count, status, ticket
  const int32_t* rows;  // [B]
  const int32_t* amount;  // [B]: new tokens (reserve) or kept tokens (truncate; null: none kept)
  int R, MB, NB, BS, B;
  int shift;  // log2(BS), or -1 where BS is no power of two
  int64_t max_tokens;
  const int32_t* next;  // [B]: truncate's rows begin anew with so many tokens (null: they do not)
  bool fresh;           // reserve: the rows have to be empty
  int32_t* offsets;    // [R]: a token's position less its index in the row (null: 0)
  int32_t* cu;         // [B + 1]
  int32_t* slots;      // [max_tokens]
  int32_t* positions;  // [max_tokens]
  int32_t* out_tables;  // [B, MB]
  int32_t* out_lens;    // [B]
  int32_t* attend_lens;  // [B]: out_lens, 0 where the call is refused (may be null)
};

constexpr uint32_t kNotCut = 1u << 30;  // internal refusal: the call's first launch has set the status

// What a CTA holds of the batch in shared memory.
struct Batch {
  int32_t* row;   // [B]; 0 where the entry is invalid (the call is refused then)
  int32_t* old;   // [B] length before the call
  int32_t* cu;    // [B + 1] exclusive scan of the new tokens (truncate: unused)
  int32_t* page;  // [B + 1] exclusive scan of the pages taken (truncate: given back)
  int32_t* off;   // [B] position offset (truncate: unused); an empty row begins at 0 again
  uint32_t* seen;  // bit per table row
};

__device__ __forceinline__ Batch carve(uint8_t* smem, int B) {
  Batch t;
  t.row = reinterpret_cast<int32_t*>(smem);
  t.old = t.row + B;
  t.cu = t.old + B;
  t.page = t.cu + B + 1;
  t.off = t.page + B + 1;
  t.seen = reinterpret_cast<uint32_t*>(t.off + B);
  return t;
}

constexpr size_t batch_smem(int B, int R) {
  return (static_cast<size_t>(5) * B + 2) * 4 + static_cast<size_t>((R + 31) / 32) * 4;
}

// x >= 0; unsigned, as a length and a block size may add up to more than 2^31.
__device__ __forceinline__ int over_bs(uint32_t x, const PageArgs& a) {
  return static_cast<int>(a.shift >= 0 ? x >> a.shift : x / static_cast<uint32_t>(a.BS));
}
__device__ __forceinline__ int pages_of(int tokens, const PageArgs& a) {
  return over_bs(static_cast<uint32_t>(tokens) + a.BS - 1, a);
}

// Reads the batch, checks it and scans it.  Returns the status bits of the
// refusal (0: accepted), the same in every thread.  total_tokens and
// total_pages are the sums (64-bit: refused sums may exceed an int).
template <int kThreads, bool kReserve, bool kRows>
__device__ uint32_t scan_batch(const PageArgs& a, const Batch& t, int64_t& total_tokens, int64_t& total_pages) {
  __shared__ uint32_t s_status;
  constexpr int kWarps = kThreads / 32;
  __shared__ int64_t s_sum[2][kWarps], s_all[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_status = 0;
  for (int i = tid; i < (a.R + 31) / 32; i += kThreads) t.seen[i] = 0;
  __syncthreads();
  uint32_t bits = 0;
  const int64_t cap = static_cast<int64_t>(a.MB) * a.BS;
  int64_t carry_n = 0, carry_p = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0, p = 0;
    if (b < a.B) {
      int row = a.rows[b], old = 0, off = 0;
      if (row < 0 || row >= a.R) {
        bits |= MEMOPT_PAGES_BAD_ROW;
        row = 0;
      } else {
        if (atomicOr(&t.seen[row >> 5], 1u << (row & 31)) & (1u << (row & 31))) bits |= MEMOPT_PAGES_BAD_ROW;
        old = a.lens[row];
        if (kReserve && kRows) off = a.offsets[row];
        if (old < 0 || old > cap) {
          bits |= MEMOPT_PAGES_CORRUPT;
          old = 0;
        }
      }
      n = a.amount ? a.amount[b] : 0;
      if (n < 0 || (!kReserve && n > old)) {
        bits |= MEMOPT_PAGES_BAD_LENGTH;
        n = 0;
      }
      if (kReserve && kRows && a.fresh && old > 0) {
        bits |= kNotCut;
        n = 0;
      }
      if (kReserve) {
        if (static_cast<int64_t>(old) + n > cap) {
          bits |= MEMOPT_PAGES_ROW_FULL;
          n = 0;
        }
        p = pages_of(old + n, a) - pages_of(old, a);
      } else {
        p = pages_of(old, a) - pages_of(n, a);
      }
      t.row[b] = row;
      t.old[b] = old;
      if (kReserve && kRows) t.off[b] = old > 0 ? off : 0;
    }
    // Block-wide exclusive scan of (n, p): within the warp, then over the warps.
    int64_t sn = n, sp = p;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t un = __shfl_up_sync(0xffffffffu, sn, d), up = __shfl_up_sync(0xffffffffu, sp, d);
      if (lane >= d) {
        sn += un;
        sp += up;
      }
    }
    if (lane == 31) {
      s_sum[0][warp] = sn;
      s_sum[1][warp] = sp;
    }
    __syncthreads();
    if (warp < 2) {  // warp 0 scans the warps' tokens, warp 1 their pages
      const int64_t own = lane < kWarps ? s_sum[warp][lane] : 0;
      int64_t sum = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (lane < kWarps) s_sum[warp][lane] = sum - own;
      if (lane == 31) s_all[warp] = sum;
    }
    __syncthreads();
    const int64_t bn = carry_n + s_sum[0][warp], bp = carry_p + s_sum[1][warp];
    carry_n += s_all[0];
    carry_p += s_all[1];
    if (b < a.B) {  // sums past an int belong to refused calls (checked below)
      t.cu[b] = static_cast<int32_t>(bn + sn - n);
      t.page[b] = static_cast<int32_t>(bp + sp - p);
    }
    __syncthreads();
  }
  if (tid == 0) {
    t.cu[a.B] = static_cast<int32_t>(carry_n);
    t.page[a.B] = static_cast<int32_t>(carry_p);
  }
  total_tokens = carry_n;
  total_pages = carry_p;
  if (kReserve && carry_n > a.max_tokens) bits |= MEMOPT_PAGES_BAD_LENGTH;
  if (bits) atomicOr(&s_status, bits);
  __syncthreads();
  return s_status;
}

// True in every thread of the CTA that arrives last; its writes and those of
// all other CTAs before their arrival are then visible to it.
__device__ bool arrive_last(int32_t* ticket) {
  __shared__ int s_last;
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (s_last) __threadfence();
  return s_last != 0;
}

// kRows: with position offsets, lengths to attend over and perhaps rows that begin
// anew (reserve_rows).  In kernels of their own, as is truncate with a next batch
// (kNext): code that a short kernel fetches and does not use costs it 0.2 to 0.5 us.
template <int kThreads, bool kRows>
__global__ void __launch_bounds__(kThreads) reserve_kernel(const PageArgs a) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ uint8_t smem[];
  const Batch t = carve(smem, a.B);
  const int tid = threadIdx.x, lane = tid & 31;
  begin_next();
  after_previous();
  const int head = a.state[0], count = a.state[1];
  int64_t tokens, pages;
  uint32_t status = scan_batch<kThreads, true, kRows>(a, t, tokens, pages);
  if (head < 0 || head >= a.NB || count < 0 || count > a.NB) status |= MEMOPT_PAGES_CORRUPT;
  if (status == 0 && pages > count) status |= MEMOPT_PAGES_EXHAUSTED;
  const bool taken = status == 0;
  uint32_t bits = 0;
  auto ring_at = [&](int i) {
    uint32_t at = static_cast<uint32_t>(head) + i;  // head < NB and i < count <= NB < 2^31
    if (at >= static_cast<uint32_t>(a.NB)) at -= a.NB;
    return a.ring[at];
  };

  // Tokens: four consecutive ones per thread, the sequence of the first by
  // binary search in the scanned lengths, then walked forward.
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads * kTokensPerThread;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kThreads + tid) * kTokensPerThread; t0 < a.max_tokens;
       t0 += step) {
    int32_t slot[kTokensPerThread], pos[kTokensPerThread];
#pragma unroll
    for (int k = 0; k < kTokensPerThread; ++k) {
      slot[k] = -1;
      pos[k] = 0;
    }
    if (taken && t0 < tokens) {
      int lo = 0, hi = a.B;  // the last b with cu[b] <= t0
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.cu[mid] <= t0) lo = mid;
        else hi = mid;
      }
      int b = lo, page_at = -1, page = -1;
#pragma unroll
      for (int k = 0; k < kTokensPerThread; ++k) {
        const int64_t tk = t0 + k;
        if (tk >= tokens) break;
        while (t.cu[b + 1] <= tk) {  // tk < cu[B]: ends at the sequence of tk
          ++b;
          page_at = -1;
        }
        const int p = t.old[b] + static_cast<int>(tk - t.cu[b]);
        const int at = over_bs(p, a);
        if (at != page_at) {
          const int had = pages_of(t.old[b], a);
          page = at < had ? a.tables[static_cast<int64_t>(t.row[b]) * a.MB + at] : ring_at(t.page[b] + at - had);
          page_at = at;
        }
        pos[k] = kRows ? p + t.off[b] : p;
        if (page >= 0 && page < a.NB) slot[k] = page * a.BS + (p - at * a.BS);
        else bits |= MEMOPT_PAGES_CORRUPT;
      }
    }
    if (t0 + kTokensPerThread <= a.max_tokens) {  // t0 is a multiple of 4 and the outputs are 16-byte aligned
      *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
      for (int k = 0; k < kTokensPerThread; ++k) {
        if (t0 + k < a.max_tokens) {
          a.slots[t0 + k] = slot[k];
          a.positions[t0 + k] = pos[k];
        }
      }
    }
  }

  // Table rows: a warp per batch row writes the new pages into the row, and all
  // its pages into the batch's own table (-1 behind them).
  const int nwarps = gridDim.x * kWarps;
  const bool bad = status & MEMOPT_PAGES_BAD_ROW;
  for (int b = blockIdx.x * kWarps + (tid >> 5); b < a.B; b += nwarps) {
    const int had = bad ? 0 : pages_of(t.old[b], a), more = taken ? t.page[b + 1] - t.page[b] : 0;
    int32_t* row = a.tables + static_cast<int64_t>(t.row[b]) * a.MB;
    int32_t* out = a.out_tables + static_cast<int64_t>(b) * a.MB;
    for (int c0 = lane; c0 < a.MB; c0 += 32 * kInFlight) {
      int32_t v[kInFlight];
#pragma unroll
      for (int i = 0; i < kInFlight; ++i) {
        const int c = c0 + 32 * i;
        v[i] = c < had ? row[c] : c < had + more ? ring_at(t.page[b] + c - had) : -1;
      }
#pragma unroll
      for (int i = 0; i < kInFlight; ++i) {
        const int c = c0 + 32 * i;
        if (c >= a.MB) break;
        if (c >= had && c < had + more) {
          if (v[i] < 0 || v[i] >= a.NB) bits |= MEMOPT_PAGES_CORRUPT;
          row[c] = v[i];
        }
        out[c] = v[i];
      }
    }
    if (lane == 0) {
      const int len = bad ? 0 : t.old[b] + (taken ? t.cu[b + 1] - t.cu[b] : 0);
      a.out_lens[b] = len;
      if (kRows) a.attend_lens[b] = taken ? len : 0;
    }
  }
  for (int i = blockIdx.x * kThreads + tid; i <= a.B; i += gridDim.x * kThreads) a.cu[i] = taken ? t.cu[i] : 0;
  if (bits) atomicOr(a.state + 2, static_cast<int>(bits));

  if (arrive_last(a.state + 3)) {
    if (taken) {
      for (int b = tid; b < a.B; b += kThreads) {
        a.lens[t.row[b]] = t.old[b] + (t.cu[b + 1] - t.cu[b]);
        if (kRows && t.old[b] == 0) a.offsets[t.row[b]] = 0;
      }
    }
    if (tid == 0) {
      if (taken) {
        a.state[0] = static_cast<int32_t>((head + pages) % a.NB);
        a.state[1] = static_cast<int32_t>(count - pages);
      }
      if (kRows) status &= ~kNotCut;
      if (status) atomicOr(a.state + 2, static_cast<int>(status));
      a.state[3] = 0;
    }
  }
}

// Whether the batch of a.next fits once the rows are empty and `free_pages` pages
// are free: the status bits that reserve would give it.
template <int kThreads>
__device__ uint32_t next_batch_fits(const PageArgs& a, int64_t free_pages) {
  __shared__ unsigned long long s_sum[2];
  __shared__ uint32_t s_bits;
  if (threadIdx.x == 0) s_sum[0] = s_sum[1] = s_bits = 0;
  __syncthreads();
  const int64_t cap = static_cast<int64_t>(a.MB) * a.BS;
  uint32_t bits = 0;
  int64_t tokens = 0, pages = 0;
  for (int b = threadIdx.x; b < a.B; b += kThreads) {
    const int n = a.next[b];
    if (n < 0) bits |= MEMOPT_PAGES_BAD_LENGTH;
    else if (n > cap) bits |= MEMOPT_PAGES_ROW_FULL;
    else tokens += n, pages += pages_of(n, a);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    tokens += __shfl_xor_sync(0xffffffffu, tokens, d);
    pages += __shfl_xor_sync(0xffffffffu, pages, d);
  }
  if ((threadIdx.x & 31) == 0) {
    atomicAdd(&s_sum[0], static_cast<unsigned long long>(tokens));
    atomicAdd(&s_sum[1], static_cast<unsigned long long>(pages));
  }
  if (bits) atomicOr(&s_bits, bits);
  __syncthreads();
  bits = s_bits;
  if (static_cast<int64_t>(s_sum[0]) > a.max_tokens) bits |= MEMOPT_PAGES_BAD_LENGTH;
  if (bits == 0 && static_cast<int64_t>(s_sum[1]) > free_pages) bits |= MEMOPT_PAGES_EXHAUSTED;
  return bits;
}

template <int kThreads, bool kNext>
__global__ void __launch_bounds__(kThreads) truncate_kernel(const PageArgs a) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ uint8_t smem[];
  const Batch t = carve(smem, a.B);
  const int tid = threadIdx.x, lane = tid & 31;
  begin_next();
  after_previous();
  const int head = a.state[0], count = a.state[1];
  int64_t kept, pages;
  uint32_t status = scan_batch<kThreads, false, false>(a, t, kept, pages);
  if (head < 0 || head >= a.NB || count < 0 || count > a.NB || (status == 0 && count + pages > a.NB))
    status |= MEMOPT_PAGES_CORRUPT;
  if (kNext) status |= next_batch_fits<kThreads>(a, count + pages);
  uint32_t bits = 0;
  if (status == 0) {
    const int nwarps = gridDim.x * kWarps;
    for (int b = blockIdx.x * kWarps + (tid >> 5); b < a.B; b += nwarps) {
      const int gone = t.page[b + 1] - t.page[b];
      const int first = pages_of(t.old[b], a) - gone;
      int32_t* row = a.tables + static_cast<int64_t>(t.row[b]) * a.MB + first;
      const uint32_t NB = a.NB;  // below 2^31
      uint32_t tail = static_cast<uint32_t>(head) + count;
      tail = tail >= NB ? tail - NB : tail;
      tail += t.page[b];
      tail = tail >= NB ? tail - NB : tail;
      for (int i0 = lane; i0 < gone; i0 += 32 * kInFlight) {
        int32_t v[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) v[i] = i0 + 32 * i < gone ? row[i0 + 32 * i] : 0;
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
          const int k = i0 + 32 * i;
          if (k >= gone) break;
          if (v[i] < 0 || v[i] >= a.NB) bits |= MEMOPT_PAGES_CORRUPT;
          const uint32_t at = tail + k;  // k < NB
          a.ring[at >= NB ? at - NB : at] = v[i];
          row[k] = -1;
        }
      }
    }
  }
  if (bits) atomicOr(a.state + 2, static_cast<int>(bits));
  if (arrive_last(a.state + 3)) {
    if (status == 0) {
      for (int b = tid; b < a.B; b += kThreads) a.lens[t.row[b]] = a.amount ? a.amount[b] : 0;
    }
    if (tid == 0) {
      if (status == 0) a.state[1] = static_cast<int32_t>(count + pages);
      else atomicOr(a.state + 2, static_cast<int>(status));
      a.state[3] = 0;
    }
  }
}

int check_pages(const char* who, const PageArgs& a) {
  const std::string w(who);
  if (a.B < 0 || a.R <= 0 || a.MB <= 0 || a.NB <= 0 || a.BS <= 0 || a.max_tokens < 0)
    return fail(MEMOPT_ERR_INVALID_ARG, w + ": invalid geometry");
  if (a.B > kMaxBatch) return fail(MEMOPT_ERR_UNSUPPORTED, w + ": more than 8192 rows in a call");
  if (a.R > kMaxRows) return fail(MEMOPT_ERR_UNSUPPORTED, w + ": more than 262144 table rows");
  if (static_cast<int64_t>(a.NB) * a.BS > 0x7fffffffLL || static_cast<int64_t>(a.MB) * a.BS > 0x7fffffffLL)
    return fail(MEMOPT_ERR_UNSUPPORTED, w + ": slots past 2^31 (the slot mapping is int32)");
  if (a.MB > 0x7fffffff - 1024)  // a lane's index of an entry runs up to 32 * kInFlight past the row
    return fail(MEMOPT_ERR_UNSUPPORTED, w + ": a block table row near 2^31 entries");
  if (a.max_tokens > 0x7fffffffLL) return fail(MEMOPT_ERR_UNSUPPORTED, w + ": max_tokens past 2^31");
  if (!a.tables || !a.lens || !a.ring || !a.state || (a.B > 0 && !a.rows))
    return fail(MEMOPT_ERR_INVALID_ARG, w + ": null pointer");
  return MEMOPT_OK;
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v && s < 30) ++s;
  return (1 << s) == v ? s : -1;
}

// One pass over the tokens and one over the rows, at most one CTA per SM: each
// repeats the scan of the batch.
template <typename K>
int launch_pages(K small, K large, const char* what, const PageArgs& a, cudaStream_t s) {
  const int threads = a.B > 256 ? 1024 : 256;
  const K kern = a.B > 256 ? large : small;
  const size_t smem = batch_smem(a.B, a.R);
  if (smem > 48 * 1024) {
    // The most that any call needs, so that a call on another host thread does not
    // lower this one's limit before its launch.
    constexpr size_t kMost = batch_smem(kMaxBatch, kMaxRows);
    static_assert(kMost <= 227 * 1024, "shared memory");
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMost));
    if (e != cudaSuccess) return cuda_fail(e, what);
  }
  const int64_t per_cta = threads * kTokensPerThread, rows = threads / 32;
  const int64_t tokens = a.next ? 0 : a.max_tokens;  // truncate expands none
  const int64_t want = std::max((tokens + per_cta - 1) / per_cta, (a.B + rows - 1) / rows);
  const int grid = static_cast<int>(std::min<int64_t>(sm_count(), std::max<int64_t>(1, want)));
  MEMOPT_LAUNCH(launch_after(kern, grid, threads, smem, s, a), what);
  return MEMOPT_OK;
}

int reserve(const char* who, PageArgs a, cudaStream_t s) {
  const int st = check_pages(who, a);
  if (st != MEMOPT_OK) return st;
  if (!a.cu || (a.B > 0 && (!a.amount || !a.out_tables || !a.out_lens)) ||
      (a.max_tokens > 0 && (!a.slots || !a.positions)))
    return fail(MEMOPT_ERR_INVALID_ARG, std::string(who) + ": null pointer");
  if ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.positions)) & 15u)
    return fail(MEMOPT_ERR_INVALID_ARG, std::string(who) + ": slot_mapping and positions must be 16-byte aligned");
  a.shift = log2_of(a.BS);
  if (a.fresh && a.B > 0) {
    PageArgs cut = a;
    cut.amount = nullptr, cut.next = a.amount;
    const int st2 = launch_pages(truncate_kernel<256, true>, truncate_kernel<1024, true>, "truncate_kernel launch", cut, s);
    if (st2 != MEMOPT_OK) return st2;
  }
  return a.offsets ? launch_pages(reserve_kernel<256, true>, reserve_kernel<1024, true>, "reserve_kernel launch", a, s)
                   : launch_pages(reserve_kernel<256, false>, reserve_kernel<1024, false>, "reserve_kernel launch", a, s);
}

}  // namespace
}  // namespace memopt

using namespace memopt;

extern "C" int memopt_reserve_slots(int32_t* block_tables, int32_t* context_lens, int num_rows, int max_blocks_per_seq,
                                    int32_t* free_pages, int num_blocks, int32_t* pool_state, const int32_t* rows,
                                    const int32_t* new_lens, int batch, int block_size, int64_t max_tokens,
                                    int32_t* cu_seqlens, int32_t* slot_mapping, int32_t* positions,
                                    int32_t* batch_tables, int32_t* batch_lens, void* stream) {
  PageArgs a{block_tables, context_lens, free_pages, pool_state, rows, new_lens, num_rows, max_blocks_per_seq,
             num_blocks, block_size, batch, 0, max_tokens, nullptr, false, nullptr, cu_seqlens, slot_mapping, positions, batch_tables,
             batch_lens, nullptr};
  return reserve("reserve_slots", a, as_stream(stream));
}

extern "C" int memopt_reserve_rows(int32_t* block_tables, int32_t* context_lens, int32_t* position_offsets,
                                   int num_rows, int max_blocks_per_seq, int32_t* free_pages, int num_blocks,
                                   int32_t* pool_state, const int32_t* rows, const int32_t* new_lens, int batch,
                                   int block_size, int64_t max_tokens, int replace, int32_t* cu_seqlens,
                                   int32_t* slot_mapping, int32_t* positions, int32_t* batch_tables,
                                   int32_t* batch_lens, int32_t* attend_lens, void* stream) {
  PageArgs a{block_tables, context_lens, free_pages, pool_state, rows, new_lens, num_rows, max_blocks_per_seq,
             num_blocks, block_size, batch, 0, max_tokens, nullptr, replace != 0, position_offsets, cu_seqlens,
             slot_mapping, positions, batch_tables, batch_lens, attend_lens};
  if (!position_offsets || (batch > 0 && !attend_lens)) return fail(MEMOPT_ERR_INVALID_ARG, "reserve_rows: null pointer");
  return reserve("reserve_rows", a, as_stream(stream));
}

extern "C" int memopt_truncate_rows(int32_t* block_tables, int32_t* context_lens, int num_rows, int max_blocks_per_seq,
                                    int32_t* free_pages, int num_blocks, int32_t* pool_state, const int32_t* rows,
                                    const int32_t* keep_lens, int batch, int block_size, void* stream) {
  PageArgs a{block_tables, context_lens, free_pages, pool_state, rows, keep_lens, num_rows, max_blocks_per_seq,
             num_blocks, block_size, batch, 0, 0, nullptr, false, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  const int st = check_pages("truncate_rows", a);
  if (st != MEMOPT_OK) return st;
  if (batch == 0) return MEMOPT_OK;
  a.shift = log2_of(block_size);
  return launch_pages(truncate_kernel<256, false>, truncate_kernel<1024, false>, "truncate_kernel launch", a, as_stream(stream));
}
