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
//             token cu_b + r has position p = o_b + r and slot
//             page(p / BS) * BS + p mod BS.
//   truncate: the pages past ceil(k_b / BS) go to the ring's tail in row and
//             page order.
//
// One launch each: every CTA reads the old lengths and the old ring state and
// repeats the scan over the batch in shared memory (a few loads per thread;
// no CTA waits for another), then expands its share of the tokens and of the
// table rows.  The CTA that arrives last at a ticket in the pool state commits
// the new lengths, head and count, so nothing reads a value that the same call
// wrote.  Whole numbers only; bound by the launch and the two dependent loads
// (row, length) except for very large batches, where the 8 bytes written per
// token count.
#include <algorithm>

#include "common.cuh"

namespace memopt {
namespace {

constexpr int kThreads = 256;
constexpr int kTokensPerThread = 4;
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
  int64_t max_tokens;
  int32_t* cu;         // [B + 1]
  int32_t* slots;      // [max_tokens]
  int32_t* positions;  // [max_tokens]
  int32_t* out_tables;  // [B, MB]
  int32_t* out_lens;    // [B]
};

// What a CTA holds of the batch in shared memory.
struct Batch {
  int32_t* row;   // [B]; 0 where the entry is invalid (the call is refused then)
  int32_t* old;   // [B] length before the call
  int32_t* cu;    // [B + 1] exclusive scan of the new tokens (truncate: unused)
  int32_t* page;  // [B + 1] exclusive scan of the pages taken (truncate: given back)
  uint32_t* seen;  // bit per table row
};

__device__ __forceinline__ Batch carve(uint8_t* smem, int B) {
  Batch t;
  t.row = reinterpret_cast<int32_t*>(smem);
  t.old = t.row + B;
  t.cu = t.old + B;
  t.page = t.cu + B + 1;
  t.seen = reinterpret_cast<uint32_t*>(t.page + B + 1);
  return t;
}

size_t batch_smem(int B, int R) {
  return (static_cast<size_t>(4) * B + 2) * 4 + static_cast<size_t>((R + 31) / 32) * 4;
}

__device__ __forceinline__ int pages_of(int tokens, int BS) { return (tokens + BS - 1) / BS; }

// Reads the batch, checks it and scans it.  Returns the status bits of the
// refusal (0: accepted), the same in every thread.  total_tokens and
// total_pages are the sums (64-bit: refused sums may exceed an int).
template <bool kReserve>
__device__ uint32_t scan_batch(const PageArgs& a, const Batch& t, int64_t& total_tokens, int64_t& total_pages) {
  __shared__ uint32_t s_status;
  __shared__ int64_t s_sum[2][kThreads / 32];
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
      int row = __ldg(a.rows + b), old = 0;
      if (row < 0 || row >= a.R) {
        bits |= MEMOPT_PAGES_BAD_ROW;
        row = 0;
      } else {
        if (atomicOr(&t.seen[row >> 5], 1u << (row & 31)) & (1u << (row & 31))) bits |= MEMOPT_PAGES_BAD_ROW;
        old = a.lens[row];
        if (old < 0 || old > cap) {
          bits |= MEMOPT_PAGES_CORRUPT;
          old = 0;
        }
      }
      n = a.amount ? __ldg(a.amount + b) : 0;
      if (n < 0 || (!kReserve && n > old)) {
        bits |= MEMOPT_PAGES_BAD_LENGTH;
        n = 0;
      }
      if (kReserve) {
        if (static_cast<int64_t>(old) + n > cap) {
          bits |= MEMOPT_PAGES_ROW_FULL;
          n = 0;
        }
        p = pages_of(old + n, a.BS) - pages_of(old, a.BS);
      } else {
        p = pages_of(old, a.BS) - pages_of(n, a.BS);
      }
      t.row[b] = row;
      t.old[b] = old;
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
    int64_t bn = carry_n, bp = carry_p;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) {
        bn += s_sum[0][w];
        bp += s_sum[1][w];
      }
      carry_n += s_sum[0][w];
      carry_p += s_sum[1][w];
    }
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
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (s_last) __threadfence();
  return s_last != 0;
}

__global__ void __launch_bounds__(kThreads) reserve_kernel(const PageArgs a) {
  extern __shared__ uint8_t smem[];
  const Batch t = carve(smem, a.B);
  const int tid = threadIdx.x, lane = tid & 31;
  const int head = a.state[0], count = a.state[1];
  int64_t tokens, pages;
  uint32_t status = scan_batch<true>(a, t, tokens, pages);
  if (head < 0 || head >= a.NB || count < 0 || count > a.NB) status |= MEMOPT_PAGES_CORRUPT;
  if (status == 0 && pages > count) status |= MEMOPT_PAGES_EXHAUSTED;
  const bool taken = status == 0;
  uint32_t bits = 0;
  auto ring_at = [&](int64_t i) {
    int64_t at = head + i;  // head < NB and i < count <= NB
    if (at >= a.NB) at -= a.NB;
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
        const int at = p / a.BS;
        if (at != page_at) {
          const int had = pages_of(t.old[b], a.BS);
          page = at < had ? a.tables[static_cast<int64_t>(t.row[b]) * a.MB + at] : ring_at(t.page[b] + at - had);
          page_at = at;
        }
        pos[k] = p;
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

  // Table rows: a warp per batch row writes the new pages into the row and
  // the whole row into the batch's own table.
  const int nwarps = gridDim.x * (kThreads / 32);
  for (int b = blockIdx.x * (kThreads / 32) + (tid >> 5); b < a.B; b += nwarps) {
    const int had = pages_of(t.old[b], a.BS), more = taken ? t.page[b + 1] - t.page[b] : 0;
    int32_t* row = a.tables + static_cast<int64_t>(t.row[b]) * a.MB;
    int32_t* out = a.out_tables + static_cast<int64_t>(b) * a.MB;
    const bool bad = status & MEMOPT_PAGES_BAD_ROW;
    for (int c = lane; c < a.MB; c += 32) {
      int32_t v = -1;
      if (!bad) {
        if (c >= had && c < had + more) {
          v = ring_at(t.page[b] + c - had);
          if (v < 0 || v >= a.NB) bits |= MEMOPT_PAGES_CORRUPT;
          row[c] = v;
        } else {
          v = row[c];
        }
      }
      out[c] = v;
    }
    if (lane == 0) a.out_lens[b] = bad ? 0 : t.old[b] + (taken ? t.cu[b + 1] - t.cu[b] : 0);
  }
  for (int i = blockIdx.x * kThreads + tid; i <= a.B; i += gridDim.x * kThreads) a.cu[i] = taken ? t.cu[i] : 0;
  if (bits) atomicOr(a.state + 2, static_cast<int>(bits));

  if (arrive_last(a.state + 3)) {
    if (taken) {
      for (int b = tid; b < a.B; b += kThreads) a.lens[t.row[b]] = t.old[b] + (t.cu[b + 1] - t.cu[b]);
    }
    if (tid == 0) {
      if (taken) {
        a.state[0] = static_cast<int32_t>((head + pages) % a.NB);
        a.state[1] = static_cast<int32_t>(count - pages);
      }
      if (status) atomicOr(a.state + 2, static_cast<int>(status));
      a.state[3] = 0;
    }
  }
}

__global__ void __launch_bounds__(kThreads) truncate_kernel(const PageArgs a) {
  extern __shared__ uint8_t smem[];
  const Batch t = carve(smem, a.B);
  const int tid = threadIdx.x, lane = tid & 31;
  const int head = a.state[0], count = a.state[1];
  int64_t kept, pages;
  uint32_t status = scan_batch<false>(a, t, kept, pages);
  if (head < 0 || head >= a.NB || count < 0 || count > a.NB || (status == 0 && count + pages > a.NB))
    status |= MEMOPT_PAGES_CORRUPT;
  uint32_t bits = 0;
  if (status == 0) {
    const int nwarps = gridDim.x * (kThreads / 32);
    for (int b = blockIdx.x * (kThreads / 32) + (tid >> 5); b < a.B; b += nwarps) {
      const int gone = t.page[b + 1] - t.page[b];
      const int first = pages_of(t.old[b], a.BS) - gone;
      int32_t* row = a.tables + static_cast<int64_t>(t.row[b]) * a.MB;
      for (int i = lane; i < gone; i += 32) {
        const int32_t v = row[first + i];
        if (v < 0 || v >= a.NB) bits |= MEMOPT_PAGES_CORRUPT;
        a.ring[(static_cast<int64_t>(head) + count + t.page[b] + i) % a.NB] = v;
        row[first + i] = -1;
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
  if (a.max_tokens > 0x7fffffffLL) return fail(MEMOPT_ERR_UNSUPPORTED, w + ": max_tokens past 2^31");
  if (!a.tables || !a.lens || !a.ring || !a.state || (a.B > 0 && !a.rows))
    return fail(MEMOPT_ERR_INVALID_ARG, w + ": null pointer");
  return MEMOPT_OK;
}

template <typename K>
int launch_pages(K kern, const char* what, const PageArgs& a, int grid, cudaStream_t s) {
  const size_t smem = batch_smem(a.B, a.R);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return cuda_fail(e, what);
  }
  kern<<<grid, kThreads, smem, s>>>(a);
  MEMOPT_LAUNCH_CHECK(what);
  return MEMOPT_OK;
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
             num_blocks, block_size, batch, max_tokens, cu_seqlens, slot_mapping, positions, batch_tables, batch_lens};
  const int st = check_pages("reserve_slots", a);
  if (st != MEMOPT_OK) return st;
  if (!cu_seqlens || (batch > 0 && (!new_lens || !batch_tables || !batch_lens)) ||
      (max_tokens > 0 && (!slot_mapping || !positions)))
    return fail(MEMOPT_ERR_INVALID_ARG, "reserve_slots: null pointer");
  if ((reinterpret_cast<uintptr_t>(slot_mapping) | reinterpret_cast<uintptr_t>(positions)) & 15u)
    return fail(MEMOPT_ERR_INVALID_ARG, "reserve_slots: slot_mapping and positions must be 16-byte aligned");
  // Enough CTAs for one pass over the tokens and the rows, at most two per SM:
  // each CTA repeats the scan of the batch.
  const int64_t by_tokens = (max_tokens + kThreads * kTokensPerThread - 1) / (kThreads * kTokensPerThread);
  const int64_t by_rows = (batch + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t most = static_cast<int64_t>(sm_count()) * 2;
  const int grid = static_cast<int>(std::min(most, std::max<int64_t>(1, std::max(by_tokens, by_rows))));
  return launch_pages(reserve_kernel, "reserve_kernel launch", a, grid, as_stream(stream));
}

extern "C" int memopt_truncate_rows(int32_t* block_tables, int32_t* context_lens, int num_rows, int max_blocks_per_seq,
                                    int32_t* free_pages, int num_blocks, int32_t* pool_state, const int32_t* rows,
                                    const int32_t* keep_lens, int batch, int block_size, void* stream) {
  PageArgs a{block_tables, context_lens, free_pages, pool_state, rows, keep_lens, num_rows, max_blocks_per_seq,
             num_blocks, block_size, batch, 0, nullptr, nullptr, nullptr, nullptr, nullptr};
  const int st = check_pages("truncate_rows", a);
  if (st != MEMOPT_OK) return st;
  if (batch == 0) return MEMOPT_OK;
  const int64_t by_rows = (batch + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t most = static_cast<int64_t>(sm_count()) * 2;
  const int grid = static_cast<int>(std::min(most, by_rows));
  return launch_pages(truncate_kernel, "truncate_kernel launch", a, grid, as_stream(stream));
}
