// Copies of pages of the 8-bit key/value cache: what a fork does not share, a
// compaction, a move into another pool.
//
// A page is H runs of K, of V and of the record, and 2 H scales; whole pages are one
// stretch of memory. One CTA copies up to 32 KB of K and as much of V of a page of a
// layer, 16 bytes a thread and load; all layers are in the grid, since a fork of a
// few pages is all launches. Two copies must not write one page, nor one read what
// another writes: up to 512 pairs, every CTA looks through all of them (4 KB, while
// its own page is on the way it costs nothing that shows); more are counted page by
// page first, which takes two launches (5 us) and would cost n^2 reads otherwise.
// Bound by memory. Measured: 1500 pages of 98 KB with records in each of 4 layers, 208
// us for 1.23 GB, 5.9 TB/s (0.90 of the copy rate); 1999 pages of 262 KB in 2 layers, 339
// us for 2.1 GB, 6.2 TB/s (0.95); 8 half full pages of 6 layers, 5 us of a call of 19.
#include "kv8_common.cuh"

#include <algorithm>

namespace kf {

constexpr int KV8_COPY_THREADS = 256;
constexpr int KV8_COPY_MOST = 256;       // layers of a call
constexpr int KV8_COPY_LAYERS = 32;      // layers of a launch
constexpr int KV8_COPY_SCAN = 512;       // pairs that every CTA looks through

struct KV8CopyLayer {
  const uint8_t *k, *v;
  const float *scale, *weight;
  uint8_t *k_to, *v_to;
  float *scale_to, *weight_to;
};
struct KV8CopyLayers {
  KV8CopyLayer at[KV8_COPY_LAYERS];
};

struct KV8Copy {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;   // or null: whole pages
  uint32_t* names;         // many pairs: how many copies name a page, [pages]
  int64_t pages_from, pages_to;
  int64_t n;
  int H, P, D;
  int parts;               // CTAs of a page of a layer
  bool same;               // one pool
};

// Tokens that pair i copies. 0: it copies nothing. *bad: an entry is no page.
__device__ __forceinline__ int kv8_copy_tokens(const KV8Copy& a, int64_t i, int* src, int* dst,
                                               bool* bad) {
  const int s = __ldg(a.src + i), d = __ldg(a.dst + i);
  const int t = a.tokens ? __ldg(a.tokens + i) : a.P;
  *src = s;
  *dst = d;
  *bad = s < 0 || s >= a.pages_from || d < 0 || d >= a.pages_to;
  if (*bad || t <= 0 || (a.same && s == d)) return 0;
  return t < a.P ? t : a.P;
}

// Many pairs: names[page] is the number of copies that write it and, within one
// pool, twice the number that read it. 1: its writer is alone.
__global__ void __launch_bounds__(KV8_COPY_THREADS) kv8_copy_names_kernel(KV8Copy a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * KV8_COPY_THREADS + threadIdx.x;
  if (i >= a.n) return;
  int s, d;
  bool bad;
  if (kv8_copy_tokens(a, i, &s, &d, &bad) == 0) return;
  atomicAdd(a.names + d, 1u);
  if (a.same) atomicAdd(a.names + s, 2u);
}

__global__ void __launch_bounds__(KV8_COPY_THREADS)
    kv8_copy_kernel(KV8CopyLayers layers, KV8Copy a) {
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int64_t i = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - i * a.parts);
  int src, dst;
  bool bad;
  const int tokens = kv8_copy_tokens(a, i, &src, &dst, &bad);
  if (tokens == 0) {
    if (bad && tid == 0) record_device_status(KF_DEV_BAD_KV_PAGE);
    return;
  }
  int clash = 0;
  if (a.names) {
    clash = a.names[dst] != 1u;
  } else {
    for (int64_t j = tid; j < a.n; j += KV8_COPY_THREADS) {
      int s, d;
      bool other;
      if (j != i && kv8_copy_tokens(a, j, &s, &d, &other) > 0 && (d == dst || (a.same && s == dst)))
        clash = 1;
    }
    clash = __syncthreads_or(clash);
  }
  if (clash) {
    if (tid == 0) record_device_status(KF_DEV_BAD_KV_PAGE);
    return;
  }
  const KV8CopyLayer& l = layers.at[blockIdx.y];
  const int64_t page = static_cast<int64_t>(a.H) * a.P * a.D;
  const int run = tokens * a.D / 16;         // 16-byte pieces of a head
  const int pitch = a.P * a.D / 16;
  const uint4* from[2] = {reinterpret_cast<const uint4*>(l.k + src * page),
                          reinterpret_cast<const uint4*>(l.v + src * page)};
  uint4* to[2] = {reinterpret_cast<uint4*>(l.k_to + dst * page),
                  reinterpret_cast<uint4*>(l.v_to + dst * page)};
  const int total = a.H * run;
  for (int u = part * KV8_COPY_THREADS + tid; u < total; u += a.parts * KV8_COPY_THREADS) {
    const int h = u / run;
    const int at = h * pitch + (u - h * run);
    to[0][at] = from[0][at];
    to[1][at] = from[1][at];
  }
  if (part) return;
  for (int u = tid; u < 2 * a.H; u += KV8_COPY_THREADS)
    l.scale_to[static_cast<int64_t>(dst) * 2 * a.H + u] = l.scale[static_cast<int64_t>(src) * 2 * a.H + u];
  if (l.weight && l.weight_to)
    for (int u = tid; u < a.H * a.P; u += KV8_COPY_THREADS)
      if ((u & (a.P - 1)) < tokens)
        l.weight_to[static_cast<int64_t>(dst) * a.H * a.P + u] =
            l.weight[static_cast<int64_t>(src) * a.H * a.P + u];
}

// ---------------------------------------------------------------- host

static bool kv8_alike(const KV8& a, const KV8& b) {
  return a.H == b.H && a.D == b.D && a.P == b.P && a.fmt == b.fmt;
}

// Whether a tensor that the call writes has memory in common with another one that
// it writes, or with one that it reads (within one pool: but for the same tensor of
// the same layer). The pairs are checked for clashes within a tensor only, so the
// result would depend on the order of CTAs.
struct KV8Range {
  uintptr_t at, end;
  bool written;
};
static bool kv8_copy_overlaps(const KV8CopyLayers* at, int64_t layers, bool same, const KV8& from,
                              const KV8& into) {
  KV8Range all[8 * KV8_COPY_MOST];
  int64_t n = 0;
  auto add = [&](const void* p, int64_t bytes, bool written) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    if (bytes > 0) all[n++] = {a, a + static_cast<uintptr_t>(bytes), written};
  };
  const int64_t codes = static_cast<int64_t>(from.H) * from.P * from.D;
  auto pool = [&](const void* k, const void* v, const void* scale, const void* weight, int64_t pages,
                  bool written) {
    add(k, pages * codes, written);
    add(v, pages * codes, written);
    add(scale, pages * from.H * 8, written);
    if (weight) add(weight, pages * from.H * from.P * 4, written);
  };
  for (int64_t i = 0; i < layers; ++i) {
    const KV8CopyLayer& l = at[i / KV8_COPY_LAYERS].at[i % KV8_COPY_LAYERS];
    const bool record = l.weight && l.weight_to;
    pool(l.k_to, l.v_to, l.scale_to, record ? l.weight_to : nullptr, into.pages, true);
    if (!same) pool(l.k, l.v, l.scale, record ? l.weight : nullptr, from.pages, false);
  }
  std::sort(all, all + n, [](const KV8Range& a, const KV8Range& b) { return a.at < b.at; });
  uintptr_t end = 0, end_written = 0;   // of what began earlier
  for (int64_t i = 0; i < n; ++i) {
    if (all[i].at < (all[i].written ? end : end_written)) return true;
    end = std::max(end, all[i].end);
    if (all[i].written) end_written = std::max(end_written, all[i].end);
  }
  return false;
}

}  // namespace kf

using namespace kf;

extern "C" int64_t kf_kv8_copy_workspace_bytes(const kf_kv8_cache* from, const kf_kv8_cache* into,
                                               int64_t n) {
  KV8 a, b;
  if (kv8_view("kf_kv8_copy_workspace_bytes", from, &a) ||
      kv8_view("kf_kv8_copy_workspace_bytes", into, &b))
    return -1;
  return n <= KV8_COPY_SCAN ? 0 : b.pages * 4;
}

extern "C" int kf_kv8_copy(const kf_kv8_cache* const* from, const kf_kv8_cache* const* into,
                           int64_t layers, const int32_t* src, const int32_t* dst,
                           const int32_t* tokens, int64_t n, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  const char* what = "kf_kv8_copy";
  if (layers < 0 || layers > KV8_COPY_MOST || n < 0 || n > (1LL << 29) || (layers && (!from || !into))) {
    set_last_error("%s: needs 0 <= layers <= 256, their caches, and 0 <= n <= 2^29", what);
    return KF_E_INVALID;
  }
  if (layers == 0) return KF_OK;
  KV8 first, first_to;
  KV8CopyLayers at[KV8_COPY_MOST / KV8_COPY_LAYERS];
  bool same = false;
  for (int64_t i = 0; i < layers; ++i) {
    KV8 a, b;
    int rc = kv8_view(what, from[i], &a);
    if (!rc) rc = kv8_view(what, into[i], &b);
    if (rc) return rc;
    if (i == 0) {
      first = a;
      first_to = b;
      same = a.k == b.k;
    }
    if (!kv8_alike(a, first) || !kv8_alike(b, first) || a.pages != first.pages ||
        b.pages != first_to.pages) {
      set_last_error("%s: the caches of a call must be alike", what);
      return KF_E_INVALID;
    }
    if (same != (a.k == b.k) || same != (a.v == b.v) || same != (a.scale == b.scale) ||
        (same && (a.pages != b.pages || a.weight != b.weight))) {
      set_last_error("%s: from and into must be one pool, or two without a tensor in common", what);
      return KF_E_INVALID;
    }
    at[i / KV8_COPY_LAYERS].at[i % KV8_COPY_LAYERS] = {a.k, a.v, a.scale, a.weight,
                                                       b.k, b.v, b.scale, b.weight};
  }
  if (n == 0) return KF_OK;
  if (!src || !dst) {
    set_last_error("%s: src and dst must not be null", what);
    return KF_E_INVALID;
  }
  const int64_t need = n <= KV8_COPY_SCAN ? 0 : first_to.pages * 4;
  if (need && (!workspace || workspace_bytes < need || !kv8_aligned(workspace, 16))) {
    set_last_error("%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
    return KF_E_INVALID;
  }
  if (kv8_copy_overlaps(at, layers, same, first, first_to)) {
    set_last_error("%s: a tensor that is written occurs twice, or is read too", what);
    return KF_E_INVALID;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KV8Copy c = {src, dst, tokens, need ? static_cast<uint32_t*>(workspace) : nullptr, first.pages,
               first_to.pages, n, first.H, first.P, first.D, 1, same};
  const int64_t pieces = static_cast<int64_t>(first.H) * first.P * first.D / 16;
  const int64_t parts = (pieces + KV8_COPY_THREADS * 8 - 1) / (KV8_COPY_THREADS * 8);
  c.parts = static_cast<int>(parts);
  if (n * parts > INT32_MAX) {
    set_last_error("%s: too many pages for one call", what);
    return KF_E_UNSUPPORTED;
  }
  cudaError_t e;
  if (need) {
    e = cudaMemsetAsync(workspace, 0, need, st);
    if (e != cudaSuccess) return cuda_status(e, "kf_kv8_copy memset");
    e = launch_chained(kv8_copy_names_kernel,
                       dim3(static_cast<unsigned>((n + KV8_COPY_THREADS - 1) / KV8_COPY_THREADS)),
                       dim3(KV8_COPY_THREADS), 0, st, c);
    if (e != cudaSuccess) return cuda_status(e, "kf_kv8_copy names launch");
  }
  for (int64_t i = 0; i < layers; i += KV8_COPY_LAYERS) {
    const int64_t m = layers - i < KV8_COPY_LAYERS ? layers - i : KV8_COPY_LAYERS;
    e = launch_chained(kv8_copy_kernel,
                       dim3(static_cast<unsigned>(n * parts), static_cast<unsigned>(m)),
                       dim3(KV8_COPY_THREADS), 0, st, at[i / KV8_COPY_LAYERS], c);
    if (e != cudaSuccess) return cuda_status(e, "kf_kv8_copy launch");
  }
  return KF_OK;
}
