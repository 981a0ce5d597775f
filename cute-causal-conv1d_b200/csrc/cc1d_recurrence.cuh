// What the tiled recurrence kernels share: pairs of channels, the shared-memory tiles with
// their loads and stores, sequence boundaries and the exchange within a cluster.
//
// A CTA owns a tile of 128 bytes of channels of one batch row and walks the sequence in
// chunks of 64 positions; warp w has the 8 positions 8w .. 8w+7 of each chunk and its lanes
// the tile's channels.  So every boundary between sequences is uniform over a warp, in both
// memory layouts.
#pragma once

#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {

constexpr int kRecWarps = 8;
constexpr int kRecThreads = 32 * kRecWarps;
constexpr int kRecSteps = kRecChunk / kRecWarps;  // positions of a warp in a chunk
constexpr int kRecMaxCluster = 16;
static_assert(kRecSteps == 8, "the tiles' packets and the boundary masks hold 8 positions");

// ------------------------------------------------------------------ V channels of a lane
template <int V> struct Lane;
template <> struct Lane<1> { float v; };
template <> struct Lane<2> { float2 v; };

__device__ __forceinline__ Lane<1> splat(float s, Lane<1>) { return {s}; }
__device__ __forceinline__ Lane<2> splat(float s, Lane<2>) { return {make_float2(s, s)}; }
__device__ __forceinline__ Lane<1> fma(Lane<1> a, Lane<1> b, Lane<1> c) { return {fmaf(a.v, b.v, c.v)}; }
__device__ __forceinline__ Lane<2> fma(Lane<2> a, Lane<2> b, Lane<2> c) { return {ffma2(a.v, b.v, c.v)}; }
__device__ __forceinline__ Lane<1> mul(Lane<1> a, Lane<1> b) { return {a.v * b.v}; }
__device__ __forceinline__ Lane<2> mul(Lane<2> a, Lane<2> b) { return {fmul2(a.v, b.v)}; }
__device__ __forceinline__ Lane<1> add(Lane<1> a, Lane<1> b) { return {a.v + b.v}; }
__device__ __forceinline__ Lane<2> add(Lane<2> a, Lane<2> b) { return {fadd2(a.v, b.v)}; }
__device__ __forceinline__ Lane<1> sub(Lane<1> a, Lane<1> b) { return {a.v - b.v}; }
__device__ __forceinline__ Lane<2> sub(Lane<2> a, Lane<2> b) {
  return {ffma2(b.v, make_float2(-1.f, -1.f), a.v)};
}
template <int V> __device__ __forceinline__ float& el(Lane<V>& a, int i) { return reinterpret_cast<float*>(&a.v)[i]; }
template <int V> __device__ __forceinline__ float el(const Lane<V>& a, int i) { return reinterpret_cast<const float*>(&a.v)[i]; }

// The affine map h -> A h + H of a stretch of positions.  A stretch in which a sequence
// starts does not depend on h at all, not even where h is infinite or NaN: A then has its
// sign bit set (a product of sigmoids never has).
template <int V, bool SEQ>
__device__ __forceinline__ Lane<V> apply(const Lane<V>& A, const Lane<V>& H, const Lane<V>& h) {
  Lane<V> r = fma(A, h, H);
  if constexpr (SEQ) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (__float_as_int(el(A, i)) < 0) el(r, i) = el(H, i);
  }
  return r;
}
// A of the map (A2, .) after (A1, .).
template <int V, bool SEQ>
__device__ __forceinline__ Lane<V> chain(const Lane<V>& A2, const Lane<V>& A1) {
  Lane<V> r = mul(A2, A1);
  if constexpr (SEQ) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (__float_as_int(el(A2, i)) < 0) el(r, i) = el(A2, i);
  }
  return r;
}

// ----------------------------------------------------------------------------- the tiles
// SKEW (16-bit only): rows that do not all start on a 4-byte boundary are copied in the
// 4-byte words that cover them, so a row lies in its tile as it does in memory, half a word
// late where it starts in the middle of one.
template <typename T, int LAYOUT, bool SKEW> struct Tile {
  static constexpr int kSize = sizeof(T);
  static constexpr int V = 4 / kSize;                // channels per lane
  static constexpr int kChannels = 32 * V;           // 128 bytes
  static constexpr int kPacket = 16 / kSize;         // elements per 16 bytes
  static constexpr bool kRows = LAYOUT == kLayoutRows;
  // channel-last: 64 rows of 128 bytes, rows 8w.. written and read by warp w alone.
  // rows: a row of 64 positions per channel, 16 bytes longer so that the 16-byte reads of
  // 8 lanes (8 channels) fall into different banks.
  static constexpr int kPitch = kRows ? kRecChunk * kSize + 16 : SKEW ? 132 : 128;
  static constexpr int kBytes = kRows ? kChannels * kPitch : kRecChunk * kPitch;
};

// Channel of value i of a lane within the tile: neighbours share a 4-byte word of a
// channel-last row; with rows they are two rows half a tile apart.
template <typename T, int LAYOUT>
__device__ __forceinline__ int lane_channel(int lane, int i) {
  return LAYOUT == kLayoutRows ? lane + 32 * i : lane * static_cast<int>(4 / sizeof(T)) + i;
}

// One of the (batch, dim, seqlen) tensors as a CTA sees it: its tile of channels in its batch
// row.  `origin` is the tensor's first element: nothing before it is read.
template <typename T>
struct Strip {
  T* origin;
  T* row;       // at channel d0, position 0
  int64_t s1, s2;
  unsigned off; // packed: byte offset of the thread's first packet from (d0, t0)
};

__device__ __forceinline__ void cp16(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <typename T, int LAYOUT, bool SKEW>
__device__ __forceinline__ Strip<T> strip_of(const TensorArg& t, int64_t b, int64_t d0) {
  using C = Tile<T, LAYOUT, SKEW>;
  Strip<T> s;
  s.origin = static_cast<T*>(t.data);
  s.row = s.origin + b * t.s0 + d0 * t.s1;
  s.s1 = t.s1;
  s.s2 = t.s2;
  // below 2^32 for packed tensors (rec_plan)
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if constexpr (C::kRows) {
    constexpr int PR = kRecChunk / C::kPacket;
    s.off = (static_cast<unsigned>(threadIdx.x / PR) * static_cast<unsigned>(t.s1) + (threadIdx.x % PR) * C::kPacket) * C::kSize;
  } else {
    s.off = (static_cast<unsigned>(w * kRecSteps + (lane >> 3)) * static_cast<unsigned>(t.s2) + (lane & 7) * C::kPacket) * C::kSize;
  }
  return s;
}

// Starts the copy of a chunk (positions t0 .. t0 + nt - 1 of nd channels) into its tile;
// places outside are zero.  packed: 16-byte packets, aligned (rec_plan);
// SKEW: 4-byte words; else element by element at any strides.  Channel-last: each warp
// copies what it reads itself.
template <typename T, int LAYOUT, bool SKEW>
__device__ __forceinline__ void load_tile(unsigned tile, unsigned char* tile_ptr, const Strip<T>& t, int64_t t0, int nd, int nt, bool packed) {
  using C = Tile<T, LAYOUT, SKEW>;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if constexpr (SKEW) {
    constexpr int R = C::kRows ? C::kChannels : kRecSteps;  // rows: the CTA's, or the warp's own
    const int64_t step = C::kRows ? t.s1 : t.s2;
    const int first = C::kRows ? 0 : w * kRecSteps;
    const int rows = C::kRows ? nd : nt, len = C::kRows ? nt : nd;
    const T* const base = t.row + (C::kRows ? t0 : t0 * t.s2);
    // word i of a row covers elements 2i - skew and 2i + 1 - skew
    auto word = [&](int r, int i) {
      const T* p = base + r * step;
      const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1;
      const int e = 2 * i - skew;  // its first element in the row
      const int n = r < rows ? max(0, min(2, len - e)) : 0;
      const unsigned dst = tile + r * C::kPitch + i * 4;
      if (n > 0 && p + e < t.origin) {  // half of the word lies before the tensor
        *reinterpret_cast<uint32_t*>(tile_ptr + r * C::kPitch + i * 4) = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + e + 1)) << 16;
      } else {
        cp4(dst, n > 0 ? p + e : t.origin + (reinterpret_cast<uintptr_t>(t.origin) >> 1 & 1), n * 2);
      }
    };
    if constexpr (C::kRows) {
#pragma unroll 4
      for (int k = 0; k < R / kRecWarps; ++k) word(w * (R / kRecWarps) + k, lane);
      if (threadIdx.x < R) word(threadIdx.x, 32);
    } else {
#pragma unroll
      for (int k = 0; k < R; ++k) word(first + k, lane);
      if (lane < R) word(first + lane, 32);
    }
    return;
  } else {
    if (packed) {
      if constexpr (C::kRows) {
        constexpr int PR = kRecChunk / C::kPacket;          // packets of a row
        constexpr int CR = kRecThreads / PR;                // rows a pass of the threads covers
        const char* const src = reinterpret_cast<const char*>(t.row + t0);
        const int c0 = threadIdx.x / PR, p = (threadIdx.x % PR) * C::kPacket;
        const int n = max(0, min(C::kPacket, nt - p)) * C::kSize;
#pragma unroll
        for (int k = 0; k < C::kChannels / CR; ++k) {
          const int m = c0 + k * CR < nd ? n : 0;
          cp16(tile + (c0 + k * CR) * C::kPitch + p * C::kSize, m ? src + k * CR * t.s1 * C::kSize + t.off : reinterpret_cast<const char*>(t.origin), m);
        }
      } else {
        const int n = max(0, min(C::kPacket, nd - (lane & 7) * C::kPacket)) * C::kSize;
        const char* const src = reinterpret_cast<const char*>(t.row + t0 * t.s2);
        const int r = w * kRecSteps + (lane >> 3);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int m = r + 4 * k < nt ? n : 0;
          cp16(tile + (r + 4 * k) * C::kPitch + (lane & 7) * 16, m ? src + 4 * k * t.s2 * C::kSize + t.off : reinterpret_cast<const char*>(t.origin), m);
        }
      }
      return;
    }
    const T* src = t.row + t0 * t.s2;
    constexpr int N = C::kRows ? C::kChannels * kRecChunk / kRecThreads : kRecSteps * C::V;
#pragma unroll 4
    for (int k = 0; k < N; ++k) {
      int ch, p;
      if constexpr (C::kRows) {
        const int i = threadIdx.x + k * kRecThreads;
        ch = i / kRecChunk;
        p = i % kRecChunk;
      } else {
        ch = lane + 32 * (k % C::V);
        p = w * kRecSteps + k / C::V;
      }
      const bool in = ch < nd && p < nt;
      const int o = C::kRows ? ch * C::kPitch + p * C::kSize : p * C::kPitch + ch * C::kSize;
      const T* from = in ? src + ch * t.s1 + p * t.s2 : t.origin;
      if constexpr (C::kSize == 4) {
        cp4(tile + o, from, in ? 4 : 0);
      } else {
        *reinterpret_cast<T*>(tile_ptr + o) = in ? *from : from_f32<T>(0.f);
      }
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ void widen(const uint32_t (&r)[N], float2 (&v)[N]) {
  unpack2<T, 2 * N>(*reinterpret_cast<const Packet<T, 2 * N>*>(&r), v);
}

// The 8 positions of warp w and the lane's V channels, as fp32.
template <typename T, int LAYOUT, bool SKEW>
__device__ __forceinline__ void read_steps(const unsigned char* tile, const Strip<T>& t, int64_t t0, int w, int lane,
                                           Lane<Tile<T, LAYOUT, SKEW>::V> (&f)[kRecSteps]) {
  using C = Tile<T, LAYOUT, SKEW>;
  if constexpr (C::kRows) {
#pragma unroll
    for (int i = 0; i < C::V; ++i) {
      const unsigned char* p = tile + (lane + 32 * i) * C::kPitch + w * kRecSteps * C::kSize;
#pragma unroll
      for (int q = 0; q < kRecSteps / C::kPacket; ++q) {
        uint4 u = *reinterpret_cast<const uint4*>(p + q * 16);
        if constexpr (SKEW) {
          const uint32_t next = *reinterpret_cast<const uint32_t*>(p + 16);
          const unsigned sh = (reinterpret_cast<uintptr_t>(t.row + t0 + (lane + 32 * i) * t.s1) & 2) * 8;
          u = make_uint4(__funnelshift_r(u.x, u.y, sh), __funnelshift_r(u.y, u.z, sh), __funnelshift_r(u.z, u.w, sh),
                         __funnelshift_r(u.w, next, sh));
        }
        float2 v[C::kPacket / 2];
        unpack2<T, C::kPacket>(*reinterpret_cast<const Packet<T, C::kPacket>*>(&u), v);
#pragma unroll
        for (int j = 0; j < C::kPacket / 2; ++j) {
          el(f[q * C::kPacket + 2 * j], i) = v[j].x;
          el(f[q * C::kPacket + 2 * j + 1], i) = v[j].y;
        }
      }
    }
  } else {
    const unsigned char* p = tile + w * kRecSteps * C::kPitch + lane * 4;
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if constexpr (C::V == 2) {
        uint32_t u = *reinterpret_cast<const uint32_t*>(p + j * C::kPitch);
        if constexpr (SKEW) {
          const unsigned sh = (reinterpret_cast<uintptr_t>(t.row + (t0 + w * kRecSteps + j) * t.s2) & 2) * 8;
          u = __funnelshift_r(u, *reinterpret_cast<const uint32_t*>(p + j * C::kPitch + 4), sh);
        }
        float2 v[1];
        unpack2<T, 2>(*reinterpret_cast<const Packet<T, 2>*>(&u), v);
        f[j].v = v[0];
      } else {
        f[j].v = *reinterpret_cast<const float*>(p + j * C::kPitch);
      }
    }
  }
}

// rows: puts 8 positions back into a tile (without a skew), to be stored by store_tile.
template <typename T, bool SKEW>
__device__ __forceinline__ void write_steps(unsigned char* tile, int w, int lane, const Lane<4 / sizeof(T)> (&f)[kRecSteps]) {
  using C = Tile<T, kLayoutRows, SKEW>;
#pragma unroll
  for (int i = 0; i < C::V; ++i) {
    unsigned char* p = tile + (lane + 32 * i) * C::kPitch + w * kRecSteps * C::kSize;
#pragma unroll
    for (int q = 0; q < kRecSteps / C::kPacket; ++q) {
      float2 v[C::kPacket / 2];
#pragma unroll
      for (int j = 0; j < C::kPacket / 2; ++j)
        v[j] = make_float2(el(f[q * C::kPacket + 2 * j], i), el(f[q * C::kPacket + 2 * j + 1], i));
      *reinterpret_cast<Packet<T, C::kPacket>*>(p + q * 16) = pack2<T, C::kPacket>(v);
    }
  }
}

// rows: stores a tile.  Without a skew each thread takes the elements that it also loads, so a
// load into the same tile may follow without a barrier.
template <typename T, bool SKEW>
__device__ __forceinline__ void store_tile(const unsigned char* tile, const Strip<T>& t, int64_t t0, int nd, int nt, bool packed) {
  using C = Tile<T, kLayoutRows, SKEW>;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if constexpr (SKEW) {
    // words of the row in memory: element 2i - skew and its successor
    auto word = [&](int r, int i) {
      if (r >= nd) return;
      T* p = t.row + t0 + r * t.s1;
      const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1;
      const int e = 2 * i - skew;
      const unsigned char* s = tile + r * C::kPitch;
      if (e >= 0 && e + 1 < nt) {
        const uint32_t lo = *reinterpret_cast<const uint32_t*>(s + (e & ~1) * 2);
        const uint32_t hi = *reinterpret_cast<const uint32_t*>(s + (e & ~1) * 2 + 4);
        *reinterpret_cast<uint32_t*>(p + e) = __funnelshift_r(lo, hi, skew * 16);
      } else {
        if (e >= 0 && e < nt) p[e] = *reinterpret_cast<const T*>(s + e * 2);
        if (e + 1 >= 0 && e + 1 < nt) p[e + 1] = *reinterpret_cast<const T*>(s + e * 2 + 2);
      }
    };
#pragma unroll 4
    for (int k = 0; k < C::kChannels / kRecWarps; ++k) word(w * (C::kChannels / kRecWarps) + k, lane);
    if (threadIdx.x < C::kChannels) word(threadIdx.x, 32);
  } else if (packed) {
    constexpr int PR = kRecChunk / C::kPacket;
    constexpr int CR = kRecThreads / PR;
    char* const dst = reinterpret_cast<char*>(t.row + t0);
    const int c0 = threadIdx.x / PR, p = (threadIdx.x % PR) * C::kPacket;
#pragma unroll
    for (int k = 0; k < C::kChannels / CR; ++k) {
      if (c0 + k * CR >= nd || p >= nt) continue;
      const Packet<T, C::kPacket> r = *reinterpret_cast<const Packet<T, C::kPacket>*>(tile + (c0 + k * CR) * C::kPitch + p * C::kSize);
      T* o = reinterpret_cast<T*>(dst + k * CR * t.s1 * C::kSize + t.off);
      if (p + C::kPacket <= nt) {
        st_packet<T, C::kPacket>(o, r);
      } else {
#pragma unroll
        for (int j = 0; j < C::kPacket; ++j)
          if (p + j < nt) o[j] = r.v[j];
      }
    }
  } else {
    T* dst = t.row + t0 * t.s2;
#pragma unroll 4
    for (int k = 0; k < C::kChannels * kRecChunk / kRecThreads; ++k) {
      const int i = threadIdx.x + k * kRecThreads;
      const int ch = i / kRecChunk, p = i % kRecChunk;
      if (ch < nd && p < nt) dst[ch * t.s1 + p * t.s2] = *reinterpret_cast<const T*>(tile + ch * C::kPitch + p * C::kSize);
    }
  }
}

// channel-last: stores the 8 positions of warp w, nt of them within the sequence.  nch: how
// many of the lane's channels there are.
template <typename T, bool SKEW>
__device__ __forceinline__ void store_steps(const Strip<T>& t, int64_t tw, int lane, int nch, int left, bool packed,
                                            const Lane<4 / sizeof(T)> (&f)[kRecSteps]) {
  constexpr int V = 4 / sizeof(T);
  char* const row = reinterpret_cast<char*>(t.row + tw * t.s2);
  if (!SKEW && packed && nch == V) {
    const unsigned o = lane * 4u;
    auto put = [&](int j) {
      char* p = row + j * t.s2 * static_cast<int64_t>(sizeof(T)) + o;
      if constexpr (V == 2) {
        float2 v[1] = {f[j].v};
        st_packet<T, 2>(reinterpret_cast<T*>(p), pack2<T, 2>(v));
      } else {
        *reinterpret_cast<float*>(p) = f[j].v;
      }
    };
    if (left >= kRecSteps) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) put(j);
    } else {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j)
        if (j < left) put(j);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {
    if (j >= left) break;
    T* p = t.row + (tw + j) * t.s2 + lane * V * t.s1;
    if (nch > 0) p[0] = from_f32<T>(el(f[j], 0));
    if (V > 1 && nch > 1) p[t.s1] = from_f32<T>(el(f[j], V - 1));
  }
}

// ---------------------------------------------------------------- sequence boundaries
// Of the 8 positions of a warp: which hold a token, which start a sequence, which end one,
// and (lane 1 + j) the id of position j.
struct Edges {
  unsigned valid, first, last;
  int id;
};
// ids of positions t - 1 .. t + 8, one per lane 0 .. 9; -1 outside the sequence.
__device__ __forceinline__ int load_ids(const RecArgs& a, int64_t b, int64_t t, int lane) {
  const int64_t p = t - 1 + lane;
  if (lane > 9 || p < 0 || p >= a.seqlen) return -1;
  return __ldg(static_cast<const int*>(a.seq_idx.data) + b * a.seq_idx.s0 + p * a.seq_idx.s1);
}
__device__ __forceinline__ Edges edges_of(int id) {
  constexpr unsigned all = 0xffffffffu;
  const int before = __shfl_up_sync(all, id, 1), after = __shfl_down_sync(all, id, 1);
  Edges e;
  e.id = id;
  e.valid = (__ballot_sync(all, id >= 0) >> 1) & 0xffu;
  e.first = (__ballot_sync(all, id >= 0 && id != before) >> 1) & 0xffu;
  e.last = (__ballot_sync(all, id >= 0 && id != after) >> 1) & 0xffu;
  return e;
}

// Row n of a (nstates, dim) fp32 tensor at the lane's channels; zero outside.
template <typename T, int LAYOUT>
__device__ __forceinline__ Lane<4 / sizeof(T)> load_state(const TensorArg& s, int64_t n, int64_t nstates, int64_t d0, int64_t dim, int lane) {
  Lane<4 / sizeof(T)> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(4 / sizeof(T)); ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    el(r, i) = s.data && n >= 0 && n < nstates && d < dim ? static_cast<const float*>(s.data)[n * s.s0 + d * s.s1] : 0.f;
  }
  return r;
}
template <typename T, int LAYOUT>
__device__ __forceinline__ void store_state(const TensorArg& s, int64_t n, int64_t nstates, int64_t d0, int64_t dim, int lane,
                                            const Lane<4 / sizeof(T)>& f) {
  if (!s.data || n < 0 || n >= nstates) return;
#pragma unroll
  for (int i = 0; i < static_cast<int>(4 / sizeof(T)); ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    if (d < dim) static_cast<float*>(s.data)[n * s.s0 + d * s.s1] = el(f, i);
  }
}

// ------------------------------------------------------------------------- clusters
// A map of a stretch of positions, as it travels between warps and CTAs.
template <int V> struct alignas(8 * V) Map { Lane<V> A, H; };

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void mbar_init(unsigned bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_init_done() { asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory"); }
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for the phase of that parity, at most about 2^20 tries of the hardware's own waiting
// time; returns whether it came.  The partners run at the same time (one cluster), so it does.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity) {
  for (int i = 0; i < (1 << 20); ++i) {
    unsigned done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
  }
  return false;
}
// Writes m to the place of `local` in the shared memory of CTA `rank`, and counts its bytes on
// that CTA's barrier at the place of `bar`: data and signal in one, without a fence that
// would wait for this CTA's stores to global memory.
template <int V>
__device__ __forceinline__ void send_map(unsigned local, unsigned bar, unsigned rank, const Map<V>& m) {
  unsigned to, on;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(to) : "r"(local), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(on) : "r"(bar), "r"(rank));
  if constexpr (V == 2) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];\n" ::"r"(to),
                 "f"(m.A.v.x), "f"(m.A.v.y), "f"(m.H.v.x), "f"(m.H.v.y), "r"(on) : "memory");
  } else {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];\n" ::"r"(to),
                 "f"(m.A.v), "f"(m.H.v), "r"(on) : "memory");
  }
}

}  // namespace cc1d
