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
template <typename T, int LAYOUT> struct Tile {
  static constexpr int kSize = sizeof(T);
  static constexpr int V = 4 / kSize;                // channels per lane
  static constexpr int kChannels = 32 * V;           // 128 bytes
  static constexpr int kPacket = 16 / kSize;         // elements per 16 bytes
  static constexpr bool kRows = LAYOUT == kLayoutRows;
  // channel-last: 64 rows of 128 bytes, rows 8w.. written and read by warp w alone.
  // rows: a row of 64 positions per channel, 16 bytes longer so that the 16-byte reads of
  // 8 lanes (8 channels) fall into different banks.
  static constexpr int kPitch = kRows ? kRecChunk * kSize + 16 : 128;
  static constexpr int kBytes = kRows ? kChannels * kPitch : kRecChunk * kPitch;
};

// Channel of value i of a lane within the tile: neighbours share a 4-byte word of a
// channel-last row; with rows they are two rows half a tile apart.
template <typename T, int LAYOUT>
__device__ __forceinline__ int lane_channel(int lane, int i) {
  return Tile<T, LAYOUT>::kRows ? lane + 32 * i : lane * Tile<T, LAYOUT>::V + i;
}

// Starts the copy of one tensor's chunk into its tile.  packed: 16-byte packets, aligned (the
// host has checked); else element by element at any strides.  Places outside the tensor are
// zero.  Channel-last: each warp copies what it reads itself.
template <typename T, int LAYOUT>
__device__ __forceinline__ void load_tile(unsigned char* tile, const T* base, int64_t s1, int64_t s2, int64_t d0,
                                          int64_t t0, int64_t dim, int64_t seqlen, bool packed) {
  using C = Tile<T, LAYOUT>;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int nd = static_cast<int>(min(dim - d0, static_cast<int64_t>(C::kChannels)));
  const int nt = static_cast<int>(min(seqlen - t0, static_cast<int64_t>(kRecChunk)));
  if (packed) {
    if constexpr (C::kRows) {
      constexpr int PR = kRecChunk / C::kPacket;
      const T* src = base + d0 * s1 + t0;
#pragma unroll
      for (int k = 0; k < C::kChannels * PR / kRecThreads; ++k) {
        const int i = threadIdx.x + k * kRecThreads;
        const int ch = i / PR, t = (i % PR) * C::kPacket;
        const int n = ch < nd ? max(0, min(C::kPacket, nt - t)) : 0;
        const unsigned s = static_cast<unsigned>(__cvta_generic_to_shared(tile + ch * C::kPitch + t * C::kSize));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(n ? src + ch * s1 + t : base),
                     "r"(n * C::kSize) : "memory");
      }
    } else {
      const int c = (lane & 7) * C::kPacket;
      const int n = max(0, min(C::kPacket, nd - c));
      const T* src = base + d0 + c + t0 * s2;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int t = w * kRecSteps + k * 4 + (lane >> 3);
        const int m = t < nt ? n : 0;
        const unsigned s = static_cast<unsigned>(__cvta_generic_to_shared(tile + t * C::kPitch + (lane & 7) * 16));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(m ? src + t * s2 : base),
                     "r"(m * C::kSize) : "memory");
      }
    }
    return;
  }
  const T* src = base + d0 * s1 + t0 * s2;
  constexpr int N = C::kRows ? C::kChannels * kRecChunk / kRecThreads : kRecSteps * C::V;
#pragma unroll 4
  for (int k = 0; k < N; ++k) {
    int ch, t;
    if constexpr (C::kRows) {
      const int i = threadIdx.x + k * kRecThreads;
      ch = i / kRecChunk;
      t = i % kRecChunk;
    } else {
      ch = lane + 32 * (k % C::V);
      t = w * kRecSteps + k / C::V;
    }
    const bool in = ch < nd && t < nt;
    unsigned char* dst = tile + (C::kRows ? ch * C::kPitch + t * C::kSize : t * C::kPitch + ch * C::kSize);
    const T* from = in ? src + ch * s1 + t * s2 : base;
    if constexpr (C::kSize == 4) {
      cp_async_packet<4>(dst, from, in);
    } else {
      *reinterpret_cast<T*>(dst) = in ? *from : from_f32<T>(0.f);
    }
  }
}

// The 8 positions of warp w and the lane's V channels, as fp32.
template <typename T, int LAYOUT>
__device__ __forceinline__ void read_steps(const unsigned char* tile, int w, int lane, Lane<Tile<T, LAYOUT>::V> (&f)[kRecSteps]) {
  using C = Tile<T, LAYOUT>;
  if constexpr (C::kRows) {
#pragma unroll
    for (int i = 0; i < C::V; ++i) {
      const unsigned char* p = tile + (lane + 32 * i) * C::kPitch + w * kRecSteps * C::kSize;
#pragma unroll
      for (int q = 0; q < kRecSteps / C::kPacket; ++q) {
        Packet<T, C::kPacket> r = *reinterpret_cast<const Packet<T, C::kPacket>*>(p + q * 16);
        float2 v[C::kPacket / 2];
        unpack2<T, C::kPacket>(r, v);
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
        Packet<T, 2> r = *reinterpret_cast<const Packet<T, 2>*>(p + j * C::kPitch);
        float2 v[1];
        unpack2<T, 2>(r, v);
        f[j].v = v[0];
      } else {
        f[j].v = *reinterpret_cast<const float*>(p + j * C::kPitch);
      }
    }
  }
}

// rows: puts 8 positions back into a tile, to be stored from there by store_tile.
template <typename T, int LAYOUT>
__device__ __forceinline__ void write_steps(unsigned char* tile, int w, int lane, const Lane<Tile<T, LAYOUT>::V> (&f)[kRecSteps]) {
  using C = Tile<T, LAYOUT>;
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

// rows: stores a tile; each thread takes the packets that it also loads (packed), so a load
// into the same tile may follow without a barrier.
template <typename T>
__device__ __forceinline__ void store_tile(const unsigned char* tile, T* base, int64_t s1, int64_t s2, int64_t d0,
                                           int64_t t0, int64_t dim, int64_t seqlen, bool packed) {
  using C = Tile<T, kLayoutRows>;
  const int nd = static_cast<int>(min(dim - d0, static_cast<int64_t>(C::kChannels)));
  const int nt = static_cast<int>(min(seqlen - t0, static_cast<int64_t>(kRecChunk)));
  T* dst = base + d0 * s1 + t0 * s2;
  if (packed) {
    constexpr int PR = kRecChunk / C::kPacket;
#pragma unroll
    for (int k = 0; k < C::kChannels * PR / kRecThreads; ++k) {
      const int i = threadIdx.x + k * kRecThreads;
      const int ch = i / PR, t = (i % PR) * C::kPacket;
      if (ch >= nd || t >= nt) continue;
      const Packet<T, C::kPacket> r = *reinterpret_cast<const Packet<T, C::kPacket>*>(tile + ch * C::kPitch + t * C::kSize);
      if (t + C::kPacket <= nt) {
        st_packet<T, C::kPacket>(dst + ch * s1 + t, r);
      } else {
#pragma unroll
        for (int j = 0; j < C::kPacket; ++j)
          if (t + j < nt) dst[ch * s1 + t + j] = r.v[j];
      }
    }
    return;
  }
#pragma unroll 4
  for (int k = 0; k < C::kChannels * kRecChunk / kRecThreads; ++k) {
    const int i = threadIdx.x + k * kRecThreads;
    const int ch = i / kRecChunk, t = i % kRecChunk;
    if (ch < nd && t < nt) dst[ch * s1 + t * s2] = *reinterpret_cast<const T*>(tile + ch * C::kPitch + t * C::kSize);
  }
}

// channel-last: one position of a lane's channels.  ptr: the lane's first channel there.
template <typename T>
__device__ __forceinline__ void store_step(T* ptr, int64_t s1, int n, bool packed, const Lane<4 / sizeof(T)>& f) {
  if constexpr (sizeof(T) == 2) {
    if (packed && n == 2) {
      float2 v[1] = {f.v};
      st_packet<T, 2>(ptr, pack2<T, 2>(v));
      return;
    }
    if (n > 0) ptr[0] = from_f32<T>(f.v.x);
    if (n > 1) ptr[s1] = from_f32<T>(f.v.y);
  } else {
    if (n > 0) ptr[0] = f.v;
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
__device__ __forceinline__ Lane<Tile<T, LAYOUT>::V> load_state(const TensorArg& s, int64_t n, int64_t nstates, int64_t d0, int64_t dim, int lane) {
  Lane<Tile<T, LAYOUT>::V> r;
#pragma unroll
  for (int i = 0; i < Tile<T, LAYOUT>::V; ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    el(r, i) = s.data && n >= 0 && n < nstates && d < dim ? static_cast<const float*>(s.data)[n * s.s0 + d * s.s1] : 0.f;
  }
  return r;
}
template <typename T, int LAYOUT>
__device__ __forceinline__ void store_state(const TensorArg& s, int64_t n, int64_t nstates, int64_t d0, int64_t dim, int lane,
                                            const Lane<Tile<T, LAYOUT>::V>& f) {
  if (!s.data || n < 0 || n >= nstates) return;
#pragma unroll
  for (int i = 0; i < Tile<T, LAYOUT>::V; ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    if (d < dim) static_cast<float*>(s.data)[n * s.s0 + d * s.s1] = el(f, i);
  }
}

// ------------------------------------------------------------------------- clusters
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
// Stores v at the place of `local` in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ void store_remote(float* local, unsigned rank, float v) {
  unsigned addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(addr) : "r"(static_cast<unsigned>(__cvta_generic_to_shared(local))), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(addr), "f"(v) : "memory");
}

}  // namespace cc1d
