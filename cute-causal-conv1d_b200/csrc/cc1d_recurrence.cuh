// What the tiled recurrence kernels share: pairs of channels, the shared-memory tiles with
// their loads and stores, sequence boundaries and the exchange within a cluster.
//
// A CTA owns a tile of 128 bytes of channels of one batch row and walks the sequence in
// chunks of 32 positions; warp w has the 8 positions 8w .. 8w+7 of each chunk and its lanes
// the tile's channels.  So every boundary between sequences is uniform over a warp, in both
// memory layouts.
#pragma once

#include <cuda.h>

#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {

struct RecMaps {
  CUtensorMap gate, x, z, out, dout, dx, dgate, dz;
};

constexpr int kRecWarps = 4;
constexpr int kRecThreads = 32 * kRecWarps;
constexpr int kRecSteps = kRecChunk / kRecWarps;  // positions of a warp in a chunk
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
template <int V> struct alignas(8 * V) Map { Lane<V> A, H; };

template <int V, bool SEQ>
__device__ __forceinline__ Lane<V> apply(const Map<V>& m, const Lane<V>& h) {
  Lane<V> r = fma(m.A, h, m.H);
  if constexpr (SEQ) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (__float_as_int(el(m.A, i)) < 0) el(r, i) = el(m.H, i);
  }
  return r;
}

// -------------------------------------------------------------------------- barriers
__device__ __forceinline__ unsigned shared_addr(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// Arrives when all cp.async that this thread has issued are done.
__device__ __forceinline__ void mbar_arrive_copies(unsigned bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(bar) : "memory");
}
// Waits for the phase of that parity, about two seconds at most (the clock is looked at every
// 65536 tries); returns whether it came.  What is waited for was issued by this CTA or by CTAs
// of its cluster, which run at the same time, so it does come.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity) {
  uint64_t begin = 0;
  for (unsigned i = 1;; ++i) {
    unsigned done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((i & 0xffffu) == 0) {
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(now));
      if (begin == 0) begin = now;
      else if (now - begin > 2000000000ull) return false;
    }
  }
}

// ----------------------------------------------------------------------------- the tiles
// channel-last: 32 strips (positions) of 128 bytes of channels.
// rows: strips of 32 positions, one per channel, in 16-byte packets that are swapped around as
// the TMA's swizzles do, so that 8 lanes reading the same packet of 8 channels use all banks.
//
// SKEW (4: kWords, 2: kHalves, with 1 added: kOwn): the aligned 16-byte packets that cover a
// strip, in order; the strip starts as many bytes into them as it lies off a 16-byte boundary in
// memory.  Results are put there without that offset.
template <typename T, int LAYOUT, int SKEW> struct Tile {
  static constexpr int kSize = sizeof(T);
  static constexpr int V = 4 / kSize;                // channels per lane
  static constexpr int kChannels = 32 * V;           // 128 bytes
  static constexpr int kPacket = 16 / kSize;         // elements per 16 bytes
  static constexpr bool kRows = LAYOUT == kLayoutRows;
  static constexpr int kStrips = kRows ? kChannels : kRecChunk;
  static constexpr int kStripBytes = kRows ? kRecChunk * kSize : 128;
  static constexpr int kPitch = kStripBytes + (SKEW ? 16 : 0);
  static constexpr int kBytes = kStrips * kPitch;
  static_assert(kStrips * kStripBytes == 4096 && (!kRows || kStripBytes == 64 || kStripBytes == 128), "");
  // byte of element (channel, position), for SKEW of a result
  static __device__ __forceinline__ int at(int ch, int pos) {
    const int r = kRows ? ch : pos, byte = (kRows ? pos : ch) * kSize;
    const int swap = !kRows || SKEW ? 0 : kStripBytes == 128 ? r & 7 : (r >> 1) & 3;
    return r * kPitch + (((byte >> 4) ^ swap) << 4) + (byte & 15);
  }
};

// Channel of value i of a lane within the tile: neighbours share a 4-byte word of a
// channel-last row; with rows they are two rows half a tile apart.
template <typename T, int LAYOUT>
__device__ __forceinline__ int lane_channel(int lane, int i) {
  return LAYOUT == kLayoutRows ? lane + 32 * i : lane * static_cast<int>(4 / sizeof(T)) + i;
}

// One of the (batch, dim, seqlen) tensors as a CTA sees it: its tile of channels in its batch
// row.  Nothing before `origin`, its first element, is read.
template <typename T>
struct Strip {
  T* origin;
  T* row;  // at channel d0, position 0
  int64_t s1, s2;
  const CUtensorMap* map;
};
template <typename T>
__device__ __forceinline__ Strip<T> strip_of(const TensorArg& t, const CUtensorMap& map, int64_t b, int64_t d0) {
  T* const o = static_cast<T*>(t.data);
  return {o, o + b * t.s0 + d0 * t.s1, t.s1, t.s2, &map};
}

__device__ __forceinline__ void cp4(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// kTma, one thread: the copy of a chunk into its tile, counted on `bar`; and back.
template <int LAYOUT>
__device__ __forceinline__ void tma_load(unsigned tile, const CUtensorMap* map, int d0, int t0, int b, unsigned bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(tile),
               "l"(map), "r"(LAYOUT == kLayoutRows ? t0 : d0), "r"(LAYOUT == kLayoutRows ? d0 : t0), "r"(b), "r"(bar) : "memory");
}
template <int LAYOUT>
__device__ __forceinline__ void tma_store(unsigned tile, const CUtensorMap* map, int d0, int t0, int b) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(map),
               "r"(LAYOUT == kLayoutRows ? t0 : d0), "r"(LAYOUT == kLayoutRows ? d0 : t0), "r"(b), "r"(tile) : "memory");
}
__device__ __forceinline__ void tma_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
// At most N committed groups still read shared memory.
template <int N> __device__ __forceinline__ void tma_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;\n" ::"n"(N) : "memory"); }
// What this thread wrote to shared memory is there for the TMA.
__device__ __forceinline__ void tma_fence() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Strips off 16 bytes: the packets that a thread copies of each chunk, every second (rows) or
// fourth of one strip.
template <typename T, int LAYOUT>
struct Cover {
  using C = Tile<T, LAYOUT, 4>;
  static constexpr int N = kRecThreads / C::kStrips;         // threads of a strip
  static constexpr int K = (C::kPitch / 16 + N - 1) / N;     // packets of a thread
  int r, c;     // the strip, and the first packet's bytes in it
  int off;      // bytes that the strip starts into its first packet
  int64_t rel;  // from the chunk's first element to the first packet
  __device__ __forceinline__ explicit Cover(const Strip<T>& t) : r(threadIdx.x / N), c(threadIdx.x % N * 16) {
    const int64_t step = (C::kRows ? t.s1 : t.s2) * C::kSize;
    off = static_cast<int>(reinterpret_cast<uintptr_t>(t.row) + r * step) & 15;
    rel = r * step - off + c;
  }
};
// All threads: starts the copy of a chunk's packets into a tile.  Places outside the chunk's nt
// positions of nd channels are zero or left as they are.  GUARD: the tensor may begin within a
// packet, and what lies before is not read.
template <typename T, int LAYOUT, bool GUARD>
__device__ __forceinline__ void load_strips(unsigned char* tile, const Strip<T>& t, const Cover<T, LAYOUT>& m, int64_t t0, int nd, int nt) {
  using C = Tile<T, LAYOUT, 4>;
  using M = Cover<T, LAYOUT>;
  const int bytes = m.r < (C::kRows ? nd : nt) ? (C::kRows ? nt : nd) * C::kSize : -16;
  const char* const first = reinterpret_cast<const char*>(t.row + (C::kRows ? t0 : t0 * t.s2));
  const char* const src = first + m.rel;
  unsigned char* const dst = tile + m.r * C::kPitch + m.c;
  const unsigned to = shared_addr(dst);
  const int left = m.off + bytes - m.c;  // up to the strip's end
  if (GUARD && bytes > 0 && m.c == 0 && src < reinterpret_cast<const char*>(t.origin)) {
    for (int e = m.off; e < min(16, left); e += C::kSize) *reinterpret_cast<T*>(dst + e) = *reinterpret_cast<const T*>(src + e);
  } else {
    const int n = max(0, min(16, left));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(src), "r"(n) : "memory");
  }
#pragma unroll
  for (int k = 1; k < M::K; ++k) {
    if ((k + 1) * M::N * 16 > C::kPitch && m.c + k * M::N * 16 >= C::kPitch) break;
    const int n = max(0, min(16, left - k * M::N * 16));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + k * M::N * 16), "l"(src + k * M::N * 16), "r"(n) : "memory");
  }
}

// kElements, all threads: positions t0 .. t0 + nt - 1 of nd channels; places outside are zero.
template <typename T, int LAYOUT>
__device__ __forceinline__ void load_tile(unsigned char* tile, const Strip<T>& t, int64_t t0, int nd, int nt) {
  using C = Tile<T, LAYOUT, 0>;
  const unsigned base = shared_addr(tile);
  const T* const src = t.row + t0 * t.s2;
  constexpr int N = C::kChannels * kRecChunk / kRecThreads;
#pragma unroll 4
  for (int k = 0; k < N; ++k) {
    const int i = threadIdx.x + k * kRecThreads;
    const int ch = C::kRows ? i / kRecChunk : i % C::kChannels, p = C::kRows ? i % kRecChunk : i / C::kChannels;
    const bool in = ch < nd && p < nt;
    const T* from = in ? src + ch * t.s1 + p * t.s2 : t.origin;
    if constexpr (C::kSize == 4) {
      cp4(base + C::at(ch, p), from, in ? 4 : 0);
    } else {
      *reinterpret_cast<T*>(tile + C::at(ch, p)) = in ? *from : from_f32<T>(0.f);
    }
  }
}

// Strips off 16 bytes: bytes that strip i of a chunk starts off a 16-byte boundary.  Chunks and warps are
// 32 and 8 positions apart, multiples of 16 bytes in either layout, so neither matters.
template <typename T, int LAYOUT>
__device__ __forceinline__ unsigned offset_of(const Strip<T>& t, int i) {
  const unsigned step = static_cast<unsigned>(LAYOUT == kLayoutRows ? t.s1 : t.s2) * static_cast<unsigned>(sizeof(T));
  return (static_cast<unsigned>(reinterpret_cast<uintptr_t>(t.row)) + static_cast<unsigned>(i) * step) & 15u;
}

// The 8 positions of warp w and the lane's V channels, as fp32.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void read_steps(const unsigned char* tile, const Strip<T>& t, int w, int lane, Lane<4 / sizeof(T)> (&f)[kRecSteps]) {
  using C = Tile<T, LAYOUT, SKEW>;
  if constexpr (C::kRows) {
#pragma unroll
    for (int i = 0; i < C::V; ++i) {
      const int ch = lane + 32 * i;
      uint4 packets[kRecSteps / C::kPacket];
      if constexpr (SKEW) {
        // From the packets that cover them; single words would be four to a bank.
        constexpr int N = kRecSteps * C::kSize / 4;
        const unsigned off = offset_of<T, LAYOUT>(t, ch);
        const uint4* p = reinterpret_cast<const uint4*>(tile + ch * C::kPitch + w * kRecSteps * C::kSize);
        uint32_t u[N + 4];
#pragma unroll
        for (int q = 0; q <= N / 4; ++q) {
          const uint4 c = p[q];
          u[4 * q] = c.x, u[4 * q + 1] = c.y, u[4 * q + 2] = c.z, u[4 * q + 3] = c.w;
        }
#pragma unroll
        for (int j = 0; j < N + 2; ++j) u[j] = off & 8 ? u[j + 2] : u[j];
#pragma unroll
        for (int j = 0; j < N + 1; ++j) u[j] = off & 4 ? u[j + 1] : u[j];
        if constexpr ((SKEW & 6) == 2) {
#pragma unroll
          for (int j = 0; j < N; ++j) u[j] = __funnelshift_r(u[j], u[j + 1], off * 8);
        }
#pragma unroll
        for (int q = 0; q < N / 4; ++q) packets[q] = make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]);
      } else {
#pragma unroll
        for (int q = 0; q < kRecSteps / C::kPacket; ++q)
          packets[q] = *reinterpret_cast<const uint4*>(tile + C::at(ch, w * kRecSteps + q * C::kPacket));
      }
#pragma unroll
      for (int q = 0; q < kRecSteps / C::kPacket; ++q) {
        const uint4 u = packets[q];
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
      const unsigned off = SKEW ? offset_of<T, LAYOUT>(t, j) : 0;
      if constexpr (C::V == 2) {
        uint32_t u;
        if constexpr ((SKEW & 6) == 2) {
          const uint32_t* q = reinterpret_cast<const uint32_t*>(p + j * C::kPitch + (off & 12));
          u = __funnelshift_r(q[0], q[1], off * 8);
        } else {
          u = *reinterpret_cast<const uint32_t*>(p + j * C::kPitch + off);
        }
        float2 v[1];
        unpack2<T, 2>(*reinterpret_cast<const Packet<T, 2>*>(&u), v);
        f[j].v = v[0];
      } else {
        f[j].v = *reinterpret_cast<const float*>(p + j * C::kPitch + off);
      }
    }
  }
}

// Puts 8 positions into a tile, without a skew.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void write_steps(unsigned char* tile, int w, int lane, const Lane<4 / sizeof(T)> (&f)[kRecSteps]) {
  using C = Tile<T, LAYOUT, SKEW>;
  if constexpr (C::kRows) {
#pragma unroll
    for (int i = 0; i < C::V; ++i) {
#pragma unroll
      for (int q = 0; q < kRecSteps / C::kPacket; ++q) {
        float2 v[C::kPacket / 2];
#pragma unroll
        for (int j = 0; j < C::kPacket / 2; ++j)
          v[j] = make_float2(el(f[q * C::kPacket + 2 * j], i), el(f[q * C::kPacket + 2 * j + 1], i));
        *reinterpret_cast<Packet<T, C::kPacket>*>(tile + C::at(lane + 32 * i, w * kRecSteps + q * C::kPacket)) = pack2<T, C::kPacket>(v);
      }
    }
  } else {
    unsigned char* p = tile + w * kRecSteps * C::kPitch + lane * 4;
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if constexpr (C::V == 2) {
        float2 v[1] = {f[j].v};
        *reinterpret_cast<Packet<T, 2>*>(p + j * C::kPitch) = pack2<T, 2>(v);
      } else {
        *reinterpret_cast<float*>(p + j * C::kPitch) = f[j].v;
      }
    }
  }
}

// Sets the positions of `mask` among the warp's 8 to zero, in a tile as it was loaded.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void zero_steps(unsigned char* tile, const Strip<T>& t, int w, int lane, unsigned mask) {
  using C = Tile<T, LAYOUT, SKEW>;
#pragma unroll 1
  for (int j = 0; j < kRecSteps; ++j) {
    if (!(mask >> j & 1u)) continue;
    const int pos = w * kRecSteps + j;
#pragma unroll
    for (int i = 0; i < C::V; ++i) {
      const int ch = lane_channel<T, LAYOUT>(lane, i);
      int o = C::at(ch, pos);
      if constexpr (SKEW) o += offset_of<T, LAYOUT>(t, C::kRows ? ch : j);
      *reinterpret_cast<T*>(tile + o) = from_f32<T>(0.f);
    }
  }
}
// Clears them in a tile of results.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void clear_steps(unsigned char* tile, int w, int lane, unsigned mask) {
  using C = Tile<T, LAYOUT, SKEW>;
#pragma unroll 1
  for (int j = 0; j < kRecSteps; ++j) {
    if (!(mask >> j & 1u)) continue;
#pragma unroll
    for (int i = 0; i < C::V; ++i)
      *reinterpret_cast<T*>(tile + C::at(lane_channel<T, LAYOUT>(lane, i), w * kRecSteps + j)) = from_f32<T>(0.f);
  }
}

// kElements, and strips off 16 bytes with rows, all threads: stores what write_steps put into a tile.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void store_tile(const unsigned char* tile, const Strip<T>& t, int64_t t0, int nd, int nt) {
  using C = Tile<T, LAYOUT, SKEW>;
  if constexpr (SKEW) {
    // The 4-byte words of a strip as it lies in memory: 64 or 128 bytes, and one more word where
    // it starts within one.  Threads have the same word of every N-th strip, all of which start
    // alike (N strips are a multiple of 16 bytes apart).
    constexpr int W = C::kStripBytes / 4, N = kRecThreads / W, E = 4 / C::kSize;
    const int i = threadIdx.x % W, r = threadIdx.x / W;
    const int64_t step = t.s1 * C::kSize;
    char* to = reinterpret_cast<char*>(t.row + t0) + r * step + 4 * i;
    const int skew = (SKEW & 6) == 2 ? static_cast<int>(reinterpret_cast<uintptr_t>(to) >> 1) & 1 : 0, e = E * i - skew;
    to -= 2 * skew;  // the word of elements e .. e + E - 1
    if (nt == kRecChunk) {
      const unsigned char* const s = tile + r * C::kPitch + 4 * i;  // the word that holds element E i
      const unsigned char* const low = s - (e > 0 ? 4 * skew : 0);
#pragma unroll
      for (int k = 0; k < C::kStrips / N; ++k, to += N * step) {
        if (r + k * N >= nd) break;
        uint32_t u = *reinterpret_cast<const uint32_t*>(s + k * N * C::kPitch);
        if constexpr ((SKEW & 6) == 2) u = __funnelshift_rc(*reinterpret_cast<const uint32_t*>(low + k * N * C::kPitch), u, skew ? 16 : 32);
        if (e >= 0) *reinterpret_cast<uint32_t*>(to) = u;
        else *reinterpret_cast<uint16_t*>(to + 2) = static_cast<uint16_t>(u >> 16);
      }
      if constexpr ((SKEW & 6) == 2) {  // a skewed strip's last element, in the word after its 16
        constexpr int last = kRecChunk - 1;
        if (threadIdx.x < nd) {
          T* const at = t.row + t0 + threadIdx.x * t.s1 + last;
          if (!(reinterpret_cast<uintptr_t>(at) & 2)) *at = *reinterpret_cast<const T*>(tile + threadIdx.x * C::kPitch + last * C::kSize);
        }
      }
    } else {
      for (int k = r; k < nd; k += N, to += N * step) {
#pragma unroll
        for (int h = 0; h < E; ++h)
          if (e + h >= 0 && e + h < nt) reinterpret_cast<T*>(to)[h] = reinterpret_cast<const T*>(tile + k * C::kPitch)[e + h];
      }
    }
  } else {
    T* const dst = t.row + t0 * t.s2;
#pragma unroll 4
    for (int k = 0; k < C::kChannels * kRecChunk / kRecThreads; ++k) {
      const int i = threadIdx.x + k * kRecThreads;
      const int ch = C::kRows ? i / kRecChunk : i % C::kChannels, p = C::kRows ? i % kRecChunk : i / C::kChannels;
      if (ch < nd && p < nt) dst[ch * t.s1 + p * t.s2] = *reinterpret_cast<const T*>(tile + C::at(ch, p));
    }
  }
}

// Strips off 16 bytes, channel-last: stores a warp's 8 positions (from tw on, `left` of them in the
// sequence) straight from registers, as words or halves; `nch`: the lane's channels that there
// are.  `clear`: positions that get zeros.
template <typename T, int SKEW>
__device__ __forceinline__ void store_steps(const Strip<T>& t, int64_t tw, int lane, int nch, int left, unsigned clear,
                                            const Lane<4 / sizeof(T)> (&f)[kRecSteps]) {
  constexpr int V = 4 / sizeof(T);
  char* p = reinterpret_cast<char*>(t.row + tw * t.s2 + lane * V);
  const int64_t step = t.s2 * static_cast<int64_t>(sizeof(T));
  const bool whole = left >= kRecSteps && nch >= V && !clear;
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {
    uint32_t u;
    if constexpr (V == 2) {
      float2 v[1] = {f[j].v};
      const Packet<T, 2> r = pack2<T, 2>(v);
      u = *reinterpret_cast<const uint32_t*>(&r);
    } else {
      u = __float_as_uint(f[j].v);
    }
    if (clear >> j & 1u) u = 0;
    if (whole || (j < left && nch >= V)) {
      if constexpr ((SKEW & 6) == 4) {
        *reinterpret_cast<uint32_t*>(p) = u;
      } else {
        *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(u);
        *reinterpret_cast<uint16_t*>(p + 2) = static_cast<uint16_t>(u >> 16);
      }
    } else if (V == 2 && j < left && nch == 1) {
      *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(u);
    }
    p += step;
  }
}

// ---------------------------------------------------------------- sequence boundaries
// Of the 8 positions of a warp: which hold a token, which start a sequence, which end one,
// and (lane 1 + j) the id of position j.
struct Edges {
  unsigned valid, first, last;
  int id;
};
// From the ids of positions t - 1 .. t + 8, in lanes 0 .. 9 (the others hold what lane 9 does).
// Mostly one sequence covers them all, which one vote shows.
__device__ __forceinline__ Edges edges_of(int id) {
  constexpr unsigned all = 0xffffffffu;
  Edges e = {0xffu, 0u, 0u, id};
  const int before = __shfl_up_sync(all, id, 1);
  if (__all_sync(all, id == before && id >= 0)) return e;  // (lane 0 gets its own)
  const int after = __shfl_down_sync(all, id, 1), lane = threadIdx.x & 31;
  e.valid = (__ballot_sync(all, id >= 0) >> 1) & 0xffu;
  e.first = (__ballot_sync(all, lane > 0 && id >= 0 && id != before) >> 1) & 0xffu;
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
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
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
