// Window and prefix attention on the 16-bit matrix cores (16-bit caches, head sizes 64 and 128, block
// sizes a multiple of 16): tiles of query rows for prompts and shared prefixes, and single tokens.
//
// Both take the query heads of a kv head together, so its keys are read once for the group: a
// tile's rows are (token, head of the group) pairs, a single token's heads are the columns of
// 16-wide MFMAs.
#pragma once

#include "attention_keys.hpp"

namespace nvf {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct AttnMma;
template <>
struct AttnMma<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnMma<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

typedef __attribute__((address_space(3))) uint8_t lds_byte;

// A buffer over `bytes` bytes at p, both wave-uniform: as scalars whatever units worked them out.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const void* p, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)at), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint8_t* lds, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, off, 0, 0, 0);
}
// ds_read_b64_tr_b16 over a 16-lane group: lane i receives, as its element e, 16-bit element i % 4 of
// the 8 bytes that lane 4 e + i / 4 addresses.  With lane s at key row key0 + s / 4, dims dim0 + 4 (s % 4),
// lane i gets dim dim0 + i of keys key0 .. key0 + 3: four of the A operand's keys of V^T.
__device__ __forceinline__ s16x4 lds_tr(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}
// Four 4-key pairs of such reads, each at its address and OFF bytes on, waited for: beside loads from memory
// that stay in flight, which the compiler would wait for in front of the builtin.
template <int OFF>
__device__ __forceinline__ void lds_tr_4x2(const uint8_t* p0, const uint8_t* p1, const uint8_t* p2, const uint8_t* p3,
                                           s16x4 (&x)[4], s16x4 (&y)[4]) {
  const auto at = [](const uint8_t* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p; };
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %1, %9\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %10\n\t"
      "ds_read_b64_tr_b16 %6, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %3, %11\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
      : "v"(at(p0)), "v"(at(p1)), "v"(at(p2)), "v"(at(p3)), "i"(OFF)
      : "memory");
}
__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, __shfl_xor(v, d));
  return v;
}

// A load at a wave-uniform address of memory that the kernel does not write, as a scalar load: it waits
// for no vector load in flight.
__device__ __forceinline__ int32_t read_scalar(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

// The cache blocks of a sequence's keys, 16 rows (a slab) at a time; end: its keys' end.  The block table's
// entry of a slab is read ahead of the slab's transfers.
struct SlabEntry {
  int k0, row;  // first key, and its row in the block
  int32_t block;
};
struct SlabTable {
  const int32_t* table;  // the sequence's row of the block tables; NULL where it has none
  int bs, max_blocks, end;
  uint32_t blocks, row_b;  // cache blocks; bytes from one cache row to the next
  FastDiv div;
  template <typename T>
  __device__ __forceinline__ SlabTable(const AttnArgs<T>& a, const FastDiv& d, int seq, int keys_end)
      : table((unsigned)seq < (unsigned)a.num_seqs ? a.tables + (int64_t)seq * a.max_blocks : nullptr), bs(a.bs),
        max_blocks(a.max_blocks), end(keys_end), blocks((uint32_t)a.num_blocks),
        row_b((uint32_t)(a.kv_heads * a.hd * (int)sizeof(T))), div(d) {}
  __device__ __forceinline__ SlabEntry entry(int k0) const {
    const int b = (int)div.div((uint32_t)k0);
    SlabEntry e{k0, k0 - b * bs, -1};
    if (table && k0 < end && b < max_blocks) e.block = __builtin_amdgcn_readfirstlane(read_scalar(table + b));
    return e;
  }
  // keys, but no block
  __device__ __forceinline__ bool bad(const SlabEntry& e) const { return e.k0 < end && (uint32_t)e.block >= blocks; }
  // bytes to read: rows past the keys' end, and all where there is no block, arrive as zeros
  __device__ __forceinline__ int bytes(const SlabEntry& e) const {
    int n = 16 * (int)row_b;
    if (e.k0 + 16 > end) n = e.k0 < end ? (end - e.k0) * (int)row_b : 0;
    return (uint32_t)e.block < blocks ? n : 0;
  }
  // where they begin, from the head's first cache row (a cache has less than 2^31 rows)
  __device__ __forceinline__ uint64_t at(const SlabEntry& e) const {
    return (uint32_t)e.block < blocks ? (uint64_t)((uint32_t)e.block * (uint32_t)bs + (uint32_t)e.row) * row_b : 0;
  }
};

// ---------------------------------------------------------------------------
// A tile: 128 rows, row r = token r / G of the tile, head r % G of the kv head's group; 32 rows a
// wave.  The keys pass in chunks of 64, DMA'd to LDS (K and V double-buffered, one barrier a chunk):
//   S^T = K . Q^T     32x32x16 MFMAs, A = K rows from LDS, B = the wave's q rows in registers
//   online softmax    a row is a lane column of S^T: its max and sum are lane-local plus one
//                     exchange with the other lane half
//   O^T += V^T . P^T  A = V^T by transpose reads, B = S^T's own registers
// The next chunk's S is worked out beside this chunk's exponentials: neither waits for the other, so the
// matrix and vector units of a SIMD run at once within one wave.
// LDS rows are unpadded, their 16-byte units XOR-swizzled by row: the K reads of 8 rows and the V
// reads of 4 rows x 64 bytes fall into distinct banks.
template <int HD>
struct TileLds {
  static constexpr int kUnits = HD * 2 / 16;   // 16-byte units of a row
  static constexpr int kRows = 64 / kUnits;    // rows of one wave's transfer
  static constexpr int kRow = HD * 2;
  static constexpr int kBuf = kChunk * kRow;
  static constexpr int kBytes = 4 * kBuf;      // K, K, V, V
  static __device__ __forceinline__ int k_swz(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int v_swz(int row) { return HD == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};
constexpr float kLazyMax = 8.0f;  // exp2 units that the running max may lag behind

// One (token, head) over the seen keys of chunks [c0, c1), by one wave without the matrix cores: lane
// = key, then dims lane + 64 i.  For rows whose MFMA result is not finite: 0 * V of a masked key that
// is no number would reach them there.
template <typename T, int HD>
__device__ __forceinline__ void attend_row(const AttnArgs<T>& a, const ChunkList& list, int c0, int c1, int seq,
                                           int64_t t, int h, int kvh, int lo, int L, int sinks, int64_t split) {
  constexpr int DPL = HD / 64, N = Pack<T>::N;
  const int lane = threadIdx.x & 63;
  const int64_t row_len = (int64_t)a.kv_heads * HD;
  const T* q = a.q + t * a.q_stride + (int64_t)h * HD;
  float m = -INFINITY, l = 0.0f, acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.0f;
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    const int key = list.chunk(c) * kChunk + lane;
    const bool seen = key < L && (key >= lo || key < sinks);
    const int block = seen ? key_block(a, seq, key) : -1;
    const int64_t row = block >= 0 ? (int64_t)block * a.bs + key % a.bs : 0;
    float s = 0.0f;
    if (block >= 0) {
      const T* kp = a.kc + row * row_len + (int64_t)kvh * HD;
#pragma unroll 1
      for (int d0 = 0; d0 < HD; d0 += N) {
        float kv[N], qv[N];
        Pack<T>::unpack(ld16(kp + d0), kv);
        Pack<T>::unpack(ld16(q + d0), qv);
#pragma unroll
        for (int e = 0; e < N; ++e) s = fmaf(qv[e], kv[e], s);
      }
    } else {
      s = __builtin_nanf("");
    }
    const float x = seen ? s * a.scale_log2 : -INFINITY;
    const float m_new = fmaxf(m, wave_max(x)), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use), p = __builtin_amdgcn_exp2f(x - m_use);
    l = l * alpha + wave_sum(p);
    m = m_new;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] *= alpha;
    for (uint64_t left = __ballot(seen); left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
      const int64_t rj = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)row, j) |
                         (int64_t)__builtin_amdgcn_readlane((int)(row >> 32), j) << 32;
      const T* vp = a.vc + rj * row_len + (int64_t)kvh * HD;
#pragma unroll
      for (int i = 0; i < DPL; ++i) acc[i] = fmaf(pj, to_f32(vp[lane + 64 * i]), acc[i]);
    }
  }
  const int64_t th = t * a.q_heads + h;
  if (a.nsplit > 1) {
    const int64_t pi = th * a.nsplit + split;
#pragma unroll
    for (int i = 0; i < DPL; ++i) a.part[pi * HD + lane + 64 * i] = acc[i];
    if (lane == 0) {
      float* ml = a.part + a.tokens * a.q_heads * a.nsplit * HD + 2 * pi;
      ml[0] = m;
      ml[1] = l;
    }
  } else {
#pragma unroll
    for (int i = 0; i < DPL; ++i) a.out[th * HD + lane + 64 * i] = from_f32<T>(l == 0.0f ? 0.0f : acc[i] / l);
  }
}

// This lane, from the hardware's count, opaque to the optimizer: what follows from it is worked out
// anew where it is needed and not kept in registers through the chunks.
__device__ __forceinline__ int opaque_lane() {
  int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(lane));
  return lane;
}

// Tokens t0 + [r0, r1) of sequence seq (rows (i, head): i G + head) over the keys below cap; split
// blockIdx.z of a.nsplit, state `first + z` of the row's.
template <typename T, int HD, bool WINDOW>
__device__ __forceinline__ void attend_tile(const AttnArgs<T>& a, const FastDiv& div, const WindowRule& rule, int64_t t0,
                                            int r0, int r1, int seq, int kvh, int cap, int z, int nz, int64_t state,
                                            uint8_t* lds) {
  using M = AttnMma<T>;
  using v8 = typename M::v8;
  using Lds = TileLds<HD>;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = opaque_lane(), half = lane >> 5;
  const int G = a.q_heads / a.kv_heads;
  const int sinks = WINDOW ? rule.sinks : 0;

  // the keys that some token sees: [0, sinks) and [lo_all, L_all)
  int L_all = 0, lo_all = INT32_MAX;
  for (int i = r0 + lane; i < r1; i += 64) {
    const int n = min(key_count(a, t0 + i), cap);
    L_all = max(L_all, n);
    if (WINDOW && n > 0) lo_all = min(lo_all, rule.lo(0, n));
  }
  L_all = __builtin_amdgcn_readfirstlane(wave_max_int(L_all));
  lo_all = WINDOW ? __builtin_amdgcn_readfirstlane(-wave_max_int(-lo_all)) : 0;
  if (L_all == 0) lo_all = 0;
  const ChunkList list(lo_all, L_all, sinks);
  const int c0 = list.split_begin(z, nz), c1 = list.split_begin(z + 1, nz);

  // this lane's row
  const int row = 32 * wave + (lane & 31), ti = row / G, head = kvh * G + (row - ti * G);
  const bool ok = ti >= r0 && ti < r1;
  const int L = ok ? min(key_count(a, t0 + ti), cap) : 0;
  const int lo = WINDOW ? rule.lo(0, L) : 0;
  const bool busy = __any(ok);  // the wave has a row
  // chunks in [lo_wave, L_wave) need no mask
  const int L_wave = __builtin_amdgcn_readfirstlane(-wave_max_int(ok ? -L : -INT32_MAX));
  const int lo_wave = WINDOW ? __builtin_amdgcn_readfirstlane(wave_max_int(ok ? lo : 0)) : 0;
  v8 qf[HD / 16];
#pragma unroll
  for (int s = 0; s < HD / 16; ++s) {
    const u32x4 v = ok ? ld16(a.q + (t0 + ti) * a.q_stride + (int64_t)head * HD + 16 * s + 8 * half) : u32x4{0, 0, 0, 0};
    qf[s] = __builtin_bit_cast(v8, v);
  }

  // Transfers: wave w brings key rows 16 w .. + 15 of a chunk, transfer i rows kRows i + lane / kUnits
  // of them, a lane the unit that belongs at position lane % kUnits.
  const SlabTable table(a, div, seq, L_all);
  constexpr int kTransfers = 16 / Lds::kRows;
  const uint8_t* const k_head = reinterpret_cast<const uint8_t*>(a.kc + (int64_t)kvh * HD);
  const uint8_t* const v_head = reinterpret_cast<const uint8_t*>(a.vc + (int64_t)kvh * HD);
  const int lrow = lane / Lds::kUnits, lpos = lane % Lds::kUnits;
  const uint32_t row_off = (uint32_t)lrow * table.row_b;
  uint8_t* const slab = lds + 16 * wave * Lds::kRow;  // of buffer 0: K, K, V, V
  const auto entry_of = [&](int c) { return table.entry(list.chunk(c) * kChunk + 16 * wave); };
  const auto load_k = [&](const SlabEntry& e, int buf) {
    uint8_t* dst = slab + buf * Lds::kBuf;
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(k_head + table.at(e), table.bytes(e));
    const uint32_t k_unit = 16u * (uint32_t)(lpos ^ Lds::k_swz(lrow));
#pragma unroll
    for (int i = 0; i < kTransfers; ++i)  // (k_swz(kRows i + lrow) = k_swz(lrow) ^ 4 i)
      dma16(r, dst + Lds::kRows * i * Lds::kRow, row_off + (k_unit ^ (64u * i)) + (uint32_t)(Lds::kRows * i) * table.row_b);
    if (table.bad(e)) {  // keys without a block: NaN rows, so NaN scores where they are seen
      __builtin_amdgcn_s_waitcnt(0x0F70);  // after the transfers' zeros
      for (int i = lane; i < 16 * Lds::kUnits; i += 64) st16(dst + 16 * i, u32x4{~0u, ~0u, ~0u, ~0u});
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): before the barrier that hands the chunk over
    }
  };
  const auto load_v = [&](const SlabEntry& e, int buf) {
    uint8_t* dst = slab + (2 + buf) * Lds::kBuf;
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(v_head + table.at(e), table.bytes(e));
    const uint32_t v_off = row_off + 16u * (uint32_t)(lpos ^ Lds::v_swz(lrow));
    if (WINDOW && e.k0 < lo_all && e.k0 + 16 > sinks) {  // rows that no token sees, below the window: zeros too
#pragma unroll
      for (int i = 0; i < kTransfers; ++i) {
        const int key = e.k0 + Lds::kRows * i + lrow;
        const uint32_t off = v_off + (uint32_t)(Lds::kRows * i) * table.row_b;
        dma16(r, dst + Lds::kRows * i * Lds::kRow, key < lo_all && key >= sinks ? 0x7fffffffu : off);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kTransfers; ++i)
        dma16(r, dst + Lds::kRows * i * Lds::kRow, v_off + (uint32_t)(Lds::kRows * i) * table.row_b);
    }
  };

  // K reads: row lane % 32 of a 32-key half, unit 2 s + half at position ^ k_swz: a lane's first address
  // ^ 32 s.  V^T reads: lane l takes dims 32 d + 16 ((l >> 4) & 1) + 4 (s % 4), keys 4 half + s / 4, s = l % 16,
  // its first address ^ 64 d.
  const uint32_t k_lane = (uint32_t)((lane & 31) * Lds::kRow + 16 * (half ^ Lds::k_swz(lane & 31)));
  uint32_t v_lane;
  {
    const int s16 = lane & 15, g16 = (lane >> 4) & 1, key = 4 * half + s16 / 4;
    v_lane = (uint32_t)(key * Lds::kRow + 16 * ((2 * g16 + (s16 & 3) / 2) ^ Lds::v_swz(key)) + 8 * (s16 & 1));
  }

  f32x16 o[HD / 32];
#pragma unroll
  for (int d = 0; d < HD / 32; ++d) o[d] = f32x16{};
  float m = -INFINITY, l = 0.0f;
  const auto hand_over = [&] {  // every wave's transfers are in LDS, and its reads before are done
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  // The entries of chunks c + 1 and c + 2 (K loaded, V not), and of c + 3, read a chunk ahead.
  SlabEntry e1{}, e2{}, e3{};
  if (c0 < c1) {
    const SlabEntry e0 = entry_of(c0);
    if (c0 + 1 < c1) e1 = entry_of(c0 + 1);
    if (c0 + 2 < c1) e2 = entry_of(c0 + 2);
    load_k(e0, 0);
    load_v(e0, 0);
    if (c0 + 1 < c1) load_k(e1, 1);
  }
  hand_over();

  constexpr int kAhead = 4;  // operand reads ahead of the MFMAs
  // K's operand for key step s of 32-key half kt
  const auto k_frag = [&](const uint8_t* buf, int s, int kt) {
    return __builtin_bit_cast(v8, ld16(buf + (k_lane ^ (32u * s)) + 32 * kt * Lds::kRow));
  };
  // Chunk c, whose scores are in st; chunk c + 1's go to sn.  One barrier: before it the exponentials and
  // S(c + 1), behind it PV(c), and then the transfers that the next step's barrier waits for, K(c + 3) over
  // K(c + 1) and V(c + 1) over V(c - 1).  (In front of the transpose reads the compiler waits for every
  // transfer in flight, so none is.)
  // (Buffer `buf` holds chunk c, the other chunk c + 1.)
  const auto step = [&](int c, auto parity, f32x16* st, f32x16* sn) {
    constexpr int buf = decltype(parity)::value;
    v8 pb[2][2];
    if (c + 3 < c1) e3 = entry_of(c + 3);
    if (busy) {
      // element j of half kt is key kb + 32 kt + 8 (j / 4) + 4 half + j % 4
      const int kb = list.chunk(c) * kChunk;
      if (!(kb + kChunk <= L_wave && (!WINDOW || kb >= lo_wave || kb + kChunk <= sinks))) {
        // the first key that the row does not see, and the first of its window, from this lane's first key on
        const int k_first = kb + 4 * half, end_k = L - k_first;
        const int lo_k = WINDOW ? lo - k_first : 0, sinks_k = WINDOW ? sinks - k_first : 0;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int key = 32 * kt + 8 * (j >> 2) + (j & 3);
            st[kt][j] = key < end_k && (!WINDOW || key >= lo_k || key < sinks_k) ? st[kt][j] : -INFINITY;
          }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], st[kt][j]);
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // The running max (exp2 units; the scale is positive, so the scaled max is the max scaled) moves
      // only where a weight above 2^kLazyMax would follow; O and l share one max either way.
      const float m_cand = fmaxf(m, mx * a.scale_log2);
      if (__any(m_cand > m + kLazyMax)) {
        const float alpha = __builtin_amdgcn_exp2f(m - (m_cand == -INFINITY ? 0.0f : m_cand));
        l *= alpha;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] *= alpha;
        m = m_cand;
      }
      const float m_use = m == -INFINITY ? 0.0f : m;
      // The exponentials, and the next chunk's scores beside them (past the last chunk: of what the buffer
      // holds, unused), in slices whose order is the one written here: K reads four MFMAs ahead of their use,
      // and after each MFMA its share of the scores, one slice an fma, the next an exponential, then sum and P.
      float ls4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      sn[0] = f32x16{};
      sn[1] = f32x16{};
      const uint8_t* kn = lds + (buf ^ 1) * Lds::kBuf;
      constexpr int kSlices = HD / 8, kPer = 32 / kSlices;  // MFMAs, and scores for each
      const auto shift = [&](int x) {
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) st[e >> 4][e & 15] = fmaf(st[e >> 4][e & 15], a.scale_log2, -m_use);
      };
      const auto sum = [&](int x) {
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) {
          const float p = st[e >> 4][e & 15];
          ls4[e & 3] += p;
          pb[e >> 4][(e & 15) >> 3][e & 7] = (T)p;  // the MFMA's operand type: half a step of T, relatively
        }
      };
      v8 kf[kSlices];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) kf[x] = k_frag(kn, x >> 1, x & 1);
      shift(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < kSlices; ++x) {
        if (x + kAhead < kSlices) kf[x + kAhead] = k_frag(kn, (x + kAhead) >> 1, x & 1);
        sn[x & 1] = M::mma(kf[x], qf[x >> 1], sn[x & 1]);
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) st[e >> 4][e & 15] = __builtin_amdgcn_exp2f(st[e >> 4][e & 15]);
        if (x + 1 < kSlices) shift(x + 1);
        if (x > 0) sum(x - 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      sum(kSlices - 1);
      l += (ls4[0] + ls4[1]) + (ls4[2] + ls4[3]);  // this lane's keys; the halves meet at the end
    }
    hand_over();
    if (busy) {
      // item i: dims 32 (i % kDims), key step u = i / kDims % 2 of half kt = i / kDims / 2, keys 32 kt + 16 u + 4 half
      // + {0..3, 8..11}, as P^T's registers hold them; V reads four MFMAs ahead
      const uint8_t* vb = lds + (2 + buf) * Lds::kBuf;
      constexpr int kDims = HD / 32, kItems = 4 * kDims;
      s16x4 vx[kItems], vy[kItems];
      const auto read_v = [&](int i) {
        const uint8_t* r = vb + (v_lane ^ (64u * (i % kDims))) + 16 * (i / kDims) * Lds::kRow;
        vx[i] = lds_tr(r);
        vy[i] = lds_tr(r + 8 * Lds::kRow);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) read_v(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (i + kAhead < kItems) read_v(i + kAhead);
        o[i % kDims] = M::mma(__builtin_bit_cast(v8, __builtin_shufflevector(vx[i], vy[i], 0, 1, 2, 3, 4, 5, 6, 7)),
                              pb[i / kDims >> 1][i / kDims & 1], o[i % kDims]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (c + 3 < c1) load_k(e3, buf ^ 1);
    if (c + 1 < c1) load_v(e1, buf ^ 1);
    e1 = e2;
    e2 = e3;
  };

  f32x16 sa[2] = {f32x16{}, f32x16{}}, sb[2];
  if (c0 < c1 && busy) {
#pragma unroll
    for (int x = 0; x < HD / 8; ++x) sa[x & 1] = M::mma(k_frag(lds, x >> 1, x & 1), qf[x >> 1], sa[x & 1]);
  }
  __syncthreads();  // every wave is done with K(c0)
  if (c0 + 2 < c1) load_k(e2, 0);
#pragma unroll 1
  for (int c = c0; c < c1; c += 2) {
    step(c, std::integral_constant<int, 0>{}, sa, sb);
    if (c + 1 < c1) step(c + 1, std::integral_constant<int, 1>{}, sb, sa);
  }

  if (!busy) return;
  const int lane_e = opaque_lane(), half_e = lane_e >> 5, row_e = 32 * wave + (lane_e & 31);
  const int ti_e = row_e / G, head_e = kvh * G + (row_e - ti_e * G);
  const bool ok_e = ti_e >= r0 && ti_e < r1;
  l += __shfl_xor(l, 32);
  float finite = l * 0.0f;  // NaN where O or l holds a value that is not finite
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) finite = fmaf(o[d][j], 0.0f, finite);
  finite += __shfl_xor(finite, 32);
  const bool again = ok_e && !(finite == 0.0f);
  if (ok_e && !again) {
    // O^T: lane column = row, dims 32 d + 8 (j / 4) + 4 half + j % 4
    const int64_t th = (t0 + ti_e) * a.q_heads + head_e;
    if (a.nsplit > 1) {
      const int64_t pi = th * a.nsplit + state;
      float* po = a.part + pi * HD;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          st16(po + 32 * d + 8 * g + 4 * half_e,
               __builtin_bit_cast(u32x4, f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]}));
      if (half_e == 0) {
        float* ml = a.part + a.tokens * a.q_heads * a.nsplit * HD + 2 * pi;
        ml[0] = m;
        ml[1] = l;
      }
    } else {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      T* po = a.out + th * HD;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          typedef T t4 __attribute__((ext_vector_type(4)));
          t4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (T)(o[d][4 * g + e] * inv);
          *reinterpret_cast<t4*>(po + 32 * d + 8 * g + 4 * half_e) = v;
        }
    }
  }
  for (uint64_t left = __ballot(again) & 0xffffffffu; left; left &= left - 1) {
    const int r = 32 * wave + __builtin_ctzll(left), i = r / G, n = min(key_count(a, t0 + i), cap);
    attend_row<T, HD>(a, list, c0, c1, seq, t0 + i, kvh * G + (r - i * G), kvh, WINDOW ? rule.lo(0, n) : 0, n, sinks,
                      state);
  }
}

// A tile's runs: maximal stretches of consecutive tokens of one sequence.
constexpr int kTileRows = 128;
constexpr int kTileMaxRuns = 4;
struct TileRuns {  // bit i: the tile's token i starts a run (token 0's bit is clear)
  uint64_t lo, hi;
  __device__ __forceinline__ TileRuns(const int32_t* __restrict__ qseq, int64_t t0, int n) {
    const int lane = threadIdx.x & 63, last = n - 1;
    const int32_t x = qseq[t0 + min(lane, last)], y = qseq[t0 + min(lane + 64, last)];  // past the end: no start
    const int32_t px = __shfl_up(x, 1), py = __shfl_up(y, 1), x63 = __builtin_amdgcn_readlane(x, 63);
    lo = __ballot(lane > 0 && x != px);
    hi = __ballot(y != (lane > 0 ? py : x63));
  }
  __device__ __forceinline__ int count() const { return 1 + __popcll(lo) + __popcll(hi); }
  // the first run start after token r, or the tile's end
  __device__ __forceinline__ int end_after(int r, int end) const {
    const uint64_t x = r < 63 ? lo >> (r + 1) << (r + 1) : 0;
    const uint64_t y = r < 64 ? hi : r < 127 ? hi >> (r - 63) << (r - 63) : 0;
    return x ? __builtin_ctzll(x) : y ? 64 + __builtin_ctzll(y) : end;
  }
};

// ---------------------------------------------------------------------------
// One token: a workgroup is (token, kv head, 16 of its heads), its 4 waves take the keys 32 at a time
// in turn, each on its own (no barrier before the end):
//   S^T = K . Q^T     16x16x32 MFMAs, A = K straight from the cache (16 keys x 64 bytes a load)
//   O^T += V^T . P^T  A = V^T by transpose reads of the wave's LDS rows, written by DMA; B = S^T's registers
// K's registers and one of two V buffers hold the keys in flight: 16 KiB a wave at head size 128, eight
// waves a CU.  Every head of a token sees the same keys, so masked values are zeros and no NaN passes.
template <int HD>
struct TokenLds {
  static constexpr int kUnits = HD * 2 / 16, kRows = 64 / kUnits, kRow = HD * 2;
  static constexpr int kBuf = 32 * kRow;
  static constexpr int kWave = 2 * kBuf > (HD * 16 + 32) * 4 ? 2 * kBuf : (HD * 16 + 32) * 4;  // V, V; then the merge
  static constexpr int kBytes = 4 * kWave;
  // units of 4 keys x 2 rows' halves: the transpose reads of 8 rows x 32 bytes fall into distinct banks
  static __device__ __forceinline__ int v_swz(int row) { return HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }
};

template <typename T, int HD, typename Rule>
__device__ __forceinline__ void attend_token(const AttnArgs<T>& a, const FastDiv& div, const Rule& rule, int64_t t,
                                             int kvh, int part, int z, int nz, int64_t state, uint8_t* lds) {
  using M = AttnMma<T>;
  using v8 = typename M::v8;
  using Lds = TokenLds<HD>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int col = lane & 15, g = lane >> 4;
  const int G = a.q_heads / a.kv_heads, h0 = kvh * G + 16 * part, heads = min(16, (kvh + 1) * G - h0);
  const uint32_t row_b = (uint32_t)(a.kv_heads * HD * (int)sizeof(T));
  const int L = __builtin_amdgcn_readfirstlane(key_count(a, t)), lo = __builtin_amdgcn_readfirstlane(rule.lo(t, L));
  const int seq = __builtin_amdgcn_readfirstlane(a.qseq[t]), sinks = rule.sinks;
  uint8_t* vt = lds + wave * Lds::kWave;

  v8 qf[HD / 32];
#pragma unroll
  for (int s = 0; s < HD / 32; ++s) {
    const u32x4 v = col < heads ? ld16(a.q + t * a.q_stride + (int64_t)(h0 + col) * HD + 32 * s + 8 * g) : u32x4{0, 0, 0, 0};
    qf[s] = __builtin_bit_cast(v8, v);
  }
  f32x4 o[HD / 16];
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  const ChunkList list(lo, L, sinks);
  const int u0 = 2 * list.split_begin(z, nz) + wave, u1 = 2 * list.split_begin(z + 1, nz);  // 32-key halves of chunks
  const auto base = [&](int u) { return list.chunk(u >> 1) * kChunk + 32 * (u & 1); };
  const int lrow = lane / Lds::kUnits, lpos = lane % Lds::kUnits;
  const uint32_t k_off = (uint32_t)col * row_b + 16u * g;
  constexpr int kTransfers = 16 / Lds::kRows;  // a slab
  u32x4 kr[2][HD / 32];
  const SlabTable table(a, div, seq, L);
  const uint8_t* const k_head = reinterpret_cast<const uint8_t*>(a.kc + (int64_t)kvh * HD);
  const uint8_t* const v_head = reinterpret_cast<const uint8_t*>(a.vc + (int64_t)kvh * HD);
  SlabEntry entry[2];  // of the next keys to load, read ahead
  const auto read_entries = [&](int u) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) entry[kt] = table.entry(base(u) + 16 * kt);
  };
  const auto load = [&](uint8_t* dst) {
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const SlabEntry& e = entry[kt];
      const uint64_t at = table.at(e);
      const int bytes = table.bytes(e);
      const __amdgpu_buffer_rsrc_t rk = rows_rsrc(k_head + at, bytes), rv = rows_rsrc(v_head + at, bytes);
#pragma unroll
      for (int s4 = 0; s4 < HD / 32; ++s4)
        kr[kt][s4] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + 64u * s4, 0, 0));
      if (table.bad(e)) {  // keys without a block: NaN, so NaN scores where they are seen
#pragma unroll
        for (int s4 = 0; s4 < HD / 32; ++s4) kr[kt][s4] = u32x4{~0u, ~0u, ~0u, ~0u};
      }
      const bool edge = e.k0 < lo && e.k0 + 16 > sinks;
#pragma unroll
      for (int i = 0; i < kTransfers; ++i) {
        const int r = Lds::kRows * i + lrow;
        uint32_t off = (uint32_t)r * row_b + 16u * (uint32_t)(lpos ^ Lds::v_swz(r));
        if (edge) off = e.k0 + r < lo && e.k0 + r >= sinks ? 0x7fffffffu : off;
        dma16(rv, dst + (16 * kt + Lds::kRows * i) * Lds::kRow, off);
      }
    }
  };
  // V^T reads: lane l takes key rows 4 g + s / 4 (+ 16), dims 16 d + 4 (s % 4), s = l % 16: its first address ^ 32 d
  const int v_key = 4 * g + col / 4;
  const uint32_t v_lane = (uint32_t)(v_key * Lds::kRow + 16 * (((col & 3) / 2) ^ Lds::v_swz(v_key)) + 8 * (col & 1));

  if (u0 < u1) {
    read_entries(u0);
    load(vt);
    if (u0 + 4 < u1) read_entries(u0 + 4);
  }
  int b = 0;
#pragma unroll 1
  for (int u = u0; u < u1; u += 4, b ^= 1) {
    const uint8_t* vb = vt + b * Lds::kBuf;
    const int kb = base(u);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): these keys' K and V
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    f32x4 st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      st[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < HD / 32; ++s) st[kt] = M::mma(__builtin_bit_cast(v8, kr[kt][s]), qf[s], st[kt]);
    }
    if (u + 4 < u1) {
      load(vt + (b ^ 1) * Lds::kBuf);  // in flight during the rest
      if (u + 8 < u1) read_entries(u + 8);
    }
    // element j of tile kt is key kb + 16 kt + 4 g + j
    float mx = -INFINITY;
    const bool whole = kb + 32 <= L && (kb >= lo || kb + 32 <= sinks);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = st[kt][j];
        if (!whole) {
          const int key = kb + 16 * kt + 4 * g + j;
          x = key < L && (key >= lo || key < sinks) ? x : -INFINITY;
        }
        st[kt][j] = x;
        mx = fmaxf(mx, x);
      }
    // (a lane's own 8 keys against the shared max: the lanes of a head meet only where it moves)
    if (__any(fmaxf(m, mx * a.scale_log2) > m + kLazyMax)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m, mx * a.scale_log2);
      const float alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.0f : m_new));
      l *= alpha;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d] *= alpha;
      m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.0f : m;
    v8 pb;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(st[kt][j], a.scale_log2, -m_use));
        l += p;
        pb[4 * kt + j] = (T)p;
      }
#pragma unroll
    for (int d = 0; d < HD / 16; d += 4) {
      s16x4 x[4], y[4];
      lds_tr_4x2<16 * Lds::kRow>(vb + (v_lane ^ (32u * d)), vb + (v_lane ^ (32u * d + 32u)), vb + (v_lane ^ (32u * d + 64u)),
                                 vb + (v_lane ^ (32u * d + 96u)), x, y);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[d + i] = M::mma(__builtin_bit_cast(v8, __builtin_shufflevector(x[i], y[i], 0, 1, 2, 3, 4, 5, 6, 7)), pb, o[d + i]);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // The waves' states: O^T [HD][16] (lane column = head, dims 16 d + 4 g + j), m[16], l[16] in each
  // wave's own LDS; then thread (head, dims) joins the four.
  float* pw = reinterpret_cast<float*>(vt);
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) pw[(16 * d + 4 * g + j) * 16 + col] = o[d][j];
  if (g == 0) {
    pw[HD * 16 + col] = m;
    pw[HD * 16 + 16 + col] = l;
  }
  __syncthreads();
  constexpr int kDims = HD / 16;  // of a thread
  const int hc = threadIdx.x & 15, d0 = kDims * (threadIdx.x >> 4);
  const auto pwave = [&](int w) { return reinterpret_cast<const float*>(lds + w * Lds::kWave); };
  float mall = -INFINITY, den = 0.0f, ov[kDims];
#pragma unroll
  for (int w = 0; w < 4; ++w) mall = fmaxf(mall, pwave(w)[HD * 16 + hc]);
#pragma unroll
  for (int e = 0; e < kDims; ++e) ov[e] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float mw = pwave(w)[HD * 16 + hc];
    const float sc = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - mall);  // (no keys: O = l = 0, or NaN)
    den += sc * pwave(w)[HD * 16 + 16 + hc];
#pragma unroll
    for (int e = 0; e < kDims; ++e) ov[e] += sc * pwave(w)[(d0 + e) * 16 + hc];
  }
  if (hc < heads) {
    const int64_t th = t * a.q_heads + h0 + hc;
    if (a.nsplit > 1) {
      const int64_t pi = th * a.nsplit + state;
#pragma unroll
      for (int e = 0; e < kDims; e += 4)
        st16(a.part + pi * HD + d0 + e, __builtin_bit_cast(u32x4, f32x4{ov[e], ov[e + 1], ov[e + 2], ov[e + 3]}));
      if (d0 == 0) {
        float* ml = a.part + a.tokens * a.q_heads * a.nsplit * HD + 2 * pi;
        ml[0] = mall;
        ml[1] = den;
      }
    } else {
      const float inv = den == 0.0f ? 0.0f : 1.0f / den;
      typedef T tv __attribute__((ext_vector_type(kDims)));
      tv v;
#pragma unroll
      for (int e = 0; e < kDims; ++e) v[e] = (T)(ov[e] * inv);
      *reinterpret_cast<tv*>(a.out + th * HD + d0) = v;
    }
  }
}

// What both tile kinds and the single tokens need of a call.
template <typename T>
inline bool attn_mfma16(const AttnArgs<T>& a) {
  return sizeof(T) == 2 && (a.hd == 64 || a.hd == 128) && a.bs % 16 == 0 && aligned16(a.q) && aligned16(a.out) &&
         aligned16(a.kc) && aligned16(a.vc) && a.q_stride % 8 == 0 && a.scale_log2 > 0.0f &&
         (int64_t)a.kv_heads * a.hd * 32 < INT32_MAX && a.num_blocks <= INT32_MAX / a.bs;
}

}  // namespace nvf
