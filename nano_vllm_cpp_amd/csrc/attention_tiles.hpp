// Window and prefix attention on the matrix cores (head sizes 64 and 128, block sizes a multiple of 16;
// 16-bit caches on the 16-bit ones, fp32 caches on the fp32 ones): tiles of query rows for prompts and
// shared prefixes, and single tokens.
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

// A softmax weight as two 16-bit MFMA operands, hi = (T)p and what that rounding left: p to 2^-16 of itself in bf16, 2^-22
// in fp16 (or half of its least subnormal), where one operand would be off by half a step of T, 2^-8 or 2^-11.
template <typename T>
__device__ __forceinline__ T rest_of(float p, T hi) {
  return (T)(p - (float)hi);
}

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

// Likewise of a prompt's rows, which lie side by side.
struct SlabRows {
  int end;
  uint32_t row_b;
  template <typename T>
  __device__ __forceinline__ SlabRows(const AttnArgs<T>& a, const FastDiv&, int, int keys_end)
      : end(keys_end), row_b((uint32_t)(a.k_stride * (int64_t)sizeof(T))) {}
  __device__ __forceinline__ SlabEntry entry(int k0) const { return SlabEntry{k0, 0, 0}; }
  __device__ __forceinline__ bool bad(const SlabEntry&) const { return false; }
  __device__ __forceinline__ int bytes(const SlabEntry& e) const {
    return e.k0 < end ? min(16, end - e.k0) * (int)row_b : 0;
  }
  __device__ __forceinline__ uint64_t at(const SlabEntry& e) const { return e.k0 < end ? (uint64_t)(uint32_t)e.k0 * row_b : 0; }
};
struct NoSlabs {
  template <typename T>
  __device__ __forceinline__ NoSlabs(const AttnArgs<T>&, const FastDiv&, int, int) {}
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
// reads of 4 rows x 64 bytes fall into distinct banks (no conflicts counted).
// Bound by the issue of matrix and vector work (32 MFMAs of 32 cycles a chunk and wave at head size 128): prompts
// of 8192, 3001 and 777 tokens, 28 / 4 heads, window 2048, fp16: 330 us, 830 TFLOP/s of the keys that are seen;
// 370 without the overlap and the operand reads ahead.
template <typename T, int HD>
struct TileLds {
  static constexpr int kUnits = HD * (int)sizeof(T) / 16;  // 16-byte units of a row
  static constexpr int kRows = 64 / kUnits;                // rows of one wave's transfer
  static constexpr int kRow = HD * (int)sizeof(T);
  static constexpr int kBuf = kChunk * kRow;
  static constexpr int kBytes = 4 * kBuf;                  // K, K, V, V
  // (of a row's bits: the swizzle of kRows i + r is that of kRows i ^ that of r)
  static __device__ __forceinline__ int k_swz(int row) { return kRow >= 256 ? row & 15 : (row >> 1) & 7; }
  static __device__ __forceinline__ int v_swz(int row) {
    return sizeof(T) == 4 ? 0 : HD == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
  }
};
constexpr float kLazyMax = 8.0f;  // exp2 units that the running max may lag behind
// fp16 weights bottom out at its least subnormal, 2^-24: those below half of it would leave P . V while the fp32 sum
// of weights still counts them (8192 keys 17.7 nats below one: 1.6e-4 of V).  So such kernels take their exponentials
// against a reference `lead` below the running max, and the largest weight is 2^lead at least and 2^(lead + lazy) at
// most, which has to stay below fp16's 2^16; states carry the reference as their max.  kLazyMax and kLead lose up to
// 2^-32 of the largest weight for a key; kFarLazy and kFarLead 2^-38, for a few more rescalings.
constexpr float kLead = 7.0f, kFarLazy = 2.0f, kFarLead = 13.0f;

// One (token, head) over the seen keys of chunks [c0, c1), by one wave without the matrix cores: lane
// = key, then dims lane + 64 i.  For rows whose MFMA result is not finite: 0 * V of a masked key that
// is no number would reach them there.
template <typename T, int HD, bool PAGED>
__device__ __forceinline__ void attend_row(const AttnArgs<T>& a, const ChunkList& list, int c0, int c1, int seq,
                                           int64_t start, int64_t t, int h, int kvh, int lo, int L, int sinks,
                                           int64_t split) {
  constexpr int DPL = HD / 64, N = Pack<T>::N;
  const int lane = threadIdx.x & 63;
  const int64_t k_len = PAGED ? (int64_t)a.kv_heads * HD : a.k_stride, v_len = PAGED ? k_len : a.v_stride;
  const T* q = a.q + t * a.q_stride + (int64_t)h * HD;
  float m = -INFINITY, l = 0.0f, acc[DPL];
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.0f;
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    const int key = list.chunk(c) * kChunk + lane;
    const bool seen = key < L && (key >= lo || key < sinks);
    const int block = !seen ? -1 : PAGED ? key_block(a, seq, key) : 0;
    const int64_t row = block < 0 ? 0 : PAGED ? (int64_t)block * a.bs + key % a.bs : start + key;
    float s = 0.0f;
    if (block >= 0) {
      const T* kp = a.kc + row * k_len + (int64_t)kvh * HD;
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
      const T* vp = a.vc + rj * v_len + (int64_t)kvh * HD;
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

// What a tile's tokens see: a shared prefix, a window, the rows of their own prompt (no pages) up to themselves, or their
// sequence's keys.
enum TileKind { kPrefixTile, kWindowTile, kPromptTile, kCausalTile };

// A tile's work: tokens t0 + [r0, r1) (rows (token, head): token G + head) over the keys below cap that the rule lets
// them see, split z of nz; `state`: where the split's softmax state goes.  A window's tokens are sequence seq's; a
// prefix's are their own sequences', whose first cap keys are the same.
struct TileJob {
  int64_t t0;
  int r0, r1, seq, kvh, cap, z, nz;
  int64_t state;
  int64_t start = 0;  // a prompt's first token
};
// What follows from it: the chunks, and this lane's row (lane column of the MFMAs).
template <typename T>
constexpr int kWaveRows = sizeof(T) == 4 ? 16 : 32;  // a wave's rows of a tile
template <typename T>
constexpr int kTileThreads = 128 / kWaveRows<T> * 64;
// (C: the type that the matrix cores take.)
template <typename T, int KIND, typename C = T>
struct TileRows {
  static constexpr bool WINDOW = KIND == kWindowTile, PREFIX = KIND == kPrefixTile;
  int L_all, lo_all, sinks;  // the keys that some token sees: [0, sinks) and [lo_all, L_all)
  int seq;                   // whose block table names them
  ChunkList list;
  int c0, c1;
  int ti, head, L, lo;       // the row's token in the tile, head and keys
  bool ok, busy;             // there is such a row; the wave has one
  int L_wave, lo_wave;       // chunks in [lo_wave, L_wave) need no mask
  uint64_t lost;             // a prefix's rows with keys but no row in the tables: the tile's keys are not theirs
  // the keys of the tile's token i
  static __device__ __forceinline__ int count(const AttnArgs<T>& a, const TileJob& job, int i) {
    if constexpr (KIND == kPromptTile) return (int)(job.t0 - job.start) + i + 1;
    else return min(key_count(a, job.t0 + i), job.cap);
  }
  __device__ __forceinline__ TileRows(const AttnArgs<T>& a, const WindowRule& rule, const TileJob& job, int lane, int wave)
      : list(0, 0, 0) {
    const int G = a.q_heads / a.kv_heads;
    sinks = WINDOW ? rule.sinks : 0;
    int most = 0, least = INT32_MAX, leads = -1, leader = -1;
    for (int i = job.r0 + lane; i < job.r1; i += 64) {
      const int n = count(a, job, i);
      most = max(most, n);
      if (WINDOW && n > 0) least = min(least, rule.lo(0, n));
      if constexpr (PREFIX) {
        const int s = a.qseq[job.t0 + i];
        const int32_t first = (unsigned)s < (unsigned)a.num_seqs ? a.tables[(int64_t)s * a.max_blocks] : -1;
        if (first >= 0 && first < a.num_blocks && n > leads) {
          leads = n;
          leader = s;
        }
      }
    }
    L_all = __builtin_amdgcn_readfirstlane(wave_max_int(most));
    seq = job.seq;
    // Not every token can stand for the others: it may be padding, its sequence may have given its pages back, it may end
    // inside the prefix.  One with the most keys of the tile, of those whose sequence has a first page, does.  (Where it
    // lacks another page, results are right by attend_rows_again, but 17 ms instead of 0.1 for 256 tokens over 8192 keys.)
    if constexpr (PREFIX) {
      const int top = wave_max_int(leads);
      seq = __builtin_amdgcn_readlane(leader, (int)__builtin_ctzll(__ballot(leads == top)));
    }
    lo_all = WINDOW ? __builtin_amdgcn_readfirstlane(-wave_max_int(-least)) : 0;
    if (L_all == 0) lo_all = 0;
    list = ChunkList(lo_all, L_all, sinks);
    c0 = list.split_begin(job.z, job.nz);
    c1 = list.split_begin(job.z + 1, job.nz);
    const int row = kWaveRows<C> * wave + (lane & (kWaveRows<C> - 1));
    ti = row / G;
    head = job.kvh * G + (row - ti * G);
    ok = ti >= job.r0 && ti < job.r1;
    L = ok ? count(a, job, ti) : 0;
    lo = WINDOW ? rule.lo(0, L) : 0;
    busy = __any(ok);
    if constexpr (PREFIX) lost = __ballot(L > 0 && (unsigned)a.qseq[job.t0 + ti] >= (unsigned)a.num_seqs);
    L_wave = __builtin_amdgcn_readfirstlane(-wave_max_int(ok ? -L : -INT32_MAX));
    lo_wave = WINDOW ? __builtin_amdgcn_readfirstlane(wave_max_int(ok ? lo : 0)) : 0;
  }
  // Scores of the chunk at key kb (element j of half kt: key kb + 32 kt + 8 (j / 4) + 4 half + j % 4): -inf
  // where the row does not see the key.
  __device__ __forceinline__ void mask(f32x16* st, int kb, int half) const {
    if (kb + kChunk <= L_wave && (!WINDOW || kb >= lo_wave || kb + kChunk <= sinks)) return;
    const int first = kb + 4 * half, end_k = L - first;  // relative to this lane's first key
    const int lo_k = WINDOW ? lo - first : 0, sinks_k = WINDOW ? sinks - first : 0;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = 32 * kt + 8 * (j >> 2) + (j & 3);
        st[kt][j] = key < end_k && (!WINDOW || key >= lo_k || key < sinks_k) ? st[kt][j] : -INFINITY;
      }
  }
  // Likewise of scores in groups of 16 keys (element j of group k: key kb + 16 k + 4 g + j).
  __device__ __forceinline__ void mask16(f32x4* st, int kb, int g) const {
    if (kb + kChunk <= L_wave && (!WINDOW || kb >= lo_wave || kb + kChunk <= sinks)) return;
    const int first = kb + 4 * g, end_k = L - first;
    const int lo_k = WINDOW ? lo - first : 0, sinks_k = WINDOW ? sinks - first : 0;
#pragma unroll
    for (int k = 0; k < kChunk / 16; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 16 * k + j;
        st[k][j] = key < end_k && (!WINDOW || key >= lo_k || key < sinks_k) ? st[k][j] : -INFINITY;
      }
  }
};

// The wave's rows of `again` (bits of the lanes 0 to kWaveRows - 1), key by key, through their own block tables.
template <typename T, int HD, int KIND>
__device__ __forceinline__ void attend_rows_again(const AttnArgs<T>& a, const WindowRule& rule, const TileJob& job,
                                                  const TileRows<T, KIND>& rows, uint64_t again, int wave) {
  const int G = a.q_heads / a.kv_heads;
  for (uint64_t left = again & ((uint64_t(1) << kWaveRows<T>) - 1); left; left &= left - 1) {
    const int r = kWaveRows<T> * wave + __builtin_ctzll(left), i = r / G, n = TileRows<T, KIND>::count(a, job, i);
    const int seq = KIND == kPrefixTile ? __builtin_amdgcn_readfirstlane(a.qseq[job.t0 + i]) : job.seq;
    attend_row<T, HD, KIND != kPromptTile>(a, rows.list, rows.c0, rows.c1, seq, job.start, job.t0 + i,
                                           job.kvh * G + (r - i * G), job.kvh, KIND == kWindowTile ? rule.lo(0, n) : 0, n,
                                           rows.sinks, job.state);
  }
}
// Every wave's transfers are in LDS, and its reads before are done.
__device__ __forceinline__ void tile_hand_over() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A tile's transfers: wave w brings key rows 16 (w % 4) .. + 15 of a chunk, transfer i rows kRows i + lane / kUnits
// of them, a lane the unit that belongs at position lane % kUnits.
template <typename T, int HD, int KIND>
struct TileLoad {
  using Compute = T;
  using Rows = TileRows<T, KIND>;
  using Lds = TileLds<T, HD>;
  static constexpr int kQParts = 1;  // operands that a row of q takes
  // P in two parts for a prefix, whose tokens are then as exact as by themselves: 256 tokens over 8192 keys, bf16, 88 us
  // in one part, 94 in two; off 64 bits by 2.4e-3 and 1.7e-3, of which rounding the outputs is 1.7e-3.  A window's prompts
  // have little but matrix and vector work: 330 us in one part, 431 in two, for 2.6e-4 and 2.0e-4 in fp16.  They round
  // P to T once, as nvf_paged_attention does.
  static constexpr bool kTwoParts = KIND == kPrefixTile;
  // (Windows and prefixes take their weights against the max itself.)
  static constexpr float kLazy = kLazyMax, kLead = KIND == kPromptTile && std::is_same_v<T, _Float16> ? nvf::kLead : 0.0f;
  static constexpr bool kEarly = false;  // loads go out behind PV: a barrier waits for transfers to LDS
  static constexpr bool WINDOW = KIND == kWindowTile, PROMPT = KIND == kPromptTile;
  static constexpr int kTransfers = 16 / Lds::kRows;
  std::conditional_t<PROMPT, SlabRows, SlabTable> table;
  std::conditional_t<PROMPT, SlabRows, NoSlabs> v_rows;  // of V, where its rows lie otherwise than K's
  const uint8_t *k_head, *v_head;
  uint8_t* slab;  // the wave's part of buffer 0: K, K, V, V
  int lane, lrow, lpos, lo_all, sinks;
  uint32_t row_off;
  __device__ __forceinline__ TileLoad(const AttnArgs<T>& a, const FastDiv& div, const TileJob& job,
                                      const Rows& rows, int ln, int wave, uint8_t* lds)
      : table(a, div, rows.seq, rows.L_all), v_rows(a, div, rows.seq, rows.L_all),
        k_head(reinterpret_cast<const uint8_t*>(a.kc + (PROMPT ? job.start * a.k_stride : 0) + (int64_t)job.kvh * HD)),
        v_head(reinterpret_cast<const uint8_t*>(a.vc + (PROMPT ? job.start * a.v_stride : 0) + (int64_t)job.kvh * HD)),
        slab(lds + 16 * (sizeof(T) == 4 ? wave & 3 : wave) * Lds::kRow),
        lane(ln), lrow(ln / Lds::kUnits), lpos(ln % Lds::kUnits), lo_all(rows.lo_all), sinks(rows.sinks),
        row_off((uint32_t)lrow * table.row_b) {
    if constexpr (PROMPT) v_rows.row_b = (uint32_t)(a.v_stride * (int64_t)sizeof(T));
  }
  __device__ __forceinline__ const auto& v_table() const {
    if constexpr (PROMPT) return v_rows;
    else return table;
  }
  // The tile's q rows as operands; what the scores are multiplied by, in exp2 units.
  template <typename V8>
  static __device__ __forceinline__ float q(const AttnArgs<T>& a, const TileJob& job, const Rows& rows, int half,
                                            V8 (&qf)[1][HD / 16]) {
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
      const u32x4 v = rows.ok ? ld16(a.q + (job.t0 + rows.ti) * a.q_stride + (int64_t)rows.head * HD + 16 * s + 8 * half)
                              : u32x4{0, 0, 0, 0};
      qf[0][s] = __builtin_bit_cast(V8, v);
    }
    return a.scale_log2;
  }
  __device__ __forceinline__ void commit() const {}  // (transfers need nothing but the wait for them)
  static __device__ __forceinline__ void hand_over() { tile_hand_over(); }
  static __device__ __forceinline__ void again(const AttnArgs<T>& a, const WindowRule& rule, const TileJob& job,
                                               const Rows& rows, uint64_t lanes, int wave) {
    attend_rows_again<T, HD, KIND>(a, rule, job, rows, lanes, wave);
  }
  __device__ __forceinline__ void k(const SlabEntry& e, int buf) const {
    uint8_t* dst = slab + buf * Lds::kBuf;
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(k_head + table.at(e), table.bytes(e));
    const uint32_t unit = 16u * (uint32_t)(lpos ^ Lds::k_swz(lrow));
#pragma unroll
    for (int i = 0; i < kTransfers; ++i)
      dma16(r, dst + Lds::kRows * i * Lds::kRow,
            row_off + (unit ^ (16u * Lds::k_swz(Lds::kRows * i))) + (uint32_t)(Lds::kRows * i) * table.row_b);
    if (table.bad(e)) {  // keys without a block: NaN rows, so NaN scores where they are seen
      __builtin_amdgcn_s_waitcnt(0x0F70);  // after the transfers' zeros
      for (int i = lane; i < 16 * Lds::kUnits; i += 64) st16(dst + 16 * i, u32x4{~0u, ~0u, ~0u, ~0u});
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): before the barrier that hands the chunk over
    }
  }
  __device__ __forceinline__ void v(const SlabEntry& e, int buf) const {
    uint8_t* dst = slab + (2 + buf) * Lds::kBuf;
    const auto& rows = v_table();
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(v_head + rows.at(e), rows.bytes(e));
    const uint32_t v_off = PROMPT ? (uint32_t)lrow * rows.row_b : row_off;
    const uint32_t off0 = v_off + 16u * (uint32_t)(lpos ^ Lds::v_swz(lrow));  // (v_swz(kRows i) is 0)
    if (WINDOW && e.k0 < lo_all && e.k0 + 16 > sinks) {  // rows that no token sees, below the window: zeros too
#pragma unroll
      for (int i = 0; i < kTransfers; ++i) {
        const int key = e.k0 + Lds::kRows * i + lrow;
        const uint32_t off = off0 + (uint32_t)(Lds::kRows * i) * rows.row_b;
        dma16(r, dst + Lds::kRows * i * Lds::kRow, key < lo_all && key >= sinks ? 0x7fffffffu : off);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kTransfers; ++i)
        dma16(r, dst + Lds::kRows * i * Lds::kRow, off0 + (uint32_t)(Lds::kRows * i) * rows.row_b);
    }
  }
};

template <typename T, int HD, int KIND, typename Load = TileLoad<T, HD, KIND>>
__device__ __forceinline__ void attend_tile(const AttnArgs<T>& a, const FastDiv& div, const WindowRule& rule,
                                            const TileJob& job, uint8_t* lds) {
  using C = typename Load::Compute;
  using M = AttnMma<C>;
  using v8 = typename M::v8;
  using Lds = TileLds<C, HD>;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = opaque_lane(), half = lane >> 5;
  const TileRows<T, KIND, C> rows(a, rule, job, lane, wave);
  const ChunkList& list = rows.list;
  const int c0 = rows.c0, c1 = rows.c1;
  const bool busy = rows.busy;
  v8 qf[Load::kQParts][HD / 16];
  const float scale = Load::q(a, job, rows, half, qf);

  Load load(a, div, job, rows, lane, wave, lds);
  const auto entry_of = [&](int c) { return load.table.entry(list.chunk(c) * kChunk + 16 * wave); };

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
  // The entries of chunks c + 1 and c + 2 (K loaded, V not), and of c + 3, read a chunk ahead.
  SlabEntry e1{}, e2{}, e3{};
  if (c0 < c1) {
    const SlabEntry e0 = entry_of(c0);
    if (c0 + 1 < c1) e1 = entry_of(c0 + 1);
    if (c0 + 2 < c1) e2 = entry_of(c0 + 2);
    load.k(e0, 0);
    load.v(e0, 0);
    load.commit();
    if (c0 + 1 < c1) load.k(e1, 1);
    load.commit();
  }
  Load::hand_over();

  constexpr int kAhead = 4;  // operand reads ahead of the MFMAs
  constexpr bool kTwoParts = Load::kTwoParts;
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
    v8 ph[4];
    if (c + 3 < c1) e3 = entry_of(c + 3);
    if (busy) {
      rows.mask(st, list.chunk(c) * kChunk, half);
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], st[kt][j]);
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      // The running max (exp2 units; the scale is positive, so the scaled max is the max scaled) moves
      // only where a weight above 2^(lead + lazy) would follow; O and l share one max either way.
      const float m_cand = fmaxf(m, Load::kLead != 0.0f ? fmaf(mx, scale, -Load::kLead) : mx * scale);
      if (__any(m_cand > m + Load::kLazy)) {
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
      const uint8_t* kn = lds + (buf ^ 1) * Lds::kBuf;
      constexpr int kSlices = HD / 8, kPer = 32 / kSlices;  // MFMAs, and scores for each
      const auto shift = [&](int x) {
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) st[e >> 4][e & 15] = fmaf(st[e >> 4][e & 15], scale, -m_use);
      };
      const auto sum = [&](int x) {
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) {
          const float p = st[e >> 4][e & 15];
          ls4[e & 3] += p;
          ph[e >> 3][e & 7] = (C)p;
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
        sn[x & 1] = M::mma(kf[x], qf[0][x >> 1], x < 2 ? f32x16{} : sn[x & 1]);
        if constexpr (Load::kQParts == 2) sn[x & 1] = M::mma(kf[x], qf[1][x >> 1], sn[x & 1]);
#pragma unroll
        for (int e = kPer * x; e < kPer * x + kPer; ++e) st[e >> 4][e & 15] = __builtin_amdgcn_exp2f(st[e >> 4][e & 15]);
        if (x + 1 < kSlices) shift(x + 1);
        if (x > 0) sum(x - 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      sum(kSlices - 1);
      l += (ls4[0] + ls4[1]) + (ls4[2] + ls4[3]);  // this lane's keys; the halves meet at the end
    }
    load.commit();
    if constexpr (Load::kEarly) {
      if (c + 3 < c1) load.k(e3, buf ^ 1);
      if (c + 1 < c1) load.v(e1, buf ^ 1);
    }
    Load::hand_over();
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
      v8 pl[4];  // worked out beside the MFMAs of the step before, two or four values an item
      constexpr int kRests = 8 / kDims;
      const auto rest = [&](int e) { pl[e >> 3][e & 7] = rest_of(st[e >> 4][e & 15], ph[e >> 3][e & 7]); };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) read_v(i);
      if constexpr (kTwoParts) {
#pragma unroll
        for (int e = 0; e < 8; ++e) rest(e);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        if (i + kAhead < kItems) read_v(i + kAhead);
        const v8 v = __builtin_bit_cast(v8, __builtin_shufflevector(vx[i], vy[i], 0, 1, 2, 3, 4, 5, 6, 7));
        o[i % kDims] = M::mma(v, ph[i / kDims], o[i % kDims]);
        if constexpr (kTwoParts) {
          o[i % kDims] = M::mma(v, pl[i / kDims], o[i % kDims]);
#pragma unroll
          for (int e = 0; e < kRests; ++e)
            if (i + kDims < kItems) rest(8 * (i / kDims + 1) + kRests * (i % kDims) + e);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (!Load::kEarly) {
      if (c + 3 < c1) load.k(e3, buf ^ 1);
      if (c + 1 < c1) load.v(e1, buf ^ 1);
    }
    e1 = e2;
    e2 = e3;
  };

  f32x16 sa[2] = {f32x16{}, f32x16{}}, sb[2];
  if (c0 < c1 && busy) {
#pragma unroll
    for (int x = 0; x < HD / 8; ++x)
#pragma unroll
      for (int p = 0; p < Load::kQParts; ++p) sa[x & 1] = M::mma(k_frag(lds, x >> 1, x & 1), qf[p][x >> 1], sa[x & 1]);
  }
  __syncthreads();  // every wave is done with K(c0)
  if (c0 + 2 < c1) load.k(e2, 0);
#pragma unroll 1
  for (int c = c0; c < c1; c += 2) {
    step(c, std::integral_constant<int, 0>{}, sa, sb);
    if (c + 1 < c1) step(c + 1, std::integral_constant<int, 1>{}, sb, sa);
  }

  if (!busy) return;
  const int lane_e = opaque_lane(), half_e = lane_e >> 5, row_e = 32 * wave + (lane_e & 31);
  const int G = a.q_heads / a.kv_heads, ti_e = row_e / G, head_e = job.kvh * G + (row_e - ti_e * G);
  const bool ok_e = ti_e >= job.r0 && ti_e < job.r1;
  l += __shfl_xor(l, 32);
  float finite = l * 0.0f;  // NaN where O or l holds a value that is not finite
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) finite = fmaf(o[d][j], 0.0f, finite);
  finite += __shfl_xor(finite, 32);
  const bool again = ok_e && (!(finite == 0.0f) || (KIND == kPrefixTile && (rows.lost >> lane_e & 1)));
  if (ok_e && !again) {
    // O^T: lane column = row, dims 32 d + 8 (j / 4) + 4 half + j % 4
    const int64_t th = (job.t0 + ti_e) * a.q_heads + head_e;
    if (a.nsplit > 1) {
      const int64_t pi = th * a.nsplit + job.state;
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
  Load::again(a, rule, job, rows, __ballot(again), wave);
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
//   O^T += V^T . P^T  A = V^T by transpose reads of the wave's LDS rows, written by DMA; B = S^T's registers, P in two
//                     parts (which costs no time: 343 to 346 us for 256 ragged sequences either way)
// K's registers and one of two V buffers hold the keys in flight: 16 KiB a wave at head size 128, eight
// waves a CU.  Every head of a token sees the same keys, so masked values are zeros and no NaN passes.
// Bound by HBM: 512 tokens of 4096 keys, 28 / 4 heads of 128, bf16, 5.9 TB/s; 256 ragged ones 5.4.
template <typename T, int HD>
struct TokenLds {
  static constexpr int kUnits = HD * 2 / 16, kRows = 64 / kUnits, kRow = HD * 2;
  static constexpr int kBuf = 32 * kRow, kState = (HD * 16 + 32) * 4;
  static constexpr int kWave = sizeof(T) == 2 && 2 * kBuf > kState ? 2 * kBuf : kState;  // V, V; then the state
  static constexpr int kBytes = 4 * kWave;
  // units of 4 keys x 2 rows' halves: the transpose reads of 8 rows x 32 bytes fall into distinct banks
  static __device__ __forceinline__ int v_swz(int row) { return HD == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }
};

// The four waves' softmax states, which each has left in its own LDS as O^T [HD][16 heads], m[16], l[16] (m =
// -inf, O = l = 0 where it had no keys): thread (head, HD / 16 dims) joins and stores them.
template <typename T, int HD>
__device__ __forceinline__ void join_waves(const AttnArgs<T>& a, const uint8_t* lds, int64_t t, int h0, int heads,
                                           int64_t state) {
  __syncthreads();
  constexpr int kDims = HD / 16;
  const int hc = threadIdx.x & 15, d0 = kDims * (threadIdx.x >> 4);
  const auto of = [&](int w) { return reinterpret_cast<const float*>(lds + w * TokenLds<T, HD>::kWave); };
  float mall = -INFINITY, den = 0.0f, ov[kDims];
#pragma unroll
  for (int w = 0; w < 4; ++w) mall = fmaxf(mall, of(w)[HD * 16 + hc]);
#pragma unroll
  for (int e = 0; e < kDims; ++e) ov[e] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float mw = of(w)[HD * 16 + hc];
    const float sc = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - mall);  // (no keys: O = l = 0, or NaN)
    den += sc * of(w)[HD * 16 + 16 + hc];
#pragma unroll
    for (int e = 0; e < kDims; ++e) ov[e] += sc * of(w)[(d0 + e) * 16 + hc];
  }
  if (hc >= heads) return;
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
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = 0; e < kDims; e += 4) {
      t4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (T)(ov[e + i] * inv);
      *reinterpret_cast<t4*>(a.out + th * HD + d0 + e) = v;
    }
  }
}

template <typename T, int HD, typename Rule>
__device__ __forceinline__ void attend_token(const AttnArgs<T>& a, const FastDiv& div, const Rule& rule, int64_t t,
                                             int kvh, int part, int z, int nz, int64_t state, uint8_t* lds) {
  using M = AttnMma<T>;
  using v8 = typename M::v8;
  using Lds = TokenLds<T, HD>;
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
  f32x4 o[HD / 16], o_lo[HD / 16];  // of P's two parts: an infinite value times the second may be any sign, or no number
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = o_lo[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
      for (int d = 0; d < HD / 16; ++d) {
        o[d] *= alpha;
        o_lo[d] *= alpha;
      }
      m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.0f : m;
    v8 ph, pl;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = __builtin_amdgcn_exp2f(fmaf(st[kt][j], a.scale_log2, -m_use));
        l += p;
        ph[4 * kt + j] = (T)p;
        pl[4 * kt + j] = rest_of(p, ph[4 * kt + j]);
      }
#pragma unroll
    for (int d = 0; d < HD / 16; d += 4) {
      s16x4 x[4], y[4];
      lds_tr_4x2<16 * Lds::kRow>(vb + (v_lane ^ (32u * d)), vb + (v_lane ^ (32u * d + 32u)), vb + (v_lane ^ (32u * d + 64u)),
                                 vb + (v_lane ^ (32u * d + 96u)), x, y);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v8 v = __builtin_bit_cast(v8, __builtin_shufflevector(x[i], y[i], 0, 1, 2, 3, 4, 5, 6, 7));
        o[d + i] = M::mma(v, ph, o[d + i]);
        o_lo[d + i] = M::mma(v, pl, o_lo[d + i]);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // (lane column = head, dims 16 d + 4 g + j)
  float* pw = reinterpret_cast<float*>(vt);
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      pw[(16 * d + 4 * g + j) * 16 + col] = __builtin_isfinite(o[d][j]) ? o[d][j] + o_lo[d][j] : o[d][j];
  if (g == 0) {
    pw[HD * 16 + col] = m;
    pw[HD * 16 + 16 + col] = l;
  }
  join_waves<T, HD>(a, lds, t, h0, heads, state);
}

// ---------------------------------------------------------------------------
// fp32 caches: v_mfma_f32_16x16x4_f32, exact products and fp32 sums.  The tiles are bound by the matrix units (256
// instructions of 32 cycles a chunk and wave at head size 128).  Two chunks of K and V take most of a CU's LDS at head
// size 128, so the workgroup has eight waves of 16 rows: two on a SIMD, one's products beside the other's softmax,
// transfers and barrier.  Four waves of 32 rows (32x32x2) kept the units busy 79% of the time: chunks of 700 and 300
// tokens after 5000, 32 / 8 heads of 128, window 2048, took 295 us, and 289 so
// (busy 84%; a large fp32 product 221).
//   S^T = K . Q^T     MFMA (i, e) contracts dim 16 i + 4 g + e (g = lane / 16): a lane's operands of four MFMAs are
//                     16 consecutive bytes of its K row and of its q
//   O^T += V^T . P^T  MFMA u of 16 keys contracts key 4 g + u, which S^T's register u of the lane holds, so P^T is
//                     those registers.  Row r of tile d is dim 64 (d / 4) + 4 r + d % 4: four tiles' operands for a
//                     key lie side by side in V's row
template <int HD, int KIND>
__device__ __forceinline__ void attend_tile_f32(const AttnArgs<float>& a, const FastDiv& div, const WindowRule& rule,
                                                const TileJob& job, uint8_t* lds) {
  using Lds = TileLds<float, HD>;
  constexpr int kGroups = kChunk / 16, kV = HD / 64;  // key groups; 16-byte reads of a V row
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = opaque_lane(), col = lane & 15, g = lane >> 4;
  const TileRows<float, KIND> rows(a, rule, job, lane, wave);
  const int c0 = rows.c0, c1 = rows.c1;
  f32x4 qf[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i)
    qf[i] = rows.ok ? __builtin_bit_cast(f32x4, ld16(a.q + (job.t0 + rows.ti) * a.q_stride + (int64_t)rows.head * HD +
                                                     16 * i + 4 * g))
                    : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const TileLoad<float, HD, KIND> load(a, div, job, rows, lane, wave, lds);
  const auto entry_of = [&](int c) { return load.table.entry(rows.list.chunk(c) * kChunk + 16 * (wave & 3)); };
  const auto fetch = [&](const SlabEntry& e, int buf) {  // waves 0 to 3 bring K, the others V
    if (wave < 4) load.k(e, buf);
    else load.v(e, buf);
  };
  // K reads: row lane % 16 of a group, unit 4 i + g at position ^ k_swz, a lane's first address ^ 64 i; V reads: key
  // 4 g + u of a group, unit lane % 16
  const uint32_t k_lane = (uint32_t)(col * Lds::kRow + 16 * (g ^ Lds::k_swz(col)));
  const uint32_t v_lane = (uint32_t)(4 * g * Lds::kRow + 16 * col);

  f32x4 o[HD / 16];
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  SlabEntry next{};
  if (c0 < c1) {
    const SlabEntry e = entry_of(c0);
    if (c0 + 1 < c1) next = entry_of(c0 + 1);
    fetch(e, 0);
  }
  tile_hand_over();
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    const int buf = (c - c0) & 1;
    if (c + 1 < c1) {
      fetch(next, buf ^ 1);
      if (c + 2 < c1) next = entry_of(c + 2);
    }
    if (rows.busy) {
      f32x4 st[kGroups];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) st[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      const uint8_t* kb = lds + buf * Lds::kBuf;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        f32x4 x[kGroups];
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
          x[k] = __builtin_bit_cast(f32x4, ld16(kb + (k_lane ^ (64u * i)) + 16 * k * Lds::kRow));
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < kGroups; ++k) st[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[k][e], qf[i][e], st[k], 0, 0, 0);
      }
      rows.mask16(st, rows.list.chunk(c) * kChunk, g);
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) mx = fmaxf(mx, fmaxf(fmaxf(st[k][0], st[k][1]), fmaxf(st[k][2], st[k][3])));
      if (__any(fmaxf(m, mx * a.scale_log2) > m + kLazyMax)) {  // as in attend_token
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
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          st[k][u] = __builtin_amdgcn_exp2f(fmaf(st[k][u], a.scale_log2, -m_use));
          l += st[k][u];
        }
      const uint8_t* vb = lds + (2 + buf) * Lds::kBuf + v_lane;
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            const f32x4 x = __builtin_bit_cast(f32x4, ld16(vb + (16 * k + u) * Lds::kRow + 256 * i));
#pragma unroll
            for (int d = 0; d < 4; ++d)
              o[4 * i + d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[d], st[k][u], o[4 * i + d], 0, 0, 0);
          }
    }
    tile_hand_over();
  }

  if (!rows.busy) return;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  float finite = l * 0.0f;  // as in attend_tile
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) finite = fmaf(o[d][j], 0.0f, finite);
  finite += __shfl_xor(finite, 16);
  finite += __shfl_xor(finite, 32);
  const bool again = rows.ok && (!(finite == 0.0f) || (KIND == kPrefixTile && (rows.lost >> lane & 1)));
  if (rows.ok && !again) {
    const int64_t th = (job.t0 + rows.ti) * a.q_heads + rows.head, pi = th * a.nsplit + job.state;
    const float inv = a.nsplit > 1 ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
    float* po = a.nsplit > 1 ? a.part + pi * HD : a.out + th * HD;
#pragma unroll
    for (int i = 0; i < kV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st16(po + 64 * i + 16 * g + 4 * j,
             __builtin_bit_cast(u32x4, f32x4{o[4 * i][j] * inv, o[4 * i + 1][j] * inv, o[4 * i + 2][j] * inv,
                                             o[4 * i + 3][j] * inv}));
    if (a.nsplit > 1 && g == 0) {
      float* ml = a.part + a.tokens * a.q_heads * a.nsplit * HD + 2 * pi;
      ml[0] = m;
      ml[1] = l;
    }
  }
  attend_rows_again<float, HD, KIND>(a, rule, job, rows, __ballot(again), wave);
}

// One token over an fp32 cache, as attend_token: a wave takes 16 keys (a slab) at a time straight into
// registers, the next slab's loads in flight.
//   S^T   MFMA (i, e) contracts dim 16 i + 4 g + e (g = lane / 16): 64 bytes of each of 16 K rows a load
//   O^T   MFMA u contracts key 4 g + u, S^T's register u; row r of tile d is dim 64 (d / 4) + 4 r + d % 4
template <int HD, typename Rule>
__device__ __forceinline__ void attend_token_f32(const AttnArgs<float>& a, const FastDiv& div, const Rule& rule, int64_t t,
                                                 int kvh, int part, int z, int nz, int64_t state, uint8_t* lds) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int col = lane & 15, g = lane >> 4;
  const int G = a.q_heads / a.kv_heads, h0 = kvh * G + 16 * part, heads = min(16, (kvh + 1) * G - h0);
  const int L = __builtin_amdgcn_readfirstlane(key_count(a, t)), lo = __builtin_amdgcn_readfirstlane(rule.lo(t, L));
  const int seq = __builtin_amdgcn_readfirstlane(a.qseq[t]), sinks = rule.sinks;
  f32x4 qf[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i)
    qf[i] = col < heads ? __builtin_bit_cast(f32x4, ld16(a.q + t * a.q_stride + (int64_t)(h0 + col) * HD + 16 * i + 4 * g))
                        : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 o[HD / 16];
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  const ChunkList list(lo, L, sinks);
  const int u0 = 4 * list.split_begin(z, nz) + wave, u1 = 4 * list.split_begin(z + 1, nz);  // slabs of chunks
  const SlabTable table(a, div, seq, L);
  const auto entry_of = [&](int u) { return table.entry(list.chunk(u >> 2) * kChunk + 16 * (u & 3)); };
  const uint8_t* const k_head = reinterpret_cast<const uint8_t*>(a.kc + (int64_t)kvh * HD);
  const uint8_t* const v_head = reinterpret_cast<const uint8_t*>(a.vc + (int64_t)kvh * HD);
  constexpr int kV = HD / 64;  // 16-byte loads of a V row
  struct Keys {
    u32x4 k[HD / 16], v[4 * kV];
    int kb;
  };
  const auto load = [&](const SlabEntry& e, Keys& x) {
    const uint64_t at = table.at(e);
    const int bytes = table.bytes(e);
    const __amdgpu_buffer_rsrc_t rk = rows_rsrc(k_head + at, bytes), rv = rows_rsrc(v_head + at, bytes);
    x.kb = e.k0;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
      x.k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, (uint32_t)col * table.row_b + 64u * i + 16u * g, 0, 0));
    if (table.bad(e)) {  // keys without a block: NaN, so NaN scores where they are seen
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) x.k[i] = u32x4{~0u, ~0u, ~0u, ~0u};
    }
    const bool edge = e.k0 < lo && e.k0 + 16 > sinks;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = 4 * g + u;
      uint32_t off = (uint32_t)r * table.row_b + 16u * col;
      if (edge) off = e.k0 + r < lo && e.k0 + r >= sinks ? 0x7fffff00u : off;
#pragma unroll
      for (int i = 0; i < kV; ++i)
        x.v[kV * u + i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, off + 256u * i, 0, 0));
    }
  };
  const auto add = [&](const Keys& x) {
    f32x4 st = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
      const f32x4 k = __builtin_bit_cast(f32x4, x.k[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) st = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], qf[i][e], st, 0, 0, 0);
    }
    float mx = -INFINITY;
    const bool whole = x.kb + 16 <= L && (x.kb >= lo || x.kb + 16 <= sinks);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!whole) {
        const int key = x.kb + 4 * g + j;
        st[j] = key < L && (key >= lo || key < sinks) ? st[j] : -INFINITY;
      }
      mx = fmaxf(mx, st[j]);
    }
    if (__any(fmaxf(m, mx * a.scale_log2) > m + kLazyMax)) {  // as in attend_token
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
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      st[j] = __builtin_amdgcn_exp2f(fmaf(st[j], a.scale_log2, -m_use));
      l += st[j];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const f32x4 v = __builtin_bit_cast(f32x4, x.v[kV * u + i]);
#pragma unroll
        for (int d = 0; d < 4; ++d) o[4 * i + d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[d], st[u], o[4 * i + d], 0, 0, 0);
      }
  };
  // two slabs a trip, the register sets trading places; the block-table entries another one ahead
  Keys x, y;
  SlabEntry e{};
  if (u0 < u1) {
    load(entry_of(u0), x);
    if (u0 + 4 < u1) e = entry_of(u0 + 4);
  }
#pragma unroll 1
  for (int u = u0; u < u1; u += 8) {
    if (u + 4 < u1) {
      load(e, y);
      if (u + 8 < u1) e = entry_of(u + 8);
    }
    add(x);
    if (u + 4 >= u1) break;
    if (u + 8 < u1) {
      load(e, x);
      if (u + 12 < u1) e = entry_of(u + 12);
    }
    add(y);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  float* pw = reinterpret_cast<float*>(lds + wave * TokenLds<float, HD>::kWave);
#pragma unroll
  for (int d = 0; d < HD / 16; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) pw[(64 * (d >> 2) + 4 * (4 * g + j) + (d & 3)) * 16 + col] = o[d][j];
  if (g == 0) {
    pw[HD * 16 + col] = m;
    pw[HD * 16 + 16 + col] = l;
  }
  join_waves<float, HD>(a, lds, t, h0, heads, state);
}

// The two of a type.
template <typename T, int HD, int KIND>
__device__ __forceinline__ void tile_of(const AttnArgs<T>& a, const FastDiv& div, const WindowRule& rule,
                                        const TileJob& job, uint8_t* lds) {
  if constexpr (sizeof(T) == 4) attend_tile_f32<HD, KIND>(a, div, rule, job, lds);
  else attend_tile<T, HD, KIND>(a, div, rule, job, lds);
}
template <typename T, int HD, typename Rule>
__device__ __forceinline__ void token_of(const AttnArgs<T>& a, const FastDiv& div, const Rule& rule, int64_t t, int kvh,
                                         int part, int z, int nz, int64_t state, uint8_t* lds) {
  if constexpr (sizeof(T) == 4) attend_token_f32<HD, Rule>(a, div, rule, t, kvh, part, z, nz, state, lds);
  else attend_token<T, HD, Rule>(a, div, rule, t, kvh, part, z, nz, state, lds);
}

// Groups of consecutive tokens (a window's sequences, a prefix's groups) as tiles of tile_tokens tokens each:
// tile x is tokens t0 + [0, n) of group g.
struct TileAt {
  int g, n;
  int64_t t0;
};
__device__ __forceinline__ TileAt tile_at(const int* start, int groups, int x, int tile_tokens) {
  int g = 0;
  for (; g < groups; ++g) {  // uniform: scalar loads of the kernel's arguments
    const int tiles = (start[g + 1] - start[g] + tile_tokens - 1) / tile_tokens;
    if (x < tiles) break;
    x -= tiles;
  }
  const int64_t t0 = start[g] + (int64_t)x * tile_tokens;
  return TileAt{g, min(tile_tokens, (int)(start[g + 1] - t0)), t0};
}
inline int tiles_of(const int* start, int groups, int tile_tokens) {
  int n = 0;
  for (int g = 0; g < groups; ++g) n += (start[g + 1] - start[g] + tile_tokens - 1) / tile_tokens;
  return n;
}

// What `n` key ranges cost beside their keys, in us: the partial states' way to memory and back, and the launch that
// joins them, which a call that has to join anyway (`joined`: a prefix's) does not count.
inline double split_us(int n, int64_t rows, int hd, bool joined) {
  return n > 1 || joined ? (joined ? 0.0 : 4.0) + (double)rows * n * (hd + 2) * 8 / 5e6 : 0.0;
}
// The number of key ranges that `wgs` workgroups of tiles, of up to `chunks` chunks each, are best cut into on
// `part` of the GPU: the rounds of workgroups that it takes at once, times a range's chunks and its start and end,
// and split_us.  Times in us, measured at head size 128, by which 64 goes too: a chunk takes 1.9 with two workgroups a CU
// and 1.1 alone (16 bits; a prefix's, with its weights in two parts, 1.3 times as long; start and end take as long as
// two), 8 on the fp32 matrix units (4 alone at head size 64; start and end half of it), where a workgroup of head size
// 128 fills a CU.
inline int tile_split(int64_t wgs, int64_t chunks, int64_t rows, int hd, int dtype_bytes, double part = 1.0,
                      bool joined = false) {
  const bool f32 = dtype_bytes == 4;
  const int64_t cus = (int64_t)(256 * part), slots = f32 && hd == 128 ? cus : 2 * cus, least_chunks = f32 ? 1 : 2;
  int best = 1;
  double least = 0.0;
  for (int n = 1; n <= 64 && (n == 1 || (n * least_chunks <= chunks && wgs * n <= 4 * slots)); ++n) {
    const bool alone = wgs * n <= cus;
    const double chunk = f32 ? (alone && hd == 64 ? 4.0 : 8.0) : (alone ? 1.1 : 1.9) * (joined ? 1.3 : 1.0);
    const double t = (double)((wgs * n + slots - 1) / slots) * ((double)((chunks + n - 1) / n) + (f32 ? 0.5 : 2.0)) * chunk +
                     split_us(n, rows, hd, joined);
    if (n == 1 || t < least) {
      best = n;
      least = t;
    }
  }
  return best;
}
// Likewise of single tokens' workgroups, 1.5 us for 128 keys, which their four waves take at a time.
inline int token_split(int64_t wgs, int64_t chunks, int64_t rows, int hd, bool joined = false) {
  int best = 1;
  double least = 0.0;
  for (int n = 1; n <= 32 && (n == 1 || (n * 2 <= chunks && wgs * n <= 2048)); ++n) {
    const double t =
        (double)((wgs * n + 511) / 512) * ((chunks + 2 * n - 1) / (2 * n) + 3) * 1.5 + split_us(n, rows, hd, joined);
    if (n == 1 || t < least) {
      best = n;
      least = t;
    }
  }
  return best;
}

// The sequences' first tokens, where the host knows the packing and there are few (n = 0: it does not): a tile
// then holds one sequence's tokens.  Otherwise tiles are cut from the batch as it is and walk their runs; a tile
// of two sequences takes twice as long as the others (fp32, 700 and 300 tokens, window 2048: 422 us, and
// 294 us with each sequence's own tiles).
constexpr int kMaxSeqs = 64;
struct SeqStarts {
  int n;
  int start[kMaxSeqs + 1];
};

// Tiles unless the caller promised single tokens, or there are no more rows than one token's MFMAs take.
inline int tiled_tokens(int64_t tokens, int q_heads, int kv_heads, int64_t max_query_len) {
  const int G = q_heads / kv_heads;
  return max_query_len != 1 && G <= kTileRows / 2 && tokens * G > 16 ? kTileRows / G : 0;
}
// What the packing on the host says: the sequences, if they are few; else the tokens [first, end) of the tiles that
// a tile kernel leaves.
struct TilePlan {
  bool known = false;
  int64_t first = 0, end = 0;
  SeqStarts seqs{};
};
inline TilePlan tile_plan(const int32_t* cu, int num_seqs, int tile_tokens) {
  TilePlan plan;
  plan.known = true;
  int n = 0;
  for (int s = 0; s < num_seqs && n <= kMaxSeqs; ++s) {
    if (cu[s] == cu[s + 1]) continue;
    if (n < kMaxSeqs) {
      plan.seqs.start[n] = cu[s];
      plan.seqs.start[n + 1] = cu[s + 1];
    }
    ++n;
  }
  if (n <= kMaxSeqs) {
    plan.seqs.n = n;
    return plan;
  }
  plan.seqs = SeqStarts{};
  int64_t tile = -1;
  int runs = 0;
  const auto close = [&] {
    if (tile < 0 || runs <= kTileMaxRuns) return;
    if (plan.end == 0) plan.first = tile * tile_tokens;
    plan.end = (tile + 1) * tile_tokens;
  };
  for (int s = 0; s < num_seqs; ++s) {
    if (cu[s] == cu[s + 1]) continue;
    const int64_t b = cu[s] / tile_tokens, e = (cu[s + 1] - 1) / tile_tokens;  // its first and last tile
    if (b != tile) {
      close();
      tile = b;
      runs = 0;
    }
    ++runs;
    if (e != tile) {
      close();
      tile = e;
      runs = 1;
    }
  }
  close();
  plan.end = std::min<int64_t>(plan.end, cu[num_seqs]);
  return plan;
}

// What both tile kinds and the single tokens need of a call.
template <typename T>
inline bool attn_mfma(const AttnArgs<T>& a) {
  return (a.hd == 64 || a.hd == 128) && a.bs % 16 == 0 && aligned16(a.q) && aligned16(a.out) &&
         aligned16(a.kc) && aligned16(a.vc) && a.q_stride % Pack<T>::N == 0 && a.scale_log2 > 0.0f &&
         (int64_t)a.kv_heads * a.hd * 64 < INT32_MAX && a.num_blocks <= INT32_MAX / a.bs;
}

}  // namespace nvf
