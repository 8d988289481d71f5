// The paged key-value cache: new tokens go into pages (position rotation applied on the way), and one or a few new tokens per
// sequence attend over them.
//
// The reference has neither (its attn_incremental.cu:329-481 is a stale bf16 header over one contiguous cache). Row kv_len + i
// of the prefill kernel (cuda/attn_fwd_i8.cuh:368-619) gives the attention's semantics: keys n - W' .. n - 1 of the sequence
// and the sink, n = kv_len + i, temperature D^-1/2 log2(min(W', n) + 4) temp_h, base-2 softmax.
//
// Layout: pages int8 [n_pages][n_kv_heads][page_size][K(D) | V(D)], scales f32 [n_pages][n_kv_heads][page_size][2]: a page of one
// head is one run of memory. page_table i32 [n_seqs][max_pages] names the pages of a sequence in order of position.
// Indexes that come from device memory (sequences, positions, pages) are checked there: what lies outside its range is left
// out and recorded in the status words.
#pragma once

#include "ptx.cuh"

namespace x17 {

constexpr f32 PAGED_TINY = 0x1p-100f;   // a head whose largest magnitude is no larger is stored as zeros

struct PagedPool {
	i8 *pages;
	f32 *scales;            // null: FixedI8
	i32 const *table;       // [n_seqs][max_pages]
	u32 n_pages, n_seqs, max_pages;
	u32 page_shift;         // log2(page_size)
	u32 n_kv_heads;
	u32 page_rows;          // rows (head, slot) of a page
	// row of (page, head, slot)
	X17_DEV u64 row(u32 page, u32 head, u32 slot) const { return u64(page) * page_rows + ((head << page_shift) + slot); }
};

// Division by a number that the host knows, for n * d up to 2^32.
struct FastDiv {
	u32 d, m;   // m: 2^32 / d, rounded up
	X17_DEV u32 operator()(u32 n) const { return d == 1 ? n : __umulhi(n, m); }
};

struct PagedAppendParams {
	PagedPool pool;
	void const *q, *kv;     // i8 or bf16, [tokens][stride]; q may be null
	i32 const *seqs, *positions;
	int16_t const *rope;    // [rope_rows][rotary / 2][cos, sin] in units of 2^-14; null with rotary 0
	i8 *q_out, *kv_out;     // kv_out may be null
	f32 *q_scale;           // [tokens][n_heads], scaled form
	u64 q_stride, kv_stride;
	u32 tokens, n_heads, rope_rows, rotary;
	u32 parts;              // warps that share a token's heads
	u32 *status;
};

struct PagedDecodeParams {
	PagedPool pool;
	i8 const *q;            // [batch * n_tokens][q_stride]
	f32 const *q_scale;     // [batch * n_tokens][n_heads], scaled form
	i32 const *kv_lens;     // [batch]
	i8 const *sink_k, *sink_v;
	f32 const *temperature;
	void *out;              // i8 or bf16, [batch * n_tokens][o_stride]
	f32 *l;                 // [batch * n_tokens][n_heads] or null
	u64 q_stride, o_stride;
	u32 n_heads, n_tokens;
	u32 chunk_rows;         // rows (query heads of a group x new tokens) of a chunk
	FastDiv chunks, group;  // chunks that a key head's rows take; query heads that share a key head
	u32 n_x;                // key heads x chunks
	u32 splits;             // 0: the list; else CTAs (a cluster) for every (sequence, x)
	u32 first_ctas;         // of the list: CTAs that the chip holds at once
	u32 window;             // 0xFFFFFFFF = unbounded
	bool out_i8;
	u32 *status;
};

// Page and slot of a token; false where an index is out of range.
X17_DEV bool paged_slot(PagedPool const &pool, i32 seq, i32 pos, u32 &page, u32 &slot) {
	u32 const at = u32(pos) >> pool.page_shift;
	if (u32(seq) >= pool.n_seqs || pos < 0 || at >= pool.max_pages) return false;
	page = u32(pool.table[u64(u32(seq)) * pool.max_pages + at]);
	slot = u32(pos) & ((1u << pool.page_shift) - 1);
	return page < pool.n_pages;
}

// ---- append ------------------------------------------------------------------------------------
//
// Reads and writes every row once: HBM-bound for prompts, one chain of four loads (position, page, row of the rope table) for a
// decode step. A warp takes a token, or where there are few tokens a part of its heads. A lane holds 32 dims of a head, in two runs
// of 16: both halves of 16 pairs, whose cosines and sines it loads once and keeps for all heads of the token. Lanes of one head
// lie side by side, so loads and stores are whole sectors. The next heads' row is on its way under the arithmetic.
// Measured: 8192 tokens of 32 + 32 heads of width 128, with a copy of the keys and values, 271 MB, 49.4 us: 5.5 TB/s. Scaled, 13001
// tokens of 64 + 8 heads of width 64, 205 MB, 41.0 us: 5.0 TB/s, with the issue slots half taken. One token 2.0 us, 121 tokens 3.0.
//
// FixedI8: x' = (x cos - y sin + 2^13) >> 14 is one dp2a (two products of 16 by 8 bits and a sum), a dp4a for the y that -sin - 1
// leaves over, and a shift, exact in 32 bits for every int16 in the table.
// Scaled: x' in f32, two pairs an instruction (46.0 us -> 41.6 for the second case); bf16 times a table value is exact, so x'
// has one rounding and is the same however it is fused; absmax over the lanes of a head; code = rint(x' * (127 / absmax)) by
// adding 1.5 * 2^23 (|code| <= 127, so its low byte is it).

namespace append_cfg {
constexpr u32 THREADS = 64, WARPS = THREADS / 32;
// CTAs of an SM: 28 warps of 72 registers; the scaled form 20 of 96, 32 of which are the cosines and sines in f32. A row ahead a
// warp and these many warps are faster than two rows ahead and the 24 or 16 that those leave place for (52.0, 46.5 us below).
template <bool SCALED>
constexpr u32 CTAS = SCALED ? 10 : 14;
}

// a: two signed 16-bit values, pair PAIR of b's signed bytes
template <u32 PAIR>
X17_DEV i32 dp2a_s16_s8(u32 a, u32 b, i32 c) {
	return PAIR == 0 ? __dp2a_lo(i32(a), i32(b), c) : __dp2a_hi(i32(a), i32(b), c);
}
// four sums in units of 2^-14 -> codes
X17_DEV u32 pack4_turned(i32 a, i32 b, i32 c, i32 d) {
	constexpr i32 LEAST = -127 * 16384;   // the pack saturates at -128
	a = max(a, LEAST) >> 14;
	b = max(b, LEAST) >> 14;
	c = max(c, LEAST) >> 14;
	d = max(d, LEAST) >> 14;
	u32 hi, packed;
	asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(d), "r"(c));
	asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(packed) : "r"(b), "r"(a), "r"(hi));
	return packed;
}

// One head's 32 dims of a lane: FixedI8 bytes, or bf16 pairs.
template <bool SCALED>
struct AppendRow {
	uint4 lo[SCALED ? 2 : 1], hi[SCALED ? 2 : 1];
};

template <u32 D, bool SCALED, bool ADJACENT>
__global__ void __launch_bounds__(append_cfg::THREADS, append_cfg::CTAS<SCALED>)
paged_append_kernel(const PagedAppendParams p) {
	constexpr u32 C = D / 32;        // lanes of a head
	constexpr u32 HEADS = 32 / C;    // heads of a warp at once
	constexpr u32 SIZE = SCALED ? 2 : 1;
	pdl_launch_dependents();
	pdl_wait();
	u32 const lane = threadIdx.x & 31, chunk = lane % C;
	u32 const n_q = p.q == nullptr ? 0u : p.n_heads, n_kv = p.pool.n_kv_heads;
	u32 const per_token = n_q + 2 * n_kv;   // heads: queries, keys, values
	u32 const unit = blockIdx.x * append_cfg::WARPS + (threadIdx.x >> 5);
	u32 const token = unit / p.parts, part = unit - token * p.parts;
	if (token >= p.tokens) return;
	i32 const seq = p.seqs[token], pos = p.positions[token];
	// the lane's two runs of 16 dims
	bool const turns = chunk < p.rotary / 32;
	u32 const off0 = turns && !ADJACENT ? chunk * 16 : chunk * 32;
	u32 const off1 = turns && !ADJACENT ? p.rotary / 2 + chunk * 16 : chunk * 32 + 16;

	u32 const rounds = (per_token + HEADS - 1) / HEADS, each = (rounds + p.parts - 1) / p.parts;
	u32 const from = part * each, to = min(from + each, rounds);
	u8 const *const q_row = static_cast<u8 const *>(p.q) + u64(token) * p.q_stride * SIZE;
	u8 const *const kv_row = static_cast<u8 const *>(p.kv) + u64(token) * p.kv_stride * SIZE;
	auto load = [&](u32 round, AppendRow<SCALED> &row) {
		u32 const h = round * HEADS + lane / C;
		if (round >= to || h >= per_token) return;
		u32 const kv = h - n_q;   // keys, then values
		u8 const *src = h < n_q ? q_row + h * D * SIZE : kv < n_kv ? kv_row + kv * 2 * D * SIZE : kv_row + ((kv - n_kv) * 2 + 1) * D * SIZE;
#pragma unroll
		for (u32 i = 0; i < SIZE; ++i) {
			row.lo[i] = reinterpret_cast<uint4 const *>(src + off0 * SIZE)[i];
			row.hi[i] = reinterpret_cast<uint4 const *>(src + off1 * SIZE)[i];
		}
	};
	AppendRow<SCALED> row;
	load(from, row);
	if (seq < 0) return;   // padding
	u32 page = 0, slot = 0;
	if (!paged_slot(p.pool, seq, pos, page, slot) || (p.rotary != 0 && u32(pos) >= p.rope_rows)) {
		if (lane == 0 && part == 0) report_status(p.status, ST_BAD_INDEX, token);
		return;
	}
	// cos | sin of the lane's 16 pairs
	__align__(16) u32 cs[16];
	if (turns) {
		uint4 const *src = reinterpret_cast<uint4 const *>(p.rope + (u64(u32(pos)) * (p.rotary / 2) + chunk * 16) * 2);
#pragma unroll
		for (u32 i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(cs + 4 * i) = src[i];
	}
	// the scaled form has them in f32
	u64 cos2[SCALED ? 8 : 1], sin2[SCALED ? 8 : 1], nothing2 = 0;
	if constexpr (SCALED) {
		f32 const nothing = __uint_as_float(p.parts >> 31);   // 0, which the compiler does not know
		nothing2 = pack_f32x2(nothing, nothing);
		if (turns) {
#pragma unroll
			for (u32 i = 0; i < 8; ++i) {
				auto c = [&](u32 j) { return f32(i32(cs[j] << 16) >> 16) * 0x1p-14f; };
				auto sn = [&](u32 j) { return f32(i32(cs[j]) >> 16) * 0x1p-14f; };
				cos2[i] = pack_f32x2(c(2 * i), c(2 * i + 1));
				sin2[i] = pack_f32x2(sn(2 * i), sn(2 * i + 1));
			}
		}
	}
	u64 const slot_row = p.pool.row(page, 0, slot);

	for (u32 round = from; round < to; ++round) {
		AppendRow<SCALED> const now = row;
		load(round + 1, row);
		u32 const h = round * HEADS + lane / C;
		bool const live = h < per_token, is_q = h < n_q, is_v = !is_q && h - n_q >= n_kv;
		u32 const kv_head = is_q ? 0u : is_v ? h - n_q - n_kv : h - n_q;
		bool const turn = turns && !is_v;
		__align__(16) u32 lo[4], hi[4];
		if constexpr (!SCALED) {
			*reinterpret_cast<uint4 *>(lo) = now.lo[0];
			*reinterpret_cast<uint4 *>(hi) = now.hi[0];
			if (turn) {
				// word w of eight: pairs 2 w, 2 w + 1 as bytes x y x y
				auto pairs = [&](u32 w) -> u32 {
					if constexpr (ADJACENT) return w < 4 ? lo[w] : hi[w - 4];
					return __byte_perm(lo[w / 2], hi[w / 2], w % 2 == 0 ? 0x5140 : 0x7362);
				};
				i32 x[16], y[16];
#pragma unroll
				for (u32 w = 0; w < 8; ++w) {
					u32 const b = pairs(w);
#pragma unroll
					for (u32 e = 0; e < 2; ++e) {
						u32 const c = cs[2 * w + e];
						// (cos, -sin - 1), and y on top, since -sin has no 16 bits where sin is -2^15; (sin, cos)
						u32 const minus = c ^ 0xFFFF0000u, swapped = __byte_perm(c, c, 0x1032);
						i32 const y1 = __dp4a(i32(b), e == 0 ? 0x100 : 0x1000000, 8192);
						x[2 * w + e] = e == 0 ? dp2a_s16_s8<0>(minus, b, y1) : dp2a_s16_s8<1>(minus, b, y1);
						y[2 * w + e] = e == 0 ? dp2a_s16_s8<0>(swapped, b, 8192) : dp2a_s16_s8<1>(swapped, b, 8192);
					}
				}
#pragma unroll
				for (u32 w = 0; w < 4; ++w) {
					if constexpr (ADJACENT) {
						lo[w] = pack4_turned(x[2 * w], y[2 * w], x[2 * w + 1], y[2 * w + 1]);
						hi[w] = pack4_turned(x[2 * w + 8], y[2 * w + 8], x[2 * w + 9], y[2 * w + 9]);
					} else {
						lo[w] = pack4_turned(x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]);
						hi[w] = pack4_turned(y[4 * w], y[4 * w + 1], y[4 * w + 2], y[4 * w + 3]);
					}
				}
			}
		} else {
			// pairs of x (and of y) lie side by side: x2[i] is x of pairs 2 i and 2 i + 1 in either order of a head's dims
			u64 x2[8], y2[8];
			auto low = [](u32 w) { return __uint_as_float(w << 16); };
			auto high = [](u32 w) { return __uint_as_float(w & 0xFFFF0000u); };
#pragma unroll
			for (u32 i = 0; i < 2; ++i) {
				u32 const a[4] = {now.lo[i].x, now.lo[i].y, now.lo[i].z, now.lo[i].w}, c[4] = {now.hi[i].x, now.hi[i].y, now.hi[i].z, now.hi[i].w};
				if constexpr (ADJACENT) {
#pragma unroll
					for (u32 w = 0; w < 2; ++w) {
						x2[2 * i + w] = pack_f32x2(low(a[2 * w]), low(a[2 * w + 1]));
						y2[2 * i + w] = pack_f32x2(high(a[2 * w]), high(a[2 * w + 1]));
						x2[4 + 2 * i + w] = pack_f32x2(low(c[2 * w]), low(c[2 * w + 1]));
						y2[4 + 2 * i + w] = pack_f32x2(high(c[2 * w]), high(c[2 * w + 1]));
					}
				} else {
#pragma unroll
					for (u32 w = 0; w < 4; ++w) {
						x2[4 * i + w] = pack_f32x2(low(a[w]), high(a[w]));
						y2[4 * i + w] = pack_f32x2(low(c[w]), high(c[w]));
					}
				}
			}
			if (turn) {
#pragma unroll
				for (u32 i = 0; i < 8; ++i) {
					u64 const x = x2[i], y = y2[i];
					x2[i] = fma_f32x2(x, cos2[i], mul_f32x2(y, sin2[i]) ^ 0x8000000080000000ull);
					y2[i] = fma_f32x2(x, sin2[i], mul_f32x2(y, cos2[i]));
				}
			}
			f32 top = 0.0f;
#pragma unroll
			for (u32 i = 0; i < 8; ++i) {
				f32 v[4];
				unpack_f32x2(x2[i], v[0], v[1]);
				unpack_f32x2(y2[i], v[2], v[3]);
#pragma unroll
				for (u32 j = 0; j < 4; ++j) top = fmaxf(top, fabsf(v[j]));
			}
#pragma unroll
			for (u32 mask = 1; mask < C; mask <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, mask));
			bool const some = top > PAGED_TINY;
			f32 const inv = some ? __fdiv_rn(127.0f, top) : 0.0f;
			if (chunk == 0 && live) {
				f32 const scale = some ? __fmul_rn(top, 1.0f / 127.0f) : 0.0f;
				if (is_q) p.q_scale[u64(token) * p.n_heads + h] = scale;
				else p.pool.scales[(slot_row + (u64(kv_head) << p.pool.page_shift)) * 2 + is_v] = scale;
			}
			// (a product plus nothing, since product and sum would become one operation, and a value on a tie another code)
			u64 const inv2 = pack_f32x2(inv, inv);
			auto codes = [&](u64 v, u32 &a, u32 &b) {
				f32 c0, c1;
				unpack_f32x2(add_f32x2(fma_f32x2(v, inv2, nothing2), pack_f32x2(12582912.0f, 12582912.0f)), c0, c1);
				a = __float_as_uint(c0);
				b = __float_as_uint(c1);
			};
#pragma unroll
			for (u32 w = 0; w < 8; ++w) {
				u32 c[4];   // of four dims in order
				if constexpr (ADJACENT) {
					codes(x2[w], c[0], c[2]);
					codes(y2[w], c[1], c[3]);
				} else {
					codes(w < 4 ? x2[2 * w] : y2[2 * w - 8], c[0], c[1]);
					codes(w < 4 ? x2[2 * w + 1] : y2[2 * w - 7], c[2], c[3]);
				}
				u32 const word = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
				if (w < 4) lo[w] = word;
				else hi[w - 4] = word;
			}
		}
		if (!live) continue;
		auto store = [&](i8 *dst) {
			*reinterpret_cast<uint4 *>(dst + off0) = *reinterpret_cast<uint4 const *>(lo);
			*reinterpret_cast<uint4 *>(dst + off1) = *reinterpret_cast<uint4 const *>(hi);
		};
		if (is_q) {
			store(p.q_out + u64(token) * p.q_stride + h * D);
		} else {
			store(p.pool.pages + (slot_row + (u64(kv_head) << p.pool.page_shift)) * 2 * D + is_v * D);
			if (p.kv_out != nullptr) store(p.kv_out + u64(token) * p.kv_stride + (kv_head * 2 + is_v) * D);
		}
	}
}

// ---- decode ------------------------------------------------------------------------------------
//
// A pass over a cache is bound by HBM: the kernel's job is to keep enough bytes in flight on every SM, whatever the sequences'
// lengths, and to stay out of their way. The rows (query heads of a group, times new tokens) that share a key head are taken up to
// twenty-four at a time, so a key is read once for all of them. A warp works alone: it fills a ring of two steps of 8 KB (32 keys at
// width 128) in shared memory (cp.async; page table entries are fetched 32 runs of keys at once). A page of a head is one run of
// memory, so pages cost no more than a contiguous cache. The work is dealt out in one of two ways (paged_places in api.cu):
//   - Where the call's warps find place on the chip at once, every (sequence, x) has a CTA of up to 12 warps or a cluster of up to 8 of
//     them, x being a key head's chunk of rows. Its warps take equal runs of its steps; parts meet in shared memory.
//   - Else the work of a call is the list of all steps of all (sequence, x), and the warps of a grid that fills the chip take equal
//     runs of it: one sequence of 131072 keys and 128 ragged ones keep the chip equally busy, and no length has to be known on
//     the host. Where a warp's run covers a whole (sequence, x) it writes the output itself. What the four warps of a CTA share
//     they join at their end; the parts of what several CTAs share go through scratch memory and a second kernel.
//
// Scores: mma m16n8k32 (s8 x s8 -> s32, exact), rows as its M, keys as its N; a lane's bytes of a key row are consecutive, the
// query's are permuted the same way. Values: mma m16n8k16 (f16 x f16 -> f32) with V transposed as its first operand (dims as M)
// and the weights as the second (rows as N), which is how the scores' fragments lie; accumulators are a lane's 16 dims of two rows.
// V's codes are exact in f16 (integer added to 1024 as bits). Weights are 2^(x - m + 8) against a maximum m that moves only when a
// score passes it by 6; m starts at the sink's score, so no key and no row leaves it undefined. A FixedI8 cache's are two f16
// numbers, hi + lo: 22 bits down to 2^-10 of m's weight, below that an error of at most 2^-33 of the total. With hi alone (11 bits)
// 0.6 to 4 % of the bf16 outputs were not those of the exact value, with both 0.02 to 0.07 %, as with f32 weights and f32 products;
// it costs 1.3 % (2.15 GB), 3 % (one user) to 6 % (64 heads of width 32, five rows), 9 % where 24 rows of width 64 are bound by it. For a FixedI8 output sums of 16 keys are added in
// f32, so that its codes are those of the exact value but for near ties: of 14.8 million codes 9 differ, 18 with f32 weights and
// matrix products in f32 (with the products' own long sums, which round toward zero, 37).
// A scaled cache's weights are multiplied by the value's scale in f32 and become two bf16 numbers: 16 bits in the whole range of f32,
// so that no scale, however large, takes another key's bits. Values of up to 2^112 / keys do not overflow.
//
// Measured, bf16 output (L2 does not hold the cache but in the first two): 1500 keys x 32 heads of width 128 6.9 us, of which launch
// and the chain length - page - keys - join - store are all but 2; 48 ragged sequences in windows of 1024 (8 key heads) 20 us, 4.5
// TB/s; 64 x 4096 x 32 heads 2.15 GB, 337 to 347 us, 6.2 to 6.4 TB/s; 128 ragged ones 543 MB, 105 to 108 us, 5.0 to 5.2 TB/s (SMs
// read at different rates, and the list's end is 8 KB a warp); one sequence of 131072 keys with scales 277 MB, 57 to 59 us, 4.8 TB/s,
// of which the merge is 4. With three tiles of rows, 24 ragged sequences of 54 MB in 24 rows of width 64 with scales take 36.7 us: latency of the products'
// chain at three warps a scheduler, not HBM.

namespace paged_cfg {
constexpr u32 WARPS = 4;         // of a CTA at least
constexpr u32 MAX_WARPS = 12;    // of any CTA
constexpr u32 KS = 32;           // keys that the products take at once
// Keys of a step, which is what a warp asks for at once: 8 KB at every width, in runs of 16 keys, each in one page.
template <u32 D>
constexpr u32 STEP = KS * (128 / D);
template <u32 D>
constexpr u32 RUNS = STEP<D> / 16;
constexpr u32 STAGES = 2;
constexpr u32 ROWS = 8;          // of a tile
constexpr u32 MOST_TILES = 3;    // of a warp
constexpr u32 LONG_RUN = 30;    // steps of a warp, from which the list is not dealt out equally
constexpr u32 MORE_CTAS = 2;    // CTAs of the list then, as a multiple of what the chip holds at once
constexpr f32 SHIFT = 8.0f, ARG_MAX = 14.0f;   // weights are 2^(x - m + SHIFT), at most 2^ARG_MAX (f16 ends below 2^16)
constexpr u32 MAX_SPLITS = 8;    // CTAs of a cluster
constexpr u32 MOST_STEPS = 23;   // of a warp, where every (sequence, x) has CTAs of its own
constexpr u32 MERGE_WARPS = 8;   // of a CTA that joins parts
// Warps on an SM: 12 with a step in work and a step on its way each, 210 KB of rings. With two or three tiles at width 128 the
// sums alone are 64 or 96 registers: eight.
template <u32 D, u32 RT>
constexpr u32 SM_WARPS = D == 128 && RT > 1 ? 8 : 12;
template <u32 D, u32 RT>
constexpr u32 REGS = 65536 / (SM_WARPS<D, RT> * 32) / 8 * 8 - (SM_WARPS<D, RT> == 8 ? 8 : 0);
// In the ring a key's row [K | V] keeps its 2 D bytes, its 16-byte pieces in places i ^ ring_swap(row): without bank conflicts for the
// fragments' loads (keys: eight rows, four lanes a row; values: every other row, eight lanes a row; at width 32 values have two).
template <u32 D>
__host__ __device__ constexpr u32 ring_swap(u32 row) {
	return D == 128 ? row & 7 : D == 64 ? ((row ^ row >> 1) & 1) << 2 | (row >> 2 & 1) << 1 : (row >> 1 & 1) << 1;
}
template <u32 D, bool SCALED>
constexpr u32 STAGE_BYTES = STEP<D> * (2 * D + (SCALED ? 8 : 0));
template <u32 D, bool SCALED>
constexpr u32 RING_BYTES = STAGES * STAGE_BYTES<D, SCALED>;   // of a warp
}  // namespace paged_cfg

// Slots for parts of a (sequence, x), each [rows]. One for every warp: of what began in an earlier warp's run and ended in its
// own, before the run did. Behind these two for every CTA: [0] of what began in an earlier CTA's run, [1] of what begins in its
// own and goes on behind it.
struct PagedScratch {
	uint2 *shared_by;   // [sequences][x]: first CTA, number of CTAs; written on every call
	float4 *ms;         // [slots][rows]: m - SHIFT, sum, the sink's score
	f32 *o;             // [slots][rows][D]
};

X17_DEV void cp_async_16(u32 dst, void const *src) {
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
X17_DEV void cp_async_8(u32 dst, void const *src) {
	asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
X17_DEV void cp_async_commit() {
	asm volatile("cp.async.commit_group;" ::: "memory");
}
template <u32 N>
X17_DEV void cp_async_wait() {
	asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// c[0], c[1]: row lane / 4, columns 2 (lane % 4) and the next one; c[2], c[3]: row lane / 4 + 8. The first product of a sum has
// no sum before it.
template <bool FIRST>
X17_DEV void mma_s8(i32 (&c)[4], u32 const (&a)[4], u32 b0, u32 b1) {
	if constexpr (FIRST) {
		asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
			: "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
			: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
	} else {
		asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
			: "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
			: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
	}
}
// the same layout with K = 16: f16, or BF16, in f32 sums
#define X17_MMA_VALUES(TYPE)                                                                                                                  \
	if constexpr (FIRST) {                                                                                                                    \
		asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"   \
			: "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                                                    \
			: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));                                                         \
	} else {                                                                                                                                  \
		asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"       \
			: "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                                                    \
			: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                                                                    \
	}
template <bool BF16, bool FIRST>
X17_DEV void mma_values(f32 (&c)[4], u32 const (&a)[4], u32 b0, u32 b1) {
	if constexpr (BF16) {
		X17_MMA_VALUES("bf16")
	} else {
		X17_MMA_VALUES("f16")
	}
}
#undef X17_MMA_VALUES
X17_DEV u32 f32x2_to_f16x2(f32 lo, f32 hi) {
	u32 r;
	asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}
X17_DEV void f16x2_values(u32 h2, f32 &lo, f32 &hi) {
	asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h2));
}
// byte J of a and of b, signed, as f16x2 (the bits 0x6400 + (code + 128) are 1024 + 128 + code) or as bf16x2, whose eight bits hold
// a code but not 128 more of it (128 + the lower seven bits, less 128 or, for a negative code, 256)
template <bool BF16, u32 J>
X17_DEV u32 codes_to_x2(u32 a, u32 b) {
	u32 const w = __byte_perm(a, b, (J + 4) << 8 | J);
	u32 r;
	if constexpr (BF16) {
		u32 low, less;
		asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(low) : "r"(w), "r"(0x007F007Fu), "r"(0x43004300u));
		asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(less) : "r"(w), "r"(0x00800080u), "r"(0x43004300u));
		asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(low), "r"(less));
	} else {
		asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(w), "r"(0x00FF00FFu), "r"(0x64806480u));
		asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0xE480E480u));
	}
	return r;
}
// N words (1, 2, 4 or 8) from shared memory
template <u32 N>
X17_DEV void ld_shared_words(u32 addr, u32 (&w)[N]) {
	if constexpr (N == 1) {
		asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
	} else if constexpr (N == 2) {
		asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
	} else {
#pragma unroll
		for (u32 i = 0; i < N; i += 4) {
			uint4 const v = ld_shared_v4(addr + i * 4);
			w[i] = v.x;
			w[i + 1] = v.y;
			w[i + 2] = v.z;
			w[i + 3] = v.w;
		}
	}
}
template <u32 N>
X17_DEV void ld_global_words(i8 const *p, u32 (&w)[N]) {
	if constexpr (N % 4 == 0) {
#pragma unroll
		for (u32 i = 0; i < N; i += 4) {
			uint4 const v = reinterpret_cast<uint4 const *>(p)[i / 4];
			w[i] = v.x;
			w[i + 1] = v.y;
			w[i + 2] = v.z;
			w[i + 3] = v.w;
		}
	} else {
		uint2 const v = *reinterpret_cast<uint2 const *>(p);
		w[0] = v.x;
		w[1] = v.y;
	}
}

// What a sequence's rows see: token i has position n = length(i) and keys [first(n), n).
template <u32 STEP>
struct PagedSpan {
	u32 len, capacity, window;
	X17_DEV PagedSpan(PagedDecodeParams const &p, i32 kv_len)
		: len(u32(max(kv_len, 0))), capacity(p.pool.max_pages << p.pool.page_shift), window(p.window) {}
	X17_DEV u32 length(u32 token) const { return min(len + token, capacity); }
	X17_DEV u32 first(u32 n) const { return n - min(n, window); }
	X17_DEV u32 base() const { return first(length(0)) & ~15u; }   // of the sequence's steps
	// one at least: a sequence without keys has its sink
	X17_DEV u32 steps(u32 n_tokens) const { return max(1u, (length(n_tokens - 1) - base() + STEP - 1) / STEP); }
};

// VD dims from d on of one row, from the keys' (m, s, v), m being a maximum less SHIFT, and the sink token.
template <u32 D, u32 VD>
X17_DEV void paged_finish(PagedDecodeParams const &p, u64 out_row, u32 head, u32 d, f32 m, f32 s, f32 (&v)[VD], f32 sink,
						   u32 const (&sink_v)[VD / 4]) {
	f32 const a = ex2_approx(sink - m);
	s += a;
	f32 const inv = rcp_approx(s);   // (one step)
	u64 const at = out_row * p.o_stride + head * D + d;
#pragma unroll
	for (u32 i = 0; i < VD; i += 4) {
		u32 const w = sink_v[i / 4];
		f32 x[4];
#pragma unroll
		for (u32 j = 0; j < 4; ++j) x[j] = __fmaf_rn(f32(i8(w >> (8 * j))) * 0.125f, a, v[i + j]) * inv;
		if (p.out_i8) {
			u32 c[4];
#pragma unroll
			for (u32 j = 0; j < 4; ++j) c[j] = u32(f32_to_fixedi8(x[j] * 8.0f));
			*reinterpret_cast<u32 *>(static_cast<i8 *>(p.out) + at + i) = pack4(c[0], c[1], c[2], c[3]);
		} else {
			*reinterpret_cast<uint2 *>(static_cast<u16 *>(p.out) + at + i) = make_uint2(cvt_bf16x2(x[0], x[1]), cvt_bf16x2(x[2], x[3]));
		}
	}
	if (d == 0 && p.l != nullptr) p.l[out_row * p.n_heads + head] = log2f(255.0f * s) + m;
}

// The list dealt out to CTAs in order. SMs do not read equally fast: with equal runs of 350 us the first are done 60 to 90 us before
// the last. From 30 steps a warp on, the CTAs that are there from the beginning get nine tenths of the work, and as many smaller
// ones the rest, each where one has ended: 64 x 4096 keys x 32 heads (148 steps a warp) 356 -> 344 us, 128 ragged sequences of 543 MB
// (37 steps) 109.3 -> 107.8; 131072 keys of one sequence (18 steps) 57.9 -> 72.3 us, so shorter runs stay equal.
struct PagedRuns {
	u32 total, first, large, small;
	PagedRuns() = default;
	X17_DEV PagedRuns(u32 total, u32 first, u32 ctas) : total(total), first(first) {
		bool const equal = ctas == first || total / (first * paged_cfg::WARPS) < paged_cfg::LONG_RUN;
		large = (equal ? total : total / 10 * 9) / first + 1;
		u32 const rest = total - min(total, large * first);
		small = equal ? 1 : rest / (ctas - first) + 1;
	}
	X17_DEV u32 start(u32 cta) const { return min(total, cta <= first ? cta * large : first * large + (cta - first) * small); }
	X17_DEV u32 cta(u32 unit) const { return unit < first * large ? unit / large : first + (unit - first * large) / small; }
};

template <u32 D, u32 VD>
X17_DEV void paged_finish(PagedDecodeParams const &p, u64 out_row, u32 head, u32 d, f32 m, f32 s, f32 (&v)[VD], f32 sink) {
	u32 sink_v[VD / 4];
#pragma unroll
	for (u32 i = 0; i < VD / 4; ++i) sink_v[i] = reinterpret_cast<u32 const *>(p.sink_v + u64(head) * D + d)[i];
	paged_finish<D, VD>(p, out_row, head, d, m, s, v, sink, sink_v);
}

constexpr f32 NO_PART = -3.0e38f;   // m of what has no keys
// Joins n parts of four dims of a row, first their maxima, so that no part waits for the one before. ms: m - SHIFT, sum, the
// sink's score; get(k, true) is a part's, get(k, false) its values.
template <typename Get>
X17_DEV void paged_join(float4 &ms, float4 &v, u32 n, Get get) {
	f32 up = ms.x;
#pragma unroll 4
	for (u32 k = 0; k < n; ++k) up = fmaxf(up, get(k, true).x);
	f32 const a = ex2_approx(ms.x - up);
	ms.x = up;
	ms.y *= a;
	v = make_float4(v.x * a, v.y * a, v.z * a, v.w * a);
#pragma unroll 4
	for (u32 k = 0; k < n; ++k) {
		float4 const m = get(k, true);
		if (m.x == NO_PART) continue;   // (where its values would lie may be anything)
		float4 const part = get(k, false);
		f32 const e = ex2_approx(m.x - up);
		v.x = __fmaf_rn(part.x, e, v.x);
		v.y = __fmaf_rn(part.y, e, v.y);
		v.z = __fmaf_rn(part.z, e, v.z);
		v.w = __fmaf_rn(part.w, e, v.w);
		ms.y = __fmaf_rn(m.y, e, ms.y);
		ms.z = m.z;   // (the same in every part)
	}
}
X17_DEV void st_cluster_f32x4(u32 addr_cluster, float4 v) {
	st_cluster_v4(addr_cluster, __float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w));
}

// One warp takes a run of steps, in order of sequence, x (key head, chunk of rows), step (the list). RT: tiles of eight
// rows that a chunk has. SUMS: sums of 16 keys leave the products and are added in f32.
template <u32 D, bool SCALED, u32 RT, bool SUMS>
__global__ void __maxnreg__((paged_cfg::REGS<D, RT>))
paged_decode_kernel(const PagedDecodeParams p, const PagedScratch scratch) {
	using namespace paged_cfg;
	constexpr u32 KW = D / 16;                       // words of a key row that a lane holds
	constexpr u32 VW = D / 32;                       // words of a value row that a lane holds
	constexpr u32 VD = D / 8;                        // dims of a lane
	constexpr u32 QT = (RT + 1) / 2;                 // products that the tiles' queries take
	constexpr u32 RB = 2 * D, SB = STAGE_BYTES<D, SCALED>, S_AT = STEP<D> * RB;   // pitch of a row, of a stage; its scales
	using Span = PagedSpan<STEP<D>>;
	constexpr u32 NEG_INF = 0xFF800000u;
	constexpr f32 ROOT = f32(D == 128 ? 0.08838834764831845 : D == 64 ? 0.125 : 0.17677669529663687);   // D^-1/2
	extern __shared__ __align__(16) u8 smem[];
	// what the warps leave for the end: [warp][of the run's beginning, of its end]; those of the end lie in the warps' rings
	enum : u32 { THERE = 1, BEGAN = 2, ENDED = 4 };
	__shared__ uint2 items[MAX_WARPS * 2];   // (sequence, x), flags
	// m, sum and the sink's score of each row of those; behind the values in the ring where an SM would else not hold three CTAs (only
	// there: 128 ragged sequences of width 128 take 108 us this way and 111 with all of it in the ring)
	constexpr bool MS_IN_RING = SM_WARPS<D, RT> / WARPS * (RING_BYTES<D, SCALED> * WARPS + MAX_WARPS * (RT * ROWS + 1) * 16 + 1024) > 228 * 1024;
	static_assert(!MS_IN_RING || RT * ROWS * (D + 4) * 4 <= RING_BYTES<D, SCALED>);
	__shared__ float4 item_ms[MS_IN_RING ? 1 : MAX_WARPS][RT * ROWS];
	auto end_ms = [&](u32 of_warp) -> float4 * {
		if constexpr (MS_IN_RING) return reinterpret_cast<float4 *>(smem + of_warp * STAGES * SB + RT * ROWS * D * 4);
		return item_ms[of_warp];
	};
	u32 const warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
	u32 const g = lane >> 2, t = lane & 3;
	u32 const n_warps = gridDim.x * warps, w = blockIdx.x * warps + warp;
	u32 const group = p.group.d;
	u32 const n_x = p.n_x;
	u32 const ring = smem_u32(smem) + warp * STAGES * SB;
	pdl_wait();

	// ---- the warp's run of units ----
	u32 start, n_units, b, x, step;
	PagedRuns runs{};
	if (p.splits == 0) {
		pdl_launch_dependents();
		u32 total = 0;
		for (u32 i = lane; i < p.pool.n_seqs; i += 32) total += Span(p, p.kv_lens[i]).steps(p.n_tokens);
#pragma unroll
		for (u32 mask = 16; mask > 0; mask >>= 1) total += __shfl_xor_sync(0xffffffffu, total, mask);
		total *= n_x;   // (below 2^32: checked on the host for sequences of full length)
		runs = PagedRuns(total, p.first_ctas, gridDim.x);
		u32 const from = runs.start(blockIdx.x), to = runs.start(blockIdx.x + 1), each = (to - from + warps - 1) / warps;
		if (from == to) return;
		start = min(from + warp * each, to);
		n_units = min(start + each, to) - start;
		u32 before = 0;
		b = 0;
		for (u32 target = start / n_x; n_units != 0; b += 32) {
			u32 const mine = b + lane < p.pool.n_seqs ? Span(p, p.kv_lens[b + lane]).steps(p.n_tokens) : 0u;
			u32 upto = mine;
#pragma unroll
			for (u32 d = 1; d < 32; d <<= 1) {
				u32 const v = __shfl_up_sync(0xffffffffu, upto, d);
				if (lane >= d) upto += v;
			}
			u32 const hit = __ballot_sync(0xffffffffu, before + upto > target);
			if (hit != 0) {
				u32 const at = __ffs(hit) - 1;
				before += __shfl_sync(0xffffffffu, upto - mine, at);
				b += at;
				break;
			}
			before += __shfl_sync(0xffffffffu, upto, 31);
		}
		u32 const steps_of = Span(p, n_units != 0 ? p.kv_lens[b] : 0).steps(p.n_tokens);
		x = (start - before * n_x) / steps_of;
		step = start - before * n_x - x * steps_of;
	} else {
		b = blockIdx.y;
		x = blockIdx.x;
		// the first pages' entries are brought closer while the length is on its way
		i32 touch = 0;
		if (lane * 8 < p.pool.max_pages) asm volatile("ld.global.b32 %0, [%1];" : "=r"(touch) : "l"(p.pool.table + u64(b) * p.pool.max_pages + lane * 8));
		u32 const all = Span(p, p.kv_lens[b]).steps(p.n_tokens), each = (all + p.splits - 1) / p.splits;
		u32 const from = min(blockIdx.z * each, all), to = min(from + each, all), mine = (to - from + warps - 1) / warps;
		start = step = min(from + warp * mine, to);
		n_units = min(start + mine, to) - start;
	}
	u32 left = n_units;

	// ---- the (sequence, x) in work, and the one behind it (whose first step is fetched under the last of this one) ----
	Span span(p, n_units != 0 ? p.kv_lens[b] : 0);
	u32 steps = span.steps(p.n_tokens);
	if (lane < 2) items[warp * 2 + lane] = make_uint2(0, 0);
	if ((!MS_IN_RING || n_units == 0) && lane < RT * ROWS) end_ms(warp)[lane] = make_float4(NO_PART, 0.0f, 0.0f, 0.0f);
	// page table entries of the 32 runs of 16 keys from `run` on, one a lane
	auto page_entries = [&](Span const &sp, u32 seq, u32 run) -> u32 {
		u32 const key = sp.base() + (run + lane) * 16;
		return key < sp.length(p.n_tokens - 1) ? u32(p.pool.table[u64(seq) * p.pool.max_pages + (key >> p.pool.page_shift)]) : 0u;
	};
	constexpr u32 PIECES = 2 * D / 16;   // of a row; a warp asks for 32
	u32 const piece = lane / PIECES * RB + (lane % PIECES ^ ring_swap<D>(lane / PIECES)) * 16;
	// this lane's bytes of key row g, and of value rows 2 t and 2 t + 1
	u32 const k_at = g * RB + (t * (D / 4) / 16 ^ ring_swap<D>(g)) * 16 + t * (D / 4) % 16;
	u32 const v_at[2] = {2 * t * RB + ((D + g * VD) / 16 ^ ring_swap<D>(2 * t)) * 16 + g * VD % 16,
						 (2 * t + 1) * RB + ((D + g * VD) / 16 ^ ring_swap<D>(2 * t + 1)) * 16 + g * VD % 16};
	u32 bad = 0;   // bit RUNS stage + run: its page is none
	// step s of a (sequence, x) into a stage; entries: of the runs from a multiple of 32 on
	auto issue = [&](Span const &sp, u32 seq, u32 kvh, u32 s, u32 entries, u32 stage) {
		u32 const n_hi = sp.length(p.n_tokens - 1);
#pragma unroll
		for (u32 j = 0; j < RUNS<D>; ++j) {
			u32 const page = __shfl_sync(0xffffffffu, entries, (s * RUNS<D> + j) & 31);
			u32 const key = sp.base() + s * STEP<D> + j * 16;
			u32 const bit = 1u << (stage * RUNS<D> + j);
			bad &= ~bit;
			if (page >= p.pool.n_pages) {
				bad |= bit;
				if (lane == 0) report_status(p.status, ST_BAD_INDEX, seq);
			} else if (key < n_hi) {
				u64 const row = p.pool.row(page, kvh, key & ((1u << p.pool.page_shift) - 1));
				i8 const *src = p.pool.pages + row * 2 * D + lane * 16;
				u32 const dst = ring + stage * SB + j * 16 * RB;
#pragma unroll
				for (u32 c = 0; c < PIECES / 2; ++c) cp_async_16(dst + c * 512 + (piece ^ ring_swap<D>(c * 32 / PIECES) * 16), src + c * 512);
				if constexpr (SCALED) {
					if (lane < 16) cp_async_8(ring + stage * SB + S_AT + (j * 16 + lane) * 8, p.pool.scales + (row + lane) * 2);
				}
			}
		}
		cp_async_commit();
	};
	u32 entries = 0, entries_ahead = 0;
	if (n_units != 0) {
		entries = page_entries(span, b, step * RUNS<D> & ~31u);
		entries_ahead = page_entries(span, b, (step * RUNS<D> & ~31u) + 32);
	}
	u32 stage = 0;
	bool asked = false;   // for the first step

	// tile j: dims g D / 8 + 2 j ([0], [1]) and + 2 j + 1 ([2], [3]) of rows 2 t ([0], [2]) and 2 t + 1 ([1], [3])
	f32 o[D / 16][RT][4];
#pragma unroll 1
	while (left != 0) {
		u32 const kvh = p.chunks(x), row0 = (x - kvh * p.chunks.d) * p.chunk_rows;
		u32 const rows = min(p.chunk_rows, group * p.n_tokens - row0);
		u32 const n_here = min(steps - step, left);
		left -= n_here;
		// the next one
		bool const b_ends = x + 1 == n_x;
		u32 const next_b = b_ends ? b + 1 : b, next_x = b_ends ? 0u : x + 1;
		Span next_span = span;
		u32 entries_next = 0;
		if (left != 0) {
			if (b_ends) next_span = Span(p, p.kv_lens[next_b]);
			entries_next = page_entries(next_span, next_b, 0);
		}

		// ---- this lane's rows: heads of the group for one of the new tokens (rows behind the last one repeat it and are not stored) ----
		u32 qa[QT][KW / 2][4];   // as the products' first operand, two tiles each
		u32 n[RT], lo[RT];
		f32 temp[RT], sink[RT], neg_m[RT], sum[RT];
		u32 qw[RT][KW], skw[RT][KW];
#pragma unroll
		for (u32 r = 0; r < RT; ++r) {
			u32 const my_row = row0 + min(g + r * ROWS, rows - 1);
			u32 const tok = p.group(my_row), head = kvh * group + my_row - tok * group;
			u64 const q_row = u64(b) * p.n_tokens + tok;
			ld_global_words(p.q + q_row * p.q_stride + head * D + t * (D / 4), qw[r]);
			ld_global_words(p.sink_k + u64(head) * D + t * (D / 4), skw[r]);
			temp[r] = p.temperature[head];
			if constexpr (SCALED) temp[r] *= p.q_scale[q_row * p.n_heads + head];
			n[r] = span.length(tok);
			lo[r] = span.first(n[r]);
		}
		if (!asked) issue(span, b, kvh, step, entries, 0);   // (under the loads above)
		asked = true;
#pragma unroll
		for (u32 r = 0; r < RT; ++r) {
			// D^-1/2 log2(min(W', n) + 4) temp_h, and the scales that are not the key's
			temp[r] *= ROOT * log2f(f32(n[r] - lo[r] + 4)) * (SCALED ? 1.0f : 0.015625f);
			i32 dot = 0;
#pragma unroll
			for (u32 k = 0; k < KW; ++k) {
				dot = __dp4a(i32(qw[r][k]), i32(skw[r][k]), dot);
				qa[r / 2][k / 2][k % 2 * 2 + r % 2] = qw[r][k];
				if (r + 1 == RT && r % 2 == 0) qa[r / 2][k / 2][k % 2 * 2 + 1] = 0;
			}
			dot += __shfl_xor_sync(0xffffffffu, dot, 1);
			dot += __shfl_xor_sync(0xffffffffu, dot, 2);
			sink[r] = f32(dot) * (SCALED ? temp[r] * 0.125f : temp[r]);
			neg_m[r] = SHIFT - sink[r];
			sum[r] = 0.0f;
		}
		// (zeros that the compiler does not know, or it would move them in front of every product)
#pragma unroll
		for (u32 k = 0; k < QT * KW / 2; ++k) {
			u32 (&q4)[4] = qa[k / (KW / 2)][k % (KW / 2)];
			asm volatile("" : "+r"(q4[0]), "+r"(q4[1]), "+r"(q4[2]), "+r"(q4[3]));
		}
#pragma unroll
		for (u32 j = 0; j < D / 16; ++j) {
#pragma unroll
			for (u32 e = 0; e < 4 * RT; ++e) o[j][e / 4][e % 4] = 0.0f;
		}
		u32 const n_min = span.length(p.group(row0));                                     // what every row sees: [lo_max, n_min)
		u32 const lo_max = span.first(span.length(p.group(row0 + rows - 1)));
		u32 key0 = span.base() + step * STEP<D>;
		u32 const n_hi = span.length(p.n_tokens - 1);

#pragma unroll 1
		for (u32 i = 0; i < n_here; ++i) {
			u32 src = ring + stage * SB, src_scales = src + S_AT;
			u32 bad_now = bad >> (stage * RUNS<D>) & ((1u << RUNS<D>) - 1);
			cp_async_wait<0>();
			__syncwarp();
			stage ^= 1;
			if (i + 1 < n_here) {
				u32 const s = step + i + 1;
				if (s * RUNS<D> % 32 == 0) {
					entries = entries_ahead;
					entries_ahead = page_entries(span, b, s * RUNS<D> + 32);
				}
				issue(span, b, kvh, s, entries, stage);
			} else if (left != 0) {
				issue(next_span, next_b, p.chunks(next_x), 0, entries_next, stage);
			}
			u32 const key_end = key0 + STEP<D>;
#pragma unroll 1
			for (u32 part = 0; part < STEP<D> / KS && (part == 0 || key0 < n_hi); ++part, key0 += KS, src += KS * RB, src_scales += KS * 8, bad_now >>= 2) {
				// ---- scores ----
				f32 arg[KS / 8][RT][2];
				f32 vs[KS / 8][2];
#pragma unroll
				for (u32 n8 = 0; n8 < KS / 8; ++n8) {
					u32 kw[KW];
					if constexpr (D == 128) {
						ld_shared_words(src + n8 * 8 * RB + k_at, *reinterpret_cast<u32 (*)[4]>(kw));
						ld_shared_words(src + n8 * 8 * RB + (k_at ^ 16), *reinterpret_cast<u32 (*)[4]>(kw + 4));
					} else {
						ld_shared_words(src + n8 * 8 * RB + k_at, kw);
					}
					i32 c[QT][4];
#pragma unroll
					for (u32 q = 0; q < QT; ++q) {
						mma_s8<true>(c[q], qa[q][0], kw[0], kw[1]);
#pragma unroll
						for (u32 k = 2; k < KW; k += 2) mma_s8<false>(c[q], qa[q][k / 2], kw[k], kw[k + 1]);
					}
					f32 ks[2] = {1.0f, 1.0f};
					if constexpr (SCALED) {
						uint4 const s4 = ld_shared_v4(src_scales + (n8 * 8 + t * 2) * 8);
						ks[0] = __uint_as_float(s4.x);
						ks[1] = __uint_as_float(s4.z);
						vs[n8][0] = __uint_as_float(s4.y);
						vs[n8][1] = __uint_as_float(s4.w);
					}
#pragma unroll
					for (u32 e = 0; e < 2 * RT; ++e) {
						f32 const x = SCALED ? f32(c[e / 4][e % 4]) * ks[e % 2] : f32(c[e / 4][e % 4]);
						arg[n8][e / 2][e % 2] = __fmaf_rn(x, temp[e / 2], neg_m[e / 2]);
					}
				}
				if (key0 < lo_max || key0 + KS > n_min || bad_now != 0) {
#pragma unroll
					for (u32 n8 = 0; n8 < KS / 8; ++n8) {
#pragma unroll
						for (u32 e = 0; e < 2; ++e) {
							u32 const key = key0 + n8 * 8 + t * 2 + e;
							bool seen = false;
#pragma unroll
							for (u32 r = 0; r < RT; ++r) {
								bool const off = key < lo[r] || key >= n[r] || (bad_now >> (n8 / 2) & 1);
								if (off) arg[n8][r][e] = __uint_as_float(NEG_INF);
								seen |= !off;
							}
							if (!seen) vs[n8][e] = 0.0f;   // (what lies there may be anything)
						}
					}
				}
				// ---- the maximum, when a score has passed it ----
				f32 top[RT];
				bool passed = false;
#pragma unroll
				for (u32 r = 0; r < RT; ++r) {
					top[r] = arg[0][r][0];
#pragma unroll
					for (u32 n8 = 0; n8 < KS / 8; ++n8) top[r] = fmaxf(top[r], fmaxf(arg[n8][r][0], arg[n8][r][1]));
					passed |= top[r] > ARG_MAX;
				}
				if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
					for (u32 r = 0; r < RT; ++r) {
						top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
						top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
						f32 const up = fmaxf(top[r] - SHIFT, 0.0f), a = ex2_approx(-up);
						f32 const a0 = __shfl_sync(0xffffffffu, a, t * 8), a1 = __shfl_sync(0xffffffffu, a, t * 8 + 4);
						neg_m[r] -= up;
						sum[r] *= a;
#pragma unroll
						for (u32 n8 = 0; n8 < KS / 8; ++n8) {
							arg[n8][r][0] -= up;
							arg[n8][r][1] -= up;
						}
#pragma unroll
						for (u32 j = 0; j < D / 16; ++j) {
							o[j][r][0] *= a0;
							o[j][r][1] *= a1;
							o[j][r][2] *= a0;
							o[j][r][3] *= a1;
						}
					}
				}
				// ---- weights and values ----
#pragma unroll
				for (u32 j = 0; j < 2; ++j) {
					u32 hi[RT][2], low[RT][2];
#pragma unroll
					for (u32 h = 0; h < 2; ++h) {
#pragma unroll
						for (u32 r = 0; r < RT; ++r) {
							f32 e0 = ex2_approx(arg[2 * j + h][r][0]), e1 = ex2_approx(arg[2 * j + h][r][1]);
							sum[r] += e0 + e1;
							f32 h0, h1;
							if constexpr (SCALED) {
								e0 *= vs[2 * j + h][0];
								e1 *= vs[2 * j + h][1];
								hi[r][h] = cvt_bf16x2(e0, e1);
								h0 = __uint_as_float(hi[r][h] << 16);
								h1 = __uint_as_float(hi[r][h] & 0xFFFF0000u);
								low[r][h] = cvt_bf16x2(e0 - h0, e1 - h1);
							} else {
								hi[r][h] = f32x2_to_f16x2(e0, e1);
								f16x2_values(hi[r][h], h0, h1);
								low[r][h] = f32x2_to_f16x2(e0 - h0, e1 - h1);
							}
						}
					}
					u32 const v0 = src + j * 16 * RB + v_at[0], v1 = src + j * 16 * RB + v_at[1];
					u32 va[VW], vb[VW], vc[VW], vd[VW];
					ld_shared_words(v0, va);
					ld_shared_words(v1, vb);
					ld_shared_words(v0 + 8 * RB, vc);
					ld_shared_words(v1 + 8 * RB, vd);
#pragma unroll
					for (u32 k = 0; k < VW; ++k) {
						u32 const v[2][4] = {{codes_to_x2<SCALED, 0>(va[k], vb[k]), codes_to_x2<SCALED, 1>(va[k], vb[k]), codes_to_x2<SCALED, 0>(vc[k], vd[k]),
											  codes_to_x2<SCALED, 1>(vc[k], vd[k])},
											 {codes_to_x2<SCALED, 2>(va[k], vb[k]), codes_to_x2<SCALED, 3>(va[k], vb[k]), codes_to_x2<SCALED, 2>(vc[k], vd[k]),
											  codes_to_x2<SCALED, 3>(vc[k], vd[k])}};
#pragma unroll
						for (u32 r = 0; r < RT; ++r) {
							if constexpr (SUMS) {
								// sums of 16 keys, low parts first: the product's own addition to a long sum rounds toward zero
#pragma unroll
								for (u32 h = 0; h < 2; ++h) {
									f32 c[4];
									mma_values<SCALED, true>(c, v[h], low[r][0], low[r][1]);
									mma_values<SCALED, false>(c, v[h], hi[r][0], hi[r][1]);
#pragma unroll
									for (u32 e = 0; e < 4; ++e) o[2 * k + h][r][e] += c[e];
								}
							} else {
#pragma unroll
								for (u32 h = 0; h < 2; ++h) mma_values<SCALED, false>(o[2 * k + h][r], v[h], low[r][0], low[r][1]);
#pragma unroll
								for (u32 h = 0; h < 2; ++h) mma_values<SCALED, false>(o[2 * k + h][r], v[h], hi[r][0], hi[r][1]);
							}
						}
					}
				}
			}
			key0 = key_end;
		}
		// ---- out, where the run had all steps; else a part: of the run's beginning to scratch memory, of its end to the ring ----
		step += n_here;
		bool const began = step == n_here, ended = step == steps, whole = p.splits == 0 && began && ended, at_end = left == 0;
		__syncwarp();
		if (lane == 0) {
			if (began && p.splits == 0) {
				u32 const last = start + n_units - left - n_here + steps - 1;
				scratch.shared_by[u64(b) * n_x + x] = make_uint2(blockIdx.x, runs.cta(last) - blockIdx.x + 1);
			}
			if (!whole) items[warp * 2 + at_end] = make_uint2(b * n_x + x, THERE | (began ? BEGAN : 0u) | (ended ? ENDED : 0u));
		}
		constexpr f32 unit = SCALED ? 1.0f : 0.125f;
#pragma unroll
		for (u32 r = 0; r < RT; ++r) {
			sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
			sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
#pragma unroll
			for (u32 e = 0; e < 2; ++e) {
				u32 const lane_of = (2 * t + e) * 4, at = r * ROWS + 2 * t + e;
				f32 const m_r = -__shfl_sync(0xffffffffu, neg_m[r], lane_of), s_r = __shfl_sync(0xffffffffu, sum[r], lane_of);
				f32 const sink_r = __shfl_sync(0xffffffffu, sink[r], lane_of);
				if (at < rows) {
					f32 v[VD];
#pragma unroll
					for (u32 j = 0; j < D / 16; ++j) {
						v[2 * j] = o[j][r][e] * unit;
						v[2 * j + 1] = o[j][r][e + 2] * unit;
					}
					if (whole) {
						u32 const row = row0 + at, tok = p.group(row);
						paged_finish<D, VD>(p, u64(b) * p.n_tokens + tok, kvh * group + row - tok * group, g * VD, m_r, s_r, v, sink_r);
					} else {
						u64 const slot = u64(w) * p.chunk_rows + at;
						f32 *dst = at_end ? reinterpret_cast<f32 *>(smem + warp * STAGES * SB) + at * D : scratch.o + slot * D;
#pragma unroll
						for (u32 j = 0; j < VD; j += 4) *reinterpret_cast<float4 *>(dst + g * VD + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
						if (g == 0) *(at_end ? end_ms(warp) + at : scratch.ms + slot) = make_float4(m_r, s_r, sink_r, 0.0f);
					}
				}
			}
		}
		step = 0;
		b = next_b;
		x = next_x;
		span = next_span;
		steps = span.steps(p.n_tokens);
		entries = entries_next;
		if (left != 0) entries_ahead = page_entries(span, b, 32);
	}

	// ---- what the CTA's warps share ----
	__syncthreads();
	if (p.splits != 0) {
		u32 const kvh = p.chunks(blockIdx.x), row0 = (blockIdx.x - kvh * p.chunks.d) * p.chunk_rows;
		u32 const rows = min(p.chunk_rows, group * p.n_tokens - row0);
		struct Place {
			u32 r, d, head;
			u64 out_row;
		};
		auto place = [&](u32 at) {
			u32 const r = at / (D / 4), row = row0 + r, tok = p.group(row);
			return Place{r, at % (D / 4) * 4, kvh * group + row - tok * group, u64(blockIdx.y) * p.n_tokens + tok};
		};
		auto join_warps = [&](Place const &at, float4 &ms, float4 &v) {
			ms = make_float4(NO_PART, 0.0f, 0.0f, 0.0f);
			v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
			paged_join(ms, v, warps, [&](u32 k, bool of_ms) {
				return of_ms ? end_ms(k)[at.r] : *reinterpret_cast<float4 const *>(reinterpret_cast<f32 const *>(smem + k * STAGES * SB) + at.r * D + at.d);
			});
		};
		auto finish = [&](Place const &at, float4 ms, float4 v, u32 sink_v) {
			f32 out[4] = {v.x, v.y, v.z, v.w};
			u32 const sv[1] = {sink_v};
			paged_finish<D, 4>(p, at.out_row, at.head, at.d, ms.x, ms.y, out, ms.z, sv);
		};
		auto sink_values = [&](Place const &at) { return *reinterpret_cast<u32 const *>(p.sink_v + u64(at.head) * D + at.d); };
		if (p.splits == 1) {
			pdl_launch_dependents();
			for (u32 i = threadIdx.x; i < rows * (D / 4); i += blockDim.x) {
				Place const at = place(i);
				u32 const sv = sink_values(at);
				float4 ms, v;
				join_warps(at, ms, v);
				finish(at, ms, v, sv);
			}
			return;
		}
		// The CTAs of a cluster: their parts go to the first one's shared memory, [splits][rows][D + 4], in place of its ring.
		static_assert(MAX_SPLITS * RT * ROWS * (D + 4) * 4 <= SM_WARPS<D, RT> * RING_BYTES<D, SCALED>);
		constexpr u32 MINE = (RT * ROWS * (D / 4) + SM_WARPS<D, RT> * 32 - 1) / (SM_WARPS<D, RT> * 32);   // (clusters' CTAs have all warps)
		float4 ms[MINE], v[MINE];
		u32 sv[MINE];
#pragma unroll
		for (u32 c = 0; c < MINE; ++c) {
			Place const at = place(threadIdx.x + c * blockDim.x);
			if (at.r < rows) {
				sv[c] = sink_values(at);
				join_warps(at, ms[c], v[c]);
			}
		}
		pdl_launch_dependents();   // not earlier: a next call's clusters would be packed onto the few SMs with room
		cluster_arrive();
		cluster_wait();            // every CTA runs, and has read its ring
		u32 const to = map_to_cta(smem_u32(smem) + blockIdx.z * rows * (D + 4) * 4, 0);
#pragma unroll
		for (u32 c = 0; c < MINE; ++c) {
			Place const at = place(threadIdx.x + c * blockDim.x);
			if (at.r < rows) {
				st_cluster_f32x4(to + (at.r * (D + 4) + at.d) * 4, v[c]);
				if (at.d == 0) st_cluster_f32x4(to + (at.r * (D + 4) + D) * 4, ms[c]);
			}
		}
		__syncwarp();
		cluster_arrive();          // this CTA's part is stored
		if (blockIdx.z != 0) return;
		cluster_wait();
#pragma unroll
		for (u32 c = 0; c < MINE; ++c) {
			Place const at = place(threadIdx.x + c * blockDim.x);
			if (at.r < rows) {
				paged_join(ms[c], v[c], p.splits - 1, [&](u32 z, bool of_ms) {
					return *reinterpret_cast<float4 const *>(reinterpret_cast<f32 const *>(smem) + ((z + 1) * rows + at.r) * (D + 4) + (of_ms ? D : at.d));
				});
				finish(at, ms[c], v[c], sv[c]);
			}
		}
		return;
	}
	// (a CTA of the list has WARPS warps)
#pragma unroll 1
	for (u32 i = 0; i < WARPS * 2;) {
		uint2 const first = items[i];
		if (!(first.y & THERE)) {
			++i;
			continue;
		}
		u32 mine = 0, last = i;   // the items of this (sequence, x): bit by item
#pragma unroll
		for (u32 k = 0; k < WARPS * 2; ++k) {
			uint2 const item = items[k];
			if ((item.y & THERE) && item.x == first.x && k >= i) {
				mine |= 1u << k;
				last = k;
			}
		}
		bool const began = first.y & BEGAN, whole = began && (items[last].y & ENDED);
		u32 const seq = first.x / n_x, x_of = first.x - seq * n_x, kvh = p.chunks(x_of), row0 = (x_of - kvh * p.chunks.d) * p.chunk_rows;
		u32 const rows = min(p.chunk_rows, group * p.n_tokens - row0);
		for (u32 at = threadIdx.x; at < rows * (D / 4); at += WARPS * 32) {
			u32 const r = at / (D / 4), d = at % (D / 4) * 4;
			u32 const row = row0 + r, tok = p.group(row), head = kvh * group + row - tok * group;
			u32 const sink_v[1] = {*reinterpret_cast<u32 const *>(p.sink_v + u64(head) * D + d)};
			// everything is on its way before any of it is used
			float4 ms[WARPS * 2], part[WARPS * 2];
#pragma unroll
			for (u32 k = 0; k < WARPS * 2; ++k) {
				ms[k] = make_float4(NO_PART, 0.0f, 0.0f, 0.0f);
				part[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				if (mine >> k & 1) {
					u64 const slot = u64(blockIdx.x * WARPS + k / 2) * p.chunk_rows + r;
					ms[k] = k & 1 ? end_ms(k / 2)[r] : scratch.ms[slot];
					part[k] = *reinterpret_cast<float4 const *>(
						(k & 1 ? reinterpret_cast<f32 const *>(smem + k / 2 * STAGES * SB) + r * D : scratch.o + slot * D) + d);
				}
			}
			float4 all = make_float4(NO_PART, 0.0f, 0.0f, 0.0f), v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
			for (u32 k = 0; k < WARPS * 2; ++k) all.x = fmaxf(all.x, ms[k].x);
#pragma unroll
			for (u32 k = 0; k < WARPS * 2; ++k) {
				f32 const e = ex2_approx(ms[k].x - all.x);
				v.x = __fmaf_rn(part[k].x, e, v.x);
				v.y = __fmaf_rn(part[k].y, e, v.y);
				v.z = __fmaf_rn(part[k].z, e, v.z);
				v.w = __fmaf_rn(part[k].w, e, v.w);
				all.y = __fmaf_rn(ms[k].y, e, all.y);
				if (mine >> k & 1) all.z = ms[k].z;   // (the same in every part)
			}
			if (whole) {
				f32 out[4] = {v.x, v.y, v.z, v.w};
				paged_finish<D, 4>(p, u64(seq) * p.n_tokens + tok, head, d, all.x, all.y, out, all.z, sink_v);
			} else {
				u64 const slot = (u64(n_warps) + blockIdx.x * 2 + began) * p.chunk_rows + r;
				*reinterpret_cast<float4 *>(scratch.o + slot * D + d) = v;
				if (d == 0) scratch.ms[slot] = all;
			}
		}
		i = last + 1;
	}
}

// Joins the parts of a (sequence, x): `cta_rows` of its rows to a CTA (1, 2, 4 or 8), as many warps to a row as that leaves, each
// every so manyth part; a lane D / 32 dims.
template <u32 D>
__global__ void __launch_bounds__(paged_cfg::MERGE_WARPS * 32)
paged_merge_kernel(const PagedDecodeParams p, const PagedScratch scratch, const u32 first_slot, const u32 cta_rows) {
	using namespace paged_cfg;
	constexpr u32 V = D / 32, W = MERGE_WARPS;
	__shared__ f32 sh_o[W][D], sh_m[W], sh_s[W];
	u32 const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	u32 const n_x = p.n_x;
	u32 const b = blockIdx.x / n_x, x = blockIdx.x - b * n_x;
	u32 const group = p.group.d;
	u32 const kvh = p.chunks(x), row0 = (x - kvh * p.chunks.d) * p.chunk_rows;
	u32 const r = blockIdx.y * cta_rows + warp % cta_rows, row = row0 + r;
	u32 const mine = warp / cta_rows, shares = W / cta_rows;
	pdl_launch_dependents();
	pdl_wait();
	uint2 const by = scratch.shared_by[blockIdx.x];
	if (by.y < 2) return;
	bool const live = r < p.chunk_rows && row < group * p.n_tokens;
	// part k is slot [1] of the first CTA, slot [0] of the others
	auto slot = [&](u32 k) { return (u64(first_slot) + (by.x + k) * 2 + (k == 0)) * p.chunk_rows + r; };
	u32 const tok = p.group(row), head = kvh * group + row - tok * group;
	f32 sink = 0.0f;
	u32 sink_v[1] = {};
	if (live && mine == 0 && lane < D / 4) {
		sink = scratch.ms[slot(0)].z;
		sink_v[0] = reinterpret_cast<u32 const *>(p.sink_v + u64(head) * D)[lane];
	}
	f32 m = -3.0e38f, s = 0.0f;
	__align__(16) f32 v[V] = {};
	constexpr u32 AHEAD = 8;
	for (u32 k0 = mine; live && k0 < by.y; k0 += shares * AHEAD) {
		float2 ms[AHEAD];
		__align__(16) f32 part[AHEAD][V];
#pragma unroll
		for (u32 i = 0; i < AHEAD; ++i) {
			u32 const k = k0 + i * shares;
			ms[i] = make_float2(-3.0e38f, 0.0f);
			if (k < by.y) {
				u64 const at = slot(k);
				ms[i] = *reinterpret_cast<float2 const *>(scratch.ms + at);
				f32 const *src = scratch.o + at * D + lane * V;
				if constexpr (V == 4) *reinterpret_cast<float4 *>(part[i]) = *reinterpret_cast<float4 const *>(src);
				else if constexpr (V == 2) *reinterpret_cast<float2 *>(part[i]) = *reinterpret_cast<float2 const *>(src);
				else part[i][0] = *src;
			} else {
#pragma unroll
				for (u32 j = 0; j < V; ++j) part[i][j] = 0.0f;
			}
		}
		f32 up = m;
#pragma unroll
		for (u32 i = 0; i < AHEAD; ++i) up = fmaxf(up, ms[i].x);
		f32 const a = ex2_approx(m - up);
		s *= a;
#pragma unroll
		for (u32 j = 0; j < V; ++j) v[j] *= a;
		m = up;
#pragma unroll
		for (u32 i = 0; i < AHEAD; ++i) {
			f32 const e = ex2_approx(ms[i].x - m);
			s = __fmaf_rn(ms[i].y, e, s);
#pragma unroll
			for (u32 j = 0; j < V; ++j) v[j] = __fmaf_rn(part[i][j], e, v[j]);
		}
	}
#pragma unroll
	for (u32 j = 0; j < V; ++j) sh_o[warp][lane * V + j] = v[j];
	if (lane == 0) {
		sh_m[warp] = m;
		sh_s[warp] = s;
	}
	__syncthreads();
	if (!live || mine != 0 || lane >= D / 4) return;
	f32 out[4] = {};
	s = 0.0f;
	for (u32 k = warp; k < W; k += cta_rows) m = fmaxf(m, sh_m[k]);
	for (u32 k = warp; k < W; k += cta_rows) {
		f32 const a = ex2_approx(sh_m[k] - m);
		s = __fmaf_rn(sh_s[k], a, s);
#pragma unroll
		for (u32 j = 0; j < 4; ++j) out[j] = __fmaf_rn(sh_o[k][lane * 4 + j], a, out[j]);
	}
	paged_finish<D, 4>(p, u64(b) * p.n_tokens + tok, head, lane * 4, m, s, out, sink, sink_v);
}

}  // namespace x17
