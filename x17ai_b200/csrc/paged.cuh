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
	// row of (page, head, slot)
	X17_DEV u64 row(u32 page, u32 head, u32 slot) const { return ((u64(page) * n_kv_heads + head) << page_shift) + slot; }
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
	bool adjacent;          // pairs (2 i, 2 i + 1); otherwise (i, i + rotary / 2)
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
	u32 chunk_rows, chunks; // rows (query heads of a group x new tokens) of a CTA, CTAs that a key head's rows take
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

// One warp per token and head (query heads, then key and value heads). FixedI8: x' = (x cos - y sin + 2^13) >> 14 in integers.
// Scaled: x' in f32 (bf16 times a 15-bit table value is exact), code = rint(x' * (127 / absmax)).
template <u32 D, bool SCALED>
__global__ void __launch_bounds__(128)
paged_append_kernel(const PagedAppendParams p) {
	pdl_launch_dependents();
	pdl_wait();
	constexpr u32 V = D / 32;
	u32 const lane = threadIdx.x & 31;
	u32 const n_q = p.q == nullptr ? 0u : p.n_heads;
	u32 const per_token = n_q + 2 * p.pool.n_kv_heads;
	u64 const item = u64(blockIdx.x) * 4 + (threadIdx.x >> 5);
	if (item >= u64(p.tokens) * per_token) return;
	u32 const token = u32(item / per_token), head = u32(item % per_token);
	i32 const seq = p.seqs[token], pos = p.positions[token];
	if (seq < 0) return;
	u32 page = 0, slot = 0;
	if (!paged_slot(p.pool, seq, pos, page, slot) || (p.rotary != 0 && u32(pos) >= p.rope_rows)) {
		if (lane == 0) report_status(p.status, ST_BAD_INDEX, token);
		return;
	}
	bool const is_q = head < n_q;
	u32 const kvh = is_q ? 0u : (head - n_q) / 2;
	bool const is_v = !is_q && ((head - n_q) & 1);
	u64 const src = is_q ? token * p.q_stride + head * D : token * p.kv_stride + (u64(kvh) * 2 + is_v) * D;
	auto load = [&](u32 d) -> f32 {
		void const *base = is_q ? p.q : p.kv;
		if constexpr (SCALED) return __uint_as_float(u32(static_cast<u16 const *>(base)[src + d]) << 16);
		else return f32(static_cast<i8 const *>(base)[src + d]);
	};
	u32 const half = p.rotary / 2;
	f32 val[V];
	f32 top = 0.0f;
#pragma unroll
	for (u32 j = 0; j < V; ++j) {
		u32 const d = j * 32 + lane;
		val[j] = load(d);
		if (!is_v && d < p.rotary) {
			u32 const pair = p.adjacent ? d / 2 : d % half;
			bool const second = p.adjacent ? d & 1 : d >= half;
			f32 const other = load(p.adjacent ? d ^ 1u : second ? d - half : d + half);
			int16_t const *cs = p.rope + (u64(u32(pos)) * half + pair) * 2;
			if constexpr (SCALED) {
				f32 const c = f32(cs[0]) * 0x1p-14f, s = f32(cs[1]) * 0x1p-14f;
				val[j] = second ? __fmaf_rn(other, s, __fmul_rn(val[j], c)) : __fmaf_rn(val[j], c, -__fmul_rn(other, s));
			} else {
				i32 const x = i32(val[j]), y = i32(other);
				i32 const acc = second ? y * cs[1] + x * cs[0] : x * cs[0] - y * cs[1];
				val[j] = f32(max(-127, min(127, (acc + 8192) >> 14)));
			}
		}
		top = fmaxf(top, fabsf(val[j]));
	}
	f32 inv = 1.0f;
	f32 scale = 0.0f;
	if constexpr (SCALED) {
#pragma unroll
		for (u32 mask = 16; mask > 0; mask >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, mask));
		bool const live = top > PAGED_TINY;
		inv = live ? __fdiv_rn(127.0f, top) : 0.0f;
		scale = live ? __fmul_rn(top, 1.0f / 127.0f) : 0.0f;
		if (lane == 0) {
			if (is_q) p.q_scale[u64(token) * p.n_heads + head] = scale;
			else p.pool.scales[p.pool.row(page, kvh, slot) * 2 + is_v] = scale;
		}
	}
#pragma unroll
	for (u32 j = 0; j < V; ++j) {
		u32 const d = j * 32 + lane;
		i8 const code = SCALED ? i8(f32_to_fixedi8(__fmul_rn(val[j], inv))) : i8(i32(val[j]));
		if (is_q) {
			p.q_out[token * p.q_stride + head * D + d] = code;
		} else {
			p.pool.pages[p.pool.row(page, kvh, slot) * 2 * D + is_v * D + d] = code;
			if (p.kv_out != nullptr) p.kv_out[src + d] = code;
		}
	}
}

// ---- decode ------------------------------------------------------------------------------------
//
// A pass over a cache is bound by HBM: the kernel's job is to keep enough bytes in flight and to stay out of their way. One
// CTA works on the rows (query heads of a group, times new tokens; eight at most) that share a key head, so a key is read
// once for all of them; up to 16 CTAs (a cluster) share a sequence's keys, four warps a CTA's. A warp takes 16 or 32 keys a
// step (4 KB) out of a ring of its own in shared memory that it fills itself, three steps ahead, with cp.async: no barrier
// among warps until the end. A page of a head is one run of memory and a step's page is known long before (32 entries of the page table
// sit in a warp's lanes), so pages cost no more than a contiguous cache.
//
// Scores: mma m16n8k32 (s8 x s8 -> s32, exact), rows as its M, keys as its N; a lane's bytes of a key row are consecutive, the
// query's are permuted the same way. Values: mma m16n8k16 (f16 x f16 -> f32) with V transposed as its first operand (dims as M)
// and the weights as the second (rows as N), which is how the scores' fragments lie; accumulators are a lane's 16 dims of two rows.
// Weights keep 22 bits: e = hi + lo in f16, two products into the same sums. V's codes are exact in f16 (integer added to 1024 as
// bits). Weights are 2^(x - m + 8) against a maximum m that moves only when a score passes it by 6: between 2^-38 and 2^14 of
// m's nothing is lost to f16's range. m starts at the sink's score, so no key and no row leaves it undefined.

namespace paged_cfg {
constexpr u32 WARPS = 4, THREADS = WARPS * 32;
#ifndef PG_STAGES
#define PG_STAGES 4
#endif
#ifndef PG_CTAS
#define PG_CTAS 3
#endif
#ifndef PG_KEYS
#define PG_KEYS 16
#endif
constexpr u32 STAGES = PG_STAGES;
constexpr u32 ROWS = 8;          // rows of a CTA
constexpr u32 MAX_SPLITS = 16;   // CTAs of a cluster
constexpr f32 SHIFT = 8.0f, ARG_MAX = 14.0f;   // weights are 2^(x - m + SHIFT), at most 2^ARG_MAX (f16 ends below 2^16)
template <u32 D>
constexpr u32 KEYS = D == 128 ? PG_KEYS : 32;       // of a step
template <u32 D>
constexpr u32 ROW_BYTES = 2 * D + 16;          // of a key in the ring: rows 16 bytes off each other's banks
template <u32 D, bool SCALED>
constexpr u32 STAGE_BYTES = KEYS<D> * (ROW_BYTES<D> + (SCALED ? 8 : 0));
template <u32 D, bool SCALED>
constexpr u32 RING_BYTES = WARPS * STAGES * STAGE_BYTES<D, SCALED>;
// the parts of a cluster's CTAs, in the first one: [splits][rows][D + 2] f32
template <u32 D>
constexpr u32 part_bytes(u32 splits, u32 rows) {
	return splits > 1 ? splits * rows * (D + 2) * 4 : 0;
}
}  // namespace paged_cfg

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
// c[0], c[1]: row lane / 4, columns 2 (lane % 4) and the next one; rows 8-15 of A are zero, their sums are not kept
X17_DEV void mma_s8(i32 (&c)[2], u32 a0, u32 a2, u32 b0, u32 b1) {
	i32 unused2, unused3;
	asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %5}, {%7, %8}, {%9, %10, %5, %5};"
		: "=r"(c[0]), "=r"(c[1]), "=r"(unused2), "=r"(unused3)
		: "r"(a0), "r"(0), "r"(a2), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]));
}
X17_DEV void mma_f16(f32 (&c)[4], u32 const (&a)[4], u32 b0, u32 b1) {
	asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
		: "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
X17_DEV u32 f32x2_to_f16x2(f32 lo, f32 hi) {
	u32 r;
	asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
	return r;
}
X17_DEV void f16x2_values(u32 h2, f32 &lo, f32 &hi) {
	asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h2));
}
// byte J of a and of b, signed, as f16x2: the bits 0x6400 + (code + 128) are 1024 + 128 + code
template <u32 J>
X17_DEV u32 codes_to_f16x2(u32 a, u32 b) {
	u32 const t = (__byte_perm(a, b, (J + 4) << 8 | J) & 0x00FF00FFu) ^ 0x64806480u;
	u32 r;
	asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(0xE480E480u));
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

// One output: the keys' (m, s, v), m being a maximum less SHIFT that is no smaller than the sink's, with the sink token.
template <u32 D>
X17_DEV void paged_finish(PagedDecodeParams const &p, u32 b, u32 kvh, u32 row0, u32 r, u32 d, f32 m, f32 s, f32 v, f32 sink) {
	u32 const group = p.n_heads / p.pool.n_kv_heads;
	u32 const row = row0 + r, head = kvh * group + row % group;
	u64 const out_row = u64(b) * p.n_tokens + row / group;
	f32 const a = ex2_approx(sink - m + paged_cfg::SHIFT);
	s += a;
	v = __fmaf_rn(f32(p.sink_v[u64(head) * D + d]) * 0.125f, a, v);
	v = __fdiv_rn(v, s);
	u64 const at = out_row * p.o_stride + head * D + d;
	if (p.out_i8) static_cast<i8 *>(p.out)[at] = i8(f32_to_fixedi8(v * 8.0f));
	else static_cast<u16 *>(p.out)[at] = u16(cvt_bf16x2(v, 0.0f));
	if (d == 0 && p.l != nullptr) p.l[out_row * p.n_heads + head] = log2f(255.0f * s) + m;
}

// Grid (key head and chunk of rows, sequence, split); the splits of one (x, y) are a cluster.
template <u32 D, bool SCALED>
__global__ void __launch_bounds__(paged_cfg::THREADS, PG_CTAS)
paged_decode_kernel(const PagedDecodeParams p) {
	using namespace paged_cfg;
	constexpr u32 KS = KEYS<D>, SUBS = KS / 16;      // a step's runs of 16 keys lie in one page each
	constexpr u32 KW = D / 16;                       // words of a key row that a lane holds
	constexpr u32 VW = D / 32;                       // words of a value row that a lane holds
	constexpr u32 RB = ROW_BYTES<D>;
	constexpr u32 NEG_INF = 0xFF800000u;
	extern __shared__ __align__(16) u8 smem[];
	__shared__ f32 sh_sink[ROWS], sh_m[WARPS][ROWS], sh_s[WARPS][ROWS];
	u32 const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	u32 const g = lane >> 2, t = lane & 3;
	u32 const splits = gridDim.z;

	if (splits > 1) cluster_arrive();   // "this CTA runs"
	pdl_wait();
	u32 const group = p.n_heads / p.pool.n_kv_heads;
	u32 const kvh = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks, b = blockIdx.y;
	u32 const n_rows_all = group * p.n_tokens;
	u32 const row0 = chunk * p.chunk_rows;
	u32 const rows = min(p.chunk_rows, n_rows_all - row0);
	i32 const len = p.kv_lens[b];

	// this lane's row: a head of the group for one of the new tokens (rows behind the last one repeat it and are not stored)
	u32 const my_row = row0 + min(g, rows - 1);
	u32 const tok = my_row / group, head = kvh * group + my_row % group;
	u64 const q_row = u64(b) * p.n_tokens + tok;
	u32 qw[KW], skw[KW];
	ld_global_words(p.q + q_row * p.q_stride + head * D + t * (D / 4), qw);
	ld_global_words(p.sink_k + u64(head) * D + t * (D / 4), skw);
	f32 temp = p.temperature[head];
	if constexpr (SCALED) temp *= p.q_scale[q_row * p.n_heads + head];

	u32 const capacity = p.pool.max_pages << p.pool.page_shift;
	auto length = [&](u32 tk) { return min(u32(max(len, 0)) + tk, capacity); };
	auto first = [&](u32 n) { return n - min(n, p.window); };
	u32 const tok_lo = row0 / group, tok_hi = (row0 + rows - 1) / group;
	u32 const n = length(tok), lo = first(n);                       // of this lane's row
	u32 const n_hi = length(tok_hi), lo_all = first(length(tok_lo));   // the union of the rows' keys: [lo_all, n_hi)
	u32 const n_min = length(tok_lo), lo_max = first(n_hi);            // what every row sees: [lo_max, n_min)

	// the CTA's steps of KS keys from `base` on, dealt out to its warps in turn
	u32 const base = lo_all & ~15u;
	u32 const n_steps = n_hi > base ? (n_hi - base + KS - 1) / KS : 0;
	u32 const per_cta = (n_steps + splits - 1) / splits;
	u32 const step_lo = min(blockIdx.z * per_cta, n_steps), step_hi = min(step_lo + per_cta, n_steps);
	u32 const n_own = step_hi - step_lo > warp ? (step_hi - step_lo - warp + WARPS - 1) / WARPS : 0;

	u32 const ring = smem_u32(smem) + warp * STAGES * STAGE_BYTES<D, SCALED>;
	u32 bad = 0;                       // bit stage * SUBS + sub: that run's page is none
	u32 page_now = 0, page_next = 0;   // page table entries of the warp's runs, one a lane
	auto run_key = [&](u32 run) { return base + ((step_lo + warp + run / SUBS * WARPS) * SUBS + run % SUBS) * 16; };
	auto page_entry = [&](u32 run) -> u32 {
		u32 const key = run_key(run);
		return run < n_own * SUBS && key < n_hi ? u32(p.pool.table[u64(b) * p.pool.max_pages + (key >> p.pool.page_shift)]) : 0u;
	};
	page_next = page_entry(lane);
	auto issue = [&](u32 i) {
		if (i < n_own) {
			u32 const stage = i % STAGES, dst0 = ring + stage * STAGE_BYTES<D, SCALED>;
			if (i * SUBS % 32 == 0) {
				page_now = page_next;
				page_next = page_entry(i * SUBS + 32 + lane);
			}
#pragma unroll
			for (u32 j = 0; j < SUBS; ++j) {
				u32 const page = __shfl_sync(0xffffffffu, page_now, (i * SUBS + j) & 31);
				u32 const key = run_key(i * SUBS + j);
				u32 const bit = 1u << (stage * SUBS + j);
				bool const ok = page < p.pool.n_pages;
				bad = ok ? bad & ~bit : bad | bit;
				if (!ok) {
					if (lane == 0 && key < n_hi) report_status(p.status, ST_BAD_INDEX, b);
				} else if (key < n_hi) {
					u64 const row = p.pool.row(page, kvh, key & ((1u << p.pool.page_shift) - 1));
					i8 const *src = p.pool.pages + row * 2 * D;
					constexpr u32 CHUNKS = 2 * D / 16;   // of a row
#pragma unroll
					for (u32 c = 0; c < CHUNKS / 2; ++c) {
						u32 const at = c * 32 + lane;
						cp_async_16(dst0 + (j * 16 + at / CHUNKS) * RB + at % CHUNKS * 16, src + at * 16);
					}
					if constexpr (SCALED) {
						if (lane < 16) cp_async_8(dst0 + KS * RB + (j * 16 + lane) * 8, p.pool.scales + (row + lane) * 2);
					}
				}
			}
		}
		cp_async_commit();
	};
#pragma unroll
	for (u32 i = 0; i + 1 < STAGES; ++i) issue(i);

	// temperature D^-1/2 log2(min(W', n) + 4) temp_h, times the scales that are not the key's
	constexpr f32 ROOT = f32(D == 128 ? 0.08838834764831845 : D == 64 ? 0.125 : 0.17677669529663687);
	temp *= ROOT * log2f(f32(n - lo + 4)) * (SCALED ? 1.0f : 0.015625f);
	i32 dot = 0;
#pragma unroll
	for (u32 i = 0; i < KW; ++i) dot = __dp4a(i32(qw[i]), i32(skw[i]), dot);
	dot += __shfl_xor_sync(0xffffffffu, dot, 1);
	dot += __shfl_xor_sync(0xffffffffu, dot, 2);
	f32 const sink = f32(dot) * (SCALED ? temp * 0.125f : temp);
	f32 neg_m = SHIFT - sink, sum = 0.0f;
	f32 v_unit = 0.0f, v_inv = 0.0f;   // SCALED: weights carry v_scale / v_unit, a power of two no smaller than any seen
	// tile j: dims g D / 8 + 2 j ([0], [1]) and + 2 j + 1 ([2], [3]) of rows 2 t ([0], [2]) and 2 t + 1 ([1], [3])
	f32 o[D / 16][4];
#pragma unroll
	for (u32 i = 0; i < D / 16; ++i) {
#pragma unroll
		for (u32 j = 0; j < 4; ++j) o[i][j] = 0.0f;
	}

#pragma unroll 1
	for (u32 i = 0; i < n_own; ++i) {
		cp_async_wait<STAGES - 2>();
		__syncwarp();
		issue(i + STAGES - 1);
		u32 const stage = i % STAGES, src = ring + stage * STAGE_BYTES<D, SCALED>;
		u32 const key0 = base + (step_lo + warp + i * WARPS) * KS;
		// ---- scores ----
		f32 arg[KS / 8][2];
		f32 vs[KS / 8][2];
#pragma unroll
		for (u32 n8 = 0; n8 < KS / 8; ++n8) {
			u32 kw[KW];
			ld_shared_words(src + (n8 * 8 + g) * RB + t * (D / 4), kw);
			i32 c[2] = {0, 0};
#pragma unroll
			for (u32 k = 0; k < KW; k += 2) mma_s8(c, qw[k], qw[k + 1], kw[k], kw[k + 1]);
			if constexpr (SCALED) {
				uint4 const s4 = ld_shared_v4(src + KS * RB + (n8 * 8 + t * 2) * 8);
				arg[n8][0] = __fmaf_rn(f32(c[0]) * __uint_as_float(s4.x), temp, neg_m);
				arg[n8][1] = __fmaf_rn(f32(c[1]) * __uint_as_float(s4.z), temp, neg_m);
				vs[n8][0] = __uint_as_float(s4.y);
				vs[n8][1] = __uint_as_float(s4.w);
			} else {
				arg[n8][0] = __fmaf_rn(f32(c[0]), temp, neg_m);
				arg[n8][1] = __fmaf_rn(f32(c[1]), temp, neg_m);
			}
		}
		u32 const bad_now = bad >> (stage * SUBS) & ((1u << SUBS) - 1);
		if (key0 < lo_max || key0 + KS > n_min || bad_now != 0) {
#pragma unroll
			for (u32 n8 = 0; n8 < KS / 8; ++n8) {
#pragma unroll
				for (u32 e = 0; e < 2; ++e) {
					u32 const key = key0 + n8 * 8 + t * 2 + e;
					if (key < lo || key >= n || (bad_now >> (n8 / 2) & 1)) {
						arg[n8][e] = __uint_as_float(NEG_INF);
						vs[n8][e] = 0.0f;   // (what lies there may be anything)
					}
				}
			}
		}
		// ---- the maximum, when a score has passed it ----
		f32 top = arg[0][0];
#pragma unroll
		for (u32 n8 = 0; n8 < KS / 8; ++n8) top = fmaxf(top, fmaxf(arg[n8][0], arg[n8][1]));
		if (__any_sync(0xffffffffu, top > ARG_MAX)) {
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
			top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
			f32 const up = fmaxf(top - SHIFT, 0.0f), a = ex2_approx(-up);
			f32 const a0 = __shfl_sync(0xffffffffu, a, t * 8), a1 = __shfl_sync(0xffffffffu, a, t * 8 + 4);
			neg_m -= up;
			sum *= a;
#pragma unroll
			for (u32 n8 = 0; n8 < KS / 8; ++n8) {
				arg[n8][0] -= up;
				arg[n8][1] -= up;
			}
#pragma unroll
			for (u32 j = 0; j < D / 16; ++j) {
				o[j][0] *= a0;
				o[j][1] *= a1;
				o[j][2] *= a0;
				o[j][3] *= a1;
			}
		}
		if constexpr (SCALED) {
			f32 most = vs[0][0];
#pragma unroll
			for (u32 n8 = 0; n8 < KS / 8; ++n8) most = fmaxf(most, fmaxf(vs[n8][0], vs[n8][1]));
			if (__any_sync(0xffffffffu, most > v_unit)) {
#pragma unroll
				for (u32 mask = 16; mask > 0; mask >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, mask));
				f32 const unit = __uint_as_float(__float_as_uint(fminf(most, 0x1p125f)) & 0x7F800000u) * 2.0f;
				f32 const a = v_unit * __frcp_rn(unit);   // powers of two
				v_unit = unit;
				v_inv = __frcp_rn(unit);
#pragma unroll
				for (u32 j = 0; j < D / 16; ++j) {
#pragma unroll
					for (u32 e = 0; e < 4; ++e) o[j][e] *= a;
				}
			}
		}
		// ---- weights and values ----
#pragma unroll
		for (u32 j = 0; j < SUBS; ++j) {
			u32 hi[2], low[2];
#pragma unroll
			for (u32 h = 0; h < 2; ++h) {
				f32 e0 = ex2_approx(arg[2 * j + h][0]), e1 = ex2_approx(arg[2 * j + h][1]);
				sum += e0 + e1;
				if constexpr (SCALED) {
					e0 *= vs[2 * j + h][0] * v_inv;
					e1 *= vs[2 * j + h][1] * v_inv;
				}
				hi[h] = f32x2_to_f16x2(e0, e1);
				f32 h0, h1;
				f16x2_values(hi[h], h0, h1);
				low[h] = f32x2_to_f16x2(e0 - h0, e1 - h1);
			}
			u32 const v0 = src + (j * 16 + t * 2) * RB + D + g * (D / 8);
			u32 va[VW], vb[VW], vc[VW], vd[VW];
			ld_shared_words(v0, va);
			ld_shared_words(v0 + RB, vb);
			ld_shared_words(v0 + 8 * RB, vc);
			ld_shared_words(v0 + 9 * RB, vd);
#pragma unroll
			for (u32 w = 0; w < VW; ++w) {
				u32 const x[4] = {codes_to_f16x2<0>(va[w], vb[w]), codes_to_f16x2<1>(va[w], vb[w]), codes_to_f16x2<0>(vc[w], vd[w]),
								  codes_to_f16x2<1>(vc[w], vd[w])};
				u32 const y[4] = {codes_to_f16x2<2>(va[w], vb[w]), codes_to_f16x2<3>(va[w], vb[w]), codes_to_f16x2<2>(vc[w], vd[w]),
								  codes_to_f16x2<3>(vc[w], vd[w])};
				mma_f16(o[2 * w], x, hi[0], hi[1]);
				mma_f16(o[2 * w + 1], y, hi[0], hi[1]);
				mma_f16(o[2 * w], x, low[0], low[1]);
				mma_f16(o[2 * w + 1], y, low[0], low[1]);
			}
		}
	}
	cp_async_wait<0>();
	sum += __shfl_xor_sync(0xffffffffu, sum, 1);
	sum += __shfl_xor_sync(0xffffffffu, sum, 2);

	// ---- merge the warps: [warp][row][D] in the ring's place ----
	__syncthreads();
	f32 *parts = reinterpret_cast<f32 *>(smem);
	f32 const unit = SCALED ? v_unit : 0.125f;
#pragma unroll
	for (u32 e = 0; e < 2; ++e) {
		if (2 * t + e < rows) {
			f32 *dst = parts + (warp * ROWS + 2 * t + e) * D + g * (D / 8);
#pragma unroll
			for (u32 j = 0; j < D / 16; j += 2) {
				*reinterpret_cast<float4 *>(dst + 2 * j) =
					make_float4(o[j][e] * unit, o[j][e + 2] * unit, o[j + 1][e] * unit, o[j + 1][e + 2] * unit);
			}
		}
	}
	if (t == 0) {
		sh_m[warp][g] = -neg_m;   // m - SHIFT
		sh_s[warp][g] = sum;
		if (warp == 0) sh_sink[g] = sink - SHIFT;
	}
	__syncthreads();
	if (splits > 1) cluster_wait();   // the first CTA runs (asked for at entry): its shared memory can be written
	f32 *recv = reinterpret_cast<f32 *>(smem + RING_BYTES<D, SCALED>);
	for (u32 at = threadIdx.x; at < rows * D; at += THREADS) {
		u32 const r = at / D, d = at % D;
		f32 m = sh_m[0][r];
#pragma unroll
		for (u32 w = 1; w < WARPS; ++w) m = fmaxf(m, sh_m[w][r]);
		f32 s = 0.0f, v = 0.0f;
#pragma unroll
		for (u32 w = 0; w < WARPS; ++w) {
			f32 const a = ex2_approx(sh_m[w][r] - m);
			s = __fmaf_rn(sh_s[w][r], a, s);
			v = __fmaf_rn(parts[(w * ROWS + r) * D + d], a, v);
		}
		if (splits > 1) {
			u32 const dst = map_to_cta(smem_u32(recv + (blockIdx.z * rows + r) * (D + 2)), 0);
			st_cluster_f32(dst + d * 4, v);
			if (d == 0) {
				st_cluster_f32(dst + D * 4, m);
				st_cluster_f32(dst + D * 4 + 4, s);
			}
		} else {
			paged_finish<D>(p, b, kvh, row0, r, d, m, s, v, sh_sink[r]);
		}
	}
	pdl_launch_dependents();   // not earlier: a next call's clusters would be packed onto the few SMs with room
	if (splits > 1) {
		__syncwarp();
		cluster_arrive();              // this CTA's part is stored
		if (blockIdx.z != 0) return;
		cluster_wait();
		for (u32 at = threadIdx.x; at < rows * D; at += THREADS) {
			u32 const r = at / D, d = at % D;
			f32 m = sh_sink[r], s = 0.0f, v = 0.0f;
			for (u32 z = 0; z < splits; ++z) m = fmaxf(m, recv[(z * rows + r) * (D + 2) + D]);
			for (u32 z = 0; z < splits; ++z) {
				f32 const *part = recv + (z * rows + r) * (D + 2);
				f32 const a = ex2_approx(part[D] - m);
				s = __fmaf_rn(part[D + 1], a, s);
				v = __fmaf_rn(part[d], a, v);
			}
			paged_finish<D>(p, b, kvh, row0, r, d, m, s, v, sh_sink[r]);
		}
	}
}

}  // namespace x17
