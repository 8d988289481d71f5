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
	u32 window;             // 0xFFFFFFFF = unbounded
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

// One CTA per (query head, new token): four warps take every fourth key, a lane D / 32 dims.
template <u32 D, bool SCALED, bool OUT_I8>
__global__ void __launch_bounds__(128)
paged_decode_kernel(const PagedDecodeParams p) {
	pdl_launch_dependents();
	pdl_wait();
	constexpr u32 V = D / 32;
	u32 const warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	u32 const head = blockIdx.x / p.n_tokens, tok = blockIdx.x % p.n_tokens, b = blockIdx.y;
	u32 const kvh = head / (p.n_heads / p.pool.n_kv_heads);
	u64 const row = u64(b) * p.n_tokens + tok;
	u32 const capacity = p.pool.max_pages << p.pool.page_shift;
	u32 const n = min(u32(max(p.kv_lens[b], 0)) + tok, capacity);
	u32 const seen = min(n, p.window), lo = n - seen;
	f32 const q_scale = SCALED ? p.q_scale[row * p.n_heads + head] : 0.125f;
	f32 const base = f32(D == 128 ? 0.08838834764831845 : D == 64 ? 0.125 : 0.17677669529663687);
	f32 const temp = base * log2f(f32(seen + 4)) * p.temperature[head] * q_scale;
	f32 q[V], o[V];
	f32 dot = 0.0f;
#pragma unroll
	for (u32 j = 0; j < V; ++j) {
		q[j] = f32(p.q[row * p.q_stride + head * D + j * 32 + lane]);
		dot += q[j] * f32(p.sink_k[head * D + j * 32 + lane]);
		o[j] = 0.0f;
	}
	auto reduce = [](f32 v) {
#pragma unroll
		for (u32 mask = 16; mask > 0; mask >>= 1) v += __shfl_xor_sync(0xffffffffu, v, mask);
		return v;
	};
	f32 const sink = reduce(dot) * (temp * 0.125f);
	f32 m = sink, sum = 0.0f;
	for (u32 key = lo + warp; key < n; key += 4) {
		u32 page, slot;
		if (!paged_slot(p.pool, i32(b), i32(key), page, slot)) {
			if (lane == 0) report_status(p.status, ST_BAD_INDEX, b);
			continue;
		}
		u64 const at = p.pool.row(page, kvh, slot);
		i8 const *k = p.pool.pages + at * 2 * D;
		f32 d = 0.0f;
#pragma unroll
		for (u32 j = 0; j < V; ++j) d += q[j] * f32(k[j * 32 + lane]);
		f32 const x = reduce(d) * (temp * (SCALED ? p.pool.scales[at * 2] : 0.125f));
		if (x > m) {
			f32 const a = exp2f(m - x);
			sum *= a;
#pragma unroll
			for (u32 j = 0; j < V; ++j) o[j] *= a;
			m = x;
		}
		f32 const e = exp2f(x - m);
		f32 const w = e * (SCALED ? p.pool.scales[at * 2 + 1] : 0.125f);
		sum += e;
#pragma unroll
		for (u32 j = 0; j < V; ++j) o[j] += w * f32(k[D + j * 32 + lane]);
	}
	__shared__ f32 sh_o[4][D], sh_m[4], sh_s[4];
#pragma unroll
	for (u32 j = 0; j < V; ++j) sh_o[warp][j * 32 + lane] = o[j];
	if (lane == 0) {
		sh_m[warp] = m;
		sh_s[warp] = sum;
	}
	__syncthreads();
	u32 const d = threadIdx.x;
	if (d >= D) return;
	f32 top = sink;
#pragma unroll
	for (u32 w = 0; w < 4; ++w) top = fmaxf(top, sh_m[w]);
	f32 const es = exp2f(sink - top);
	f32 total = es, acc = es * f32(p.sink_v[head * D + d]) * 0.125f;
#pragma unroll
	for (u32 w = 0; w < 4; ++w) {
		f32 const a = exp2f(sh_m[w] - top);
		total += a * sh_s[w];
		acc += a * sh_o[w][d];
	}
	f32 const v = __fdiv_rn(acc, total);
	u64 const at = row * p.o_stride + head * D + d;
	if constexpr (OUT_I8) static_cast<i8 *>(p.out)[at] = i8(f32_to_fixedi8(v * 8.0f));
	else static_cast<u16 *>(p.out)[at] = u16(cvt_bf16x2(v, 0.0f));
	if (d == 0 && p.l != nullptr) p.l[row * p.n_heads + head] = log2f(255.0f * total) + top;
}

}  // namespace x17
