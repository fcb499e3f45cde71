// kv.cuh — what rope.cu, kvcache.cu and kvattn.cu share: the handles behind
// moe_rope / moe_kv_cache, argument checks, packed batches on the device, and
// 16-byte vectors of fp32, fp16 or bf16 values.
#pragma once

#include "common.cuh"
#include "kernels.h"
#include "moe_b200.h"

#include <cuda_bf16.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>

// angle tables of moe_rope_create: for pair i and position p the angle is the
// sum of lo[p % 1024][i]'s and hi[p / 1024][i]'s, whose cosines and sines (hi's
// times the magnitude) are held in 64 bits
struct moe_rope {
	int device = 0;
	int64_t rot = 0, max_position = 0;
	int layout = 0;
	double2 *lo = nullptr, *hi = nullptr;
	int32_t *err = nullptr;
};

struct moe_kv_cache {
	moe_kv_desc d{};
	int device = 0;
	int page_log2 = 0;
	size_t page_bytes = 0;
	uint8_t *pages = nullptr;
	bool owned = false;
	int32_t *err = nullptr;
	bool err_owned = false;
};

namespace moe {

constexpr int kRopeLow = 1024;   // rows of the low table

// bits of a handle's error word
enum { kKvErrBatch = 1, kKvErrPage = 2, kKvErrPos = 4, kKvErrWait = 8 };

// ---------------------------------------------------------------- host side
inline int kv_fail(int code, const char *fmt, ...)
{
	char buf[512];
	va_list ap;
	va_start(ap, fmt);
	vsnprintf(buf, sizeof buf, fmt, ap);
	va_end(ap);
	set_last_error(buf);
	return code;
}

inline int kv_cuda(cudaError_t e, const char *what)
{
	return kv_fail(e == cudaErrorMemoryAllocation ? MOE_ERR_NOMEM : MOE_ERR_CUDA, "%s: %s", what,
		       cudaGetErrorString(e));
}

#define KV_CK(what, call)                                          \
	do {                                                       \
		cudaError_t e_ = (call);                           \
		if (e_ != cudaSuccess)                             \
			return moe::kv_cuda(e_, what);             \
	} while (0)

// the handle's device for the length of a call
struct DeviceGuard {
	int before = -1;
	cudaError_t e = cudaSuccess;
	explicit DeviceGuard(int device)
	{
		e = cudaGetDevice(&before);
		if (e == cudaSuccess && before != device)
			e = cudaSetDevice(device);
		else
			before = -1;
	}
	~DeviceGuard()
	{
		if (before >= 0)
			cudaSetDevice(before);
	}
	DeviceGuard(const DeviceGuard &) = delete;
	DeviceGuard &operator=(const DeviceGuard &) = delete;
};

inline int row_type_bytes(int type)
{
	return type == MOE_F32 ? 4 : type == MOE_F16 || type == MOE_BF16 ? 2 : 0;
}

// the largest offset (in elements) that rows of these sizes reach must fit
// 64-bit arithmetic with room to spare
constexpr int64_t kMaxStride = (int64_t)1 << 40;

inline int check_rows(const char *what, const char *name, const moe_rows *r, int64_t n_tokens,
		      int64_t head_len, int type, int64_t n_heads, bool output)
{
	if (!r || (!r->data && n_tokens > 0))
		return kv_fail(MOE_ERR_INVALID, "%s: %s missing", what, name);
	if (!row_type_bytes(r->type))
		return kv_fail(MOE_ERR_UNSUPPORTED, "%s: %s has type %d", what, name, r->type);
	if (r->type != type)
		return kv_fail(MOE_ERR_UNSUPPORTED, "%s: %s has type %d beside %d", what, name, r->type,
			       type);
	if (r->n_heads <= 0 || r->n_heads > (1 << 19) / head_len ||
	    (n_heads > 0 && r->n_heads != n_heads))
		return kv_fail(MOE_ERR_INVALID, "%s: %s has %lld heads", what, name,
			       (long long)r->n_heads);
	if ((uintptr_t)r->data % row_type_bytes(r->type))
		return kv_fail(MOE_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
	const int64_t ts = r->token_stride, hs = r->head_stride;
	if (ts < 0 || hs < 0 || ts > kMaxStride || hs > kMaxStride)
		return kv_fail(MOE_ERR_INVALID, "%s: %s has strides %lld, %lld", what, name,
			       (long long)ts, (long long)hs);
	if (output) {
		// rows apart: the smaller stride spans a row, the larger one the
		// other dimension's extent
		const bool t1 = n_tokens <= 1, h1 = r->n_heads == 1;
		const int64_t over_h = (r->n_heads - 1) * hs + head_len;
		const bool ok = t1 && h1 ? true
				: t1 ? hs >= head_len
				: h1 ? ts >= head_len
				     // (the tokens' extent may pass 64 bits)
				     : (hs >= head_len && ts >= over_h) ||
				       (ts >= head_len && hs >= head_len && n_tokens - 1 <= (hs - head_len) / ts);
		if (!ok)
			return kv_fail(MOE_ERR_INVALID, "%s: rows of %s overlap (strides %lld, %lld)", what,
				       name, (long long)ts, (long long)hs);
	}
	return MOE_OK;
}

inline bool rows_vec16(const moe_rows *r)
{
	const int es = row_type_bytes(r->type);
	return (uintptr_t)r->data % 16 == 0 && r->token_stride * es % 16 == 0 &&
	       r->head_stride * es % 16 == 0;
}

inline int check_batch(const char *what, const moe_kv_cache *c, const moe_kv_batch *b,
		       bool arrays = true)
{
	if (!b)
		return kv_fail(MOE_ERR_INVALID, "%s: batch missing", what);
	if (b->n_seqs < 0 || b->n_seqs > (1 << 20) || b->n_tokens < 0 || b->n_tokens > (1 << 30) ||
	    b->max_q < 0 || b->max_q > (1 << 30) || b->max_kv < 0 || b->max_kv > (1 << 30) ||
	    b->table_stride < 0 || b->table_stride > (1 << 30))
		return kv_fail(MOE_ERR_INVALID, "%s: batch of %lld sequences, %lld tokens (max_q %lld, "
			       "max_kv %lld, table_stride %lld)", what, (long long)b->n_seqs,
			       (long long)b->n_tokens, (long long)b->max_q, (long long)b->max_kv,
			       (long long)b->table_stride);
	if (b->max_kv > b->table_stride * c->d.page_size)
		return kv_fail(MOE_ERR_INVALID, "%s: max_kv %lld needs more than table_stride %lld pages "
			       "of %lld", what, (long long)b->max_kv, (long long)b->table_stride,
			       (long long)c->d.page_size);
	if (arrays && b->n_seqs > 0 && b->n_tokens > 0 &&
	    (!b->q_start || !b->kv_len || (b->max_kv > 0 && !b->page_table)))
		return kv_fail(MOE_ERR_INVALID, "%s: batch arrays missing", what);
	if (arrays && ((uintptr_t)b->q_start | (uintptr_t)b->kv_len | (uintptr_t)b->page_table) % 4)
		return kv_fail(MOE_ERR_INVALID, "%s: batch arrays are not aligned", what);
	return MOE_OK;
}

// stream argument of the C ABI: NULL is the library stream, which must be
// of the handle's device
inline int resolve_stream(const char *what, int device, void *stream, cudaStream_t *st)
{
	if (stream) {
		*st = static_cast<cudaStream_t>(stream);
		return MOE_OK;
	}
	DeviceGuard g(device);
	KV_CK(what, g.e);
	if (int rc = ensure_library())
		return rc;
	*st = library_stream();
	return MOE_OK;
}

// ---------------------------------------------------------------- device side
struct BatchArgs {
	const int32_t *q_start, *kv_len, *table;
	int64_t table_stride;
	int B, T, max_q, max_kv;
	int n_pages, page_log2;
	int32_t *err;
};

inline BatchArgs batch_args(const moe_kv_cache *c, const moe_kv_batch *b)
{
	BatchArgs a;
	a.q_start = b->q_start;
	a.kv_len = b->kv_len;
	a.table = b->page_table;
	a.table_stride = b->table_stride;
	a.B = (int)b->n_seqs;
	a.T = (int)b->n_tokens;
	a.max_q = (int)b->max_q;
	a.max_kv = (int)b->max_kv;
	a.n_pages = (int)c->d.n_pages;
	a.page_log2 = c->page_log2;
	a.err = c->err;
	return a;
}

// the sequence of token t: the number of sequences that end at or before
// it (B for padding).  A warp narrows 32-fold a round, all probes of a round
// in flight together: 2 rounds up to 1024 sequences.
__device__ __forceinline__ int find_seq(const int32_t *q_start, int B, int t)
{
	const int lane = threadIdx.x % 32;
	int lo = 0, n = B;
	while (n > 0) {
		const int step = (n + 31) / 32, off = (lane + 1) * step;
		const bool le = off <= n && q_start[lo + off] <= t;
		const int cnt = __popc(__ballot_sync(0xffffffffu, le));
		lo += cnt * step;
		n = min(step - 1, n - cnt * step);
	}
	return lo;
}

// where a token's row lies: its sequence's cache row, page and row of the page;
// not ok (and the error word) if the arrays are out of range, silently for padding
struct TokenRow {
	int ok, row, page, at;
};
// by a warp: lane l's is token t0 + l (l < n).  One search finds the first token's
// sequence; the others lie in it or in the next ones.
__device__ __forceinline__ TokenRow find_rows(const BatchArgs &a, int t0, int n)
{
	const int lane = threadIdx.x % 32, t = t0 + lane;
	TokenRow r{0, 0, 0, 0};
	int b = find_seq(a.q_start, a.B, t0);
	if (lane >= n)
		return r;
	int s1 = b < a.B ? a.q_start[b + 1] : 0;
	for (; b < a.B && s1 <= t; s1 = b < a.B ? a.q_start[b + 1] : 0)
		b++;
	if (b >= a.B)
		return r;
	const int s0 = a.q_start[b], kv = a.kv_len[b];
	r.row = kv - (s1 - t);
	if (s0 < 0 || s0 > t || s1 <= t || s1 > a.T || s1 - s0 > a.max_q || kv < s1 - s0 ||
	    kv > a.max_kv) {
		atomicOr(a.err, kKvErrBatch);
		return r;
	}
	r.page = a.table[b * a.table_stride + (r.row >> a.page_log2)];
	r.at = r.row & ((1 << a.page_log2) - 1);
	if (r.page < 0 || r.page >= a.n_pages) {
		atomicOr(a.err, kKvErrPage);
		return r;
	}
	r.ok = 1;
	return r;
}

// by a warp of the first CTA: sequences that no token leads to (a q_start that
// falls names none) are reported too
__device__ __forceinline__ void check_sequences(const BatchArgs &a)
{
	bool bad = threadIdx.x % 32 == 0 && a.q_start[0] != 0;
	for (int b = threadIdx.x % 32; b < a.B; b += 32)
		bad |= a.q_start[b + 1] < a.q_start[b] || a.q_start[b + 1] > a.T;
	if (bad)
		atomicOr(a.err, kKvErrBatch);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
	return __float2bfloat16_rn(v);
}

// N values side by side as they lie in memory: 16-byte accesses (VEC) or single
// ones.  Loads in flight hold no more registers than they bring bytes.
template <typename T, int N, bool VEC>
struct Raw {
	static_assert(!VEC || N * sizeof(T) % 16 == 0, "whole vectors");
	union {
		T v[N];
		uint32_t w[(N * sizeof(T) + 3) / 4];
		uint4 u[(N * sizeof(T) + 15) / 16];
	};
	__device__ Raw() {}
	__device__ void load(const T *p)
	{
		if constexpr (VEC) {
#pragma unroll
			for (int i = 0; i < (int)(N * sizeof(T) / 16); i++)
				u[i] = reinterpret_cast<const uint4 *>(p)[i];
		} else {
#pragma unroll
			for (int i = 0; i < N; i++)
				v[i] = p[i];
		}
	}
	__device__ void store(T *p) const
	{
		if constexpr (VEC) {
#pragma unroll
			for (int i = 0; i < (int)(N * sizeof(T) / 16); i++)
				reinterpret_cast<uint4 *>(p)[i] = u[i];
		} else {
#pragma unroll
			for (int i = 0; i < N; i++)
				p[i] = v[i];
		}
	}
	__device__ void get(float (&f)[N]) const
	{
#pragma unroll
		for (int i = 0; i < N; i++)
			f[i] = to_f32(v[i]);
	}
	__device__ void set(const float (&f)[N])
	{
#pragma unroll
		for (int i = 0; i < N; i++)
			v[i] = from_f32<T>(f[i]);
	}
	// another lane's
	__device__ Raw from_lane(int lane) const
	{
		Raw r;
#pragma unroll
		for (int i = 0; i < (int)(N * sizeof(T) / 4); i++)
			r.w[i] = __shfl_sync(0xffffffffu, w[i], lane);
		return r;
	}
};

// ---------------------------------------------------------------- rotation
struct RopeArgs {
	const double2 *lo, *hi;
	int half;            // turning pairs of a head (0: none)
	int max_position;
};

inline RopeArgs rope_args(const moe_rope *r)
{
	RopeArgs a{nullptr, nullptr, 0, 0};
	if (r) {
		a.lo = r->lo;
		a.hi = r->hi;
		a.half = (int)(r->rot / 2);
		a.max_position = (int)r->max_position;
	}
	return a;
}

// cosine and sine of pair i at a position: the sum of the two tables' angles,
// (cos + i sin) multiplied in 64 bits, so the fp32 result is the 64-bit one
// rounded
__device__ __forceinline__ float2 rope_angle(const RopeArgs &r, int pos, int i)
{
	const double2 a = r.lo[(int64_t)(pos % kRopeLow) * r.half + i];
	const double2 b = r.hi[(int64_t)(pos / kRopeLow) * r.half + i];
	return make_float2((float)(a.x * b.x - a.y * b.y), (float)(a.x * b.y + a.y * b.x));
}

// each product and the sum rounded once (rope_apply's operations, nn.c:192-219)
__device__ __forceinline__ void turn(float &a, float &b, float2 cs)
{
	const float y0 = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
	const float y1 = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
	a = y0;
	b = y1;
}

// heads of a tensor as the kernels take them
template <typename T>
struct Heads {
	const T *in;
	T *out;
	int64_t in_ts, in_hs, out_ts, out_hs;
	int n;
};

template <typename T>
inline Heads<T> heads_of(const moe_rows *in, const moe_rows *out)
{
	Heads<T> h{nullptr, nullptr, 0, 0, 0, 0, 0};
	if (in) {
		h.in = static_cast<const T *>(in->data);
		h.in_ts = in->token_stride;
		h.in_hs = in->head_stride;
		h.n = (int)in->n_heads;
	}
	if (out) {
		h.out = static_cast<T *>(out->data);
		h.out_ts = out->token_stride;
		h.out_hs = out->head_stride;
	}
	return h;
}

// j / n for j * n < 2^32 by the high half of a product; or (zero) 0
struct FastDiv {
	unsigned n = 1, m = 0;
	FastDiv() {}
	explicit FastDiv(unsigned n_, bool zero = false)
		: n(zero ? 2 : n_), m(n_ > 1 && !zero ? (unsigned)(0x100000000ull / n_) + 1 : 0)
	{
	}
	__device__ unsigned div(unsigned j) const { return n > 1 ? __umulhi(j, m) : j; }
};

// How a kernel takes the turning pairs: beside each other; in two halves whose
// 8-value vectors are partners (half % 8 == 0; a head's vectors in lanes of one
// warp); or in halves of any size, value by value
enum { kTurnPairs = 0, kTurnHalves = 1, kTurnAny = 2 };
inline int turn_of(int layout, int half)
{
	return layout == MOE_ROPE_PAIRS ? kTurnPairs : half % 8 == 0 ? kTurnHalves : kTurnAny;
}

// A lane's 8 values e0 .. of any head of a token, with the token's angles for them in
// registers (a row's vectors stand in consecutive lanes, so every row that a lane
// takes part in has the same place for it).
template <int TURN>
struct Turn8 {
	static_assert(TURN != kTurnAny, "by value");
	static constexpr int kAngles = TURN == kTurnPairs ? 4 : 8;
	float2 c[kAngles];
	int turning;   // PAIRS: of the 4 pairs; HALVES: all or none
	int from;      // HALVES: the partners' lane
	bool low;      // HALVES: in the first half
	__device__ Turn8(int e0, int half)
	{
		if (TURN == kTurnPairs) {
			turning = min(max(half - e0 / 2, 0), 4);
			low = true;
			from = 0;
		} else {
			const int lane = threadIdx.x % 32;
			low = e0 < half;
			turning = e0 < 2 * half ? 8 : 0;
			from = !turning ? lane : low ? lane + half / 8 : lane - half / 8;
		}
	}
	__device__ void angles(const float2 *cs, int e0, int half)
	{
		const float2 *p = cs + (TURN == kTurnPairs ? e0 / 2 : low ? e0 : e0 - half);
#pragma unroll
		for (int k = 0; k < kAngles; k++)
			if (k < turning)
				c[k] = p[k];
		if (TURN == kTurnHalves && low) {
			// the low value's partner counts negatively: a + (-b) is a - b
#pragma unroll
			for (int k = 0; k < kAngles; k++)
				c[k].y = -c[k].y;
		}
	}
	// every lane of the warp calls it: partners come from their lanes, so an output
	// may be its input
	template <typename R>
	__device__ void apply(const R &x, float (&f)[8]) const
	{
		x.get(f);
		if constexpr (TURN == kTurnPairs) {
#pragma unroll
			for (int k = 0; k < 4; k++)
				if (k < turning)
					turn(f[2 * k], f[2 * k + 1], c[k]);
		} else {
			float g[8];
			x.from_lane(from).get(g);
			if (turning) {
#pragma unroll
				for (int k = 0; k < 8; k++)
					f[k] = __fadd_rn(__fmul_rn(f[k], c[k].x), __fmul_rn(g[k], c[k].y));
			}
		}
	}
};

// The rounds of a token, a round being 32 lanes of whole rows: a group's tokens go to
// the CTA's warps in turn; with fewer tokens than warps (1, 2, 4) a token's rounds
// are dealt to several warps, and over the grid's slices.
struct Rounds {
	int token, token_step;   // first and next of the warp's tokens
	int first, step_log2;    // of a token's rounds
	__device__ __forceinline__ Rounds(const struct TokenSplit &s, int slice);
	__device__ __forceinline__ int step() const { return 1 << step_log2; }
	// the first of the warp's rounds of a sort of rows that `before` rounds precede
	__device__ __forceinline__ int start(int before) const
	{
		const int d = before - first;
		return d <= 0 ? -d : -d & (step() - 1);
	}
};

// value i of a head's first half and its partner, or a value behind the turning
// ones: an item of kTurnAny
template <typename T>
struct PairItem {
	T a, b;
	__device__ static int first(int i, int half) { return i < half ? i : i + half; }
	__device__ void load(const T *head, int i, int half)
	{
		a = head[first(i, half)];
		if (i < half)
			b = head[i + half];
	}
	__device__ void turn_store(T *head, int i, const float2 *cs, int half) const
	{
		if (i < half) {
			float x = to_f32(a), y = to_f32(b);
			turn(x, y, cs[i]);
			head[i] = from_f32<T>(x);
			head[i + half] = from_f32<T>(y);
		} else {
			head[i + half] = a;
		}
	}
};

// How a packed batch is cut into CTAs of 8 warps (a token's items are `rounds` warps
// of them): as many tokens to a CTA (up to kGroupTokens, and 2048 angles) as leave a
// wave and a half of resident CTAs, so that the look-ups and angles that a CTA waits
// for are paid once for much work.  Against 1 and 2 waves: 2048 tokens' rotation 17.2
// us (17.3, 18.5), 16383 tokens' 58.8 (59.8, 59.1), 16383 appended 54.2 (57.6, 54.0).
// Few tokens: several warps and CTAs a token.  Powers of two, for the divisions that
// a decode step would wait for.
constexpr int kGroupTokens = 32;
struct TokenSplit {
	int tokens;       // of a CTA: 1, 2, 4 or a multiple of 8
	int share_log2;   // warps of a token: 8, 4, 2 or 1
	int slices_log2;  // CTAs of a token
};
inline TokenSplit split_tokens(int64_t n_tokens, int64_t rounds, int half)
{
	const int64_t wave = 4 * (int64_t)sm_count();
	int64_t tokens = (2 * n_tokens + 3 * wave - 1) / (3 * wave);
	tokens = tokens < kGroupTokens ? tokens : kGroupTokens;
	while (tokens > 1 && tokens * half > 2048)
		tokens--;
	if (tokens > 1) {
		tokens = tokens < 3 ? 2 : tokens < 7 ? 4 : (tokens + 4) / 8 * 8;
		return {(int)tokens, tokens == 2 ? 2 : tokens == 4 ? 1 : 0, 0};
	}
	int y = 0;
	while (y < 15 && (int64_t)8 << y < rounds && n_tokens << (y + 1) <= 2 * wave)
		y++;
	return {1, 3, y};
}

__device__ __forceinline__ Rounds::Rounds(const TokenSplit &s, int slice)
{
	const int warp = threadIdx.x / 32;
	token = warp >> s.share_log2;
	token_step = 8 >> s.share_log2;
	first = (slice << s.share_log2) + (warp & ((1 << s.share_log2) - 1));
	step_log2 = s.share_log2 + s.slices_log2;
}

// A warp's rows in flight to slots of its own in shared memory, kDepth rounds of them:
// loads that hold no registers, so that a warp keeps 2 KB on the way whatever its work
// needs (64 KB an SM; with 3 KB 16383 tokens take 60.9 us instead of 59.8 to rotate).
// Rounds come out in the order in which they went in.  A lane gets 8 values side by
// side; those of fp32 rows are 32 bytes, which reach memory as two times 16 that
// neighbouring lanes hold together (each 32-byte sector once).  Rows that are not
// 16-byte aligned are read where they come out.
template <typename T, bool VEC>
struct RowStream {
	static constexpr int kParts = 8 * sizeof(T) / 16, kDepth = 8 / (int)sizeof(T);
	static constexpr int kWarpBytes = VEC ? kDepth * kParts * 512 : 0;
	uint32_t mine, part;   // the lane's 8 values of a slot, its 16 bytes of a row's first part
	int across, jump;      // bytes from part to part, and from the values to part 0 in memory
	int in = 0, out = 0;
	const T *next[VEC ? 1 : kDepth];
	__device__ RowStream(uint8_t *slots, int row_lanes)
	{
		const uint32_t base = (uint32_t)__cvta_generic_to_shared(slots) + threadIdx.x / 32 * kWarpBytes;
		const int lane = threadIdx.x % 32, j = lane & (row_lanes - 1);
		mine = base + lane * 16 * kParts;
		across = kParts == 1 ? 0 : 16 * row_lanes;
		jump = kParts == 1 ? 0 : -16 * j;
		part = mine + jump;
	}
	__device__ __forceinline__ void push(const T *p)   // NULL: no row
	{
		if constexpr (VEC) {
			if (p) {
				const uint8_t *q = reinterpret_cast<const uint8_t *>(p) + jump;
#pragma unroll
				for (int i = 0; i < kParts; i++)
					asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
							     part + in * (512 * kParts) + i * across),
						     "l"(q + i * across)
						     : "memory");
			}
			asm volatile("cp.async.commit_group;" ::: "memory");
			in = in + 1 == kDepth ? 0 : in + 1;
		} else {
#pragma unroll
			for (int i = 0; i + 1 < kDepth; i++)
				next[i] = next[i + 1];
			next[kDepth - 1] = p;
		}
	}
	__device__ __forceinline__ void idle()   // keeps the count of groups in step
	{
		if constexpr (VEC)
			asm volatile("cp.async.commit_group;" ::: "memory");
		else
			push(nullptr);
	}
	__device__ __forceinline__ void pop(Raw<T, 8, VEC> &x)
	{
		if constexpr (VEC) {
			asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
			if (kParts > 1)
				__syncwarp();   // the other lanes' parts
#pragma unroll
			for (int i = 0; i < kParts; i++)
				asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
					     : "=r"(x.u[i].x), "=r"(x.u[i].y), "=r"(x.u[i].z), "=r"(x.u[i].w)
					     : "r"(mine + out * (512 * kParts) + 16 * i)
					     : "memory");
			out = out + 1 == kDepth ? 0 : out + 1;
			if (kParts > 1)
				__syncwarp();   // read by all before a next row overwrites it
		} else if (next[0]) {
			x.load(next[0]);
		}
	}
	// the round popped last, written to p (NULL: nothing) before the next push
	__device__ __forceinline__ void store(const Raw<T, 8, VEC> &x, T *p)
	{
		if constexpr (VEC && kParts > 1) {
			const uint32_t slot = (out == 0 ? kDepth - 1 : out - 1) * (512 * kParts);
#pragma unroll
			for (int i = 0; i < kParts; i++)
				asm volatile("st.shared.v4.u32 [%4], {%0, %1, %2, %3};" ::"r"(x.u[i].x),
					     "r"(x.u[i].y), "r"(x.u[i].z), "r"(x.u[i].w),
					     "r"(mine + slot + 16 * i)
					     : "memory");
			__syncwarp();
#pragma unroll
			for (int i = 0; i < kParts; i++) {
				uint4 v;
				asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
					     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
					     : "r"(part + slot + i * across)
					     : "memory");
				if (p)
					*reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p) + jump +
								   i * across) = v;
			}
			__syncwarp();
		} else if (p) {
			x.store(p);
		}
	}
	__device__ __forceinline__ void finish()
	{
		if constexpr (VEC)
			asm volatile("cp.async.wait_group 0;" ::: "memory");
	}
};

// A warp's rounds of one sort of rows of a token, in turn: round r's row of a lane is
// row r * m + sub of heads.n
template <typename T>
struct RowWalk {
	int row, rows, left, step_rows;   // the lane's next row, of how many; rounds left
	__device__ __forceinline__ RowWalk(int n, int m_log2, int sub, int start, int step_log2)
		: row((start << m_log2) + sub), rows(n)
	{
		const int rounds = (n + (1 << m_log2) - 1) >> m_log2;
		left = rounds > start ? (rounds - start + (1 << step_log2) - 1) >> step_log2 : 0;
		step_rows = 1 << (m_log2 + step_log2);
	}
	__device__ __forceinline__ bool has() const { return row < rows; }
};

// the same rows on their way, kDepth rounds ahead of the work
template <typename T, bool VEC>
struct RowReader {
	RowStream<T, VEC> &stream;
	RowWalk<T> w;
	const T *p;
	int64_t d;
	__device__ __forceinline__ RowReader(RowStream<T, VEC> &s, const Heads<T> &h, int64_t token, int n,
					     int m_log2, int sub, int e0, int start, int step_log2)
		: stream(s), w(n, m_log2, sub, start, step_log2),
		  p(h.in + token * h.in_ts + (int64_t)w.row * h.in_hs + e0), d((int64_t)w.step_rows * h.in_hs)
	{
	}
	__device__ __forceinline__ void next()
	{
		if (w.left > 0) {
			stream.push(w.has() ? p : nullptr);
			w.left--;
			w.row += w.step_rows;
			p += d;
		} else {
			stream.idle();
		}
	}
	__device__ __forceinline__ void begin()
	{
		if (w.left == 0)   // what another reader has begun stays next
			return;
#pragma unroll
		for (int i = 0; i < RowStream<T, VEC>::kDepth; i++)
			next();
	}
	// the same rows begun by another reader
	__device__ __forceinline__ void skip_begun()
	{
		const int n = min(w.left, RowStream<T, VEC>::kDepth);
		w.left -= n;
		w.row += n * w.step_rows;
		p += n * d;
	}
};

}  // namespace moe
