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
};

namespace moe {

constexpr int kRopeLow = 1024;   // rows of the low table

// bits of a handle's error word
enum { kKvErrBatch = 1, kKvErrPage = 2, kKvErrPos = 4 };

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
	if (r->n_heads <= 0 || r->n_heads > 65535 || (n_heads > 0 && r->n_heads != n_heads))
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
		const int64_t over_t = (n_tokens > 0 ? n_tokens - 1 : 0) * ts + head_len;
		const bool ok = t1 && h1 ? true
				: t1 ? hs >= head_len
				: h1 ? ts >= head_len
				     : (hs >= head_len && ts >= over_h) || (ts >= head_len && hs >= over_t);
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

// where token t's row lies: its sequence's cache row, page and row of the
// page; false (and the error word) if the arrays are out of range, silently
// for padding
struct TokenRow {
	int row, page, at;
};
__device__ __forceinline__ bool find_row(const BatchArgs &a, int t, TokenRow &r)
{
	const int b = find_seq(a.q_start, a.B, t);
	if (b >= a.B)
		return false;
	const int s0 = a.q_start[b], s1 = a.q_start[b + 1], kv = a.kv_len[b];
	r.row = kv - (s1 - t);
	if (s0 < 0 || s0 > t || s1 <= t || s1 > a.T || s1 - s0 > a.max_q || kv < s1 - s0 ||
	    kv > a.max_kv) {
		if (threadIdx.x == 0)
			atomicOr(a.err, kKvErrBatch);
		return false;
	}
	r.page = a.table[b * a.table_stride + (r.row >> a.page_log2)];
	r.at = r.row & ((1 << a.page_log2) - 1);
	if (r.page < 0 || r.page >= a.n_pages) {
		if (threadIdx.x == 0)
			atomicOr(a.err, kKvErrPage);
		return false;
	}
	return true;
}

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);   // values of a 16-byte vector

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

template <typename T>
union Vec16 {
	uint4 u;
	T v[kVec<T>];
	__device__ Vec16() {}
};

// N consecutive values: one 16-byte access (VEC, N = kVec<T>) or N single ones
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_n(const T *p, float (&f)[N])
{
	if constexpr (VEC) {
		static_assert(N == kVec<T>, "one vector");
		Vec16<T> x;
		x.u = *reinterpret_cast<const uint4 *>(p);
#pragma unroll
		for (int i = 0; i < N; i++)
			f[i] = to_f32(x.v[i]);
	} else {
#pragma unroll
		for (int i = 0; i < N; i++)
			f[i] = to_f32(p[i]);
	}
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_n(T *p, const float (&f)[N])
{
	if constexpr (VEC) {
		static_assert(N == kVec<T>, "one vector");
		Vec16<T> x;
#pragma unroll
		for (int i = 0; i < N; i++)
			x.v[i] = from_f32<T>(f[i]);
		*reinterpret_cast<uint4 *>(p) = x.u;
	} else {
#pragma unroll
		for (int i = 0; i < N; i++)
			p[i] = from_f32<T>(f[i]);
	}
}

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

// cosine and sine of every pair at a position, by the CTA's threads: the
// sum of the two tables' angles, (cos + i sin) multiplied in 64 bits, so
// the fp32 result is the 64-bit one rounded
__device__ __forceinline__ void rope_angles(const RopeArgs &r, int pos, float2 *cs)
{
	for (int i = threadIdx.x; i < r.half; i += blockDim.x) {
		const double2 a = r.lo[(int64_t)(pos % kRopeLow) * r.half + i];
		const double2 b = r.hi[(int64_t)(pos / kRopeLow) * r.half + i];
		cs[i] = make_float2((float)(a.x * b.x - a.y * b.y), (float)(a.x * b.y + a.y * b.x));
	}
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

// A head's values in items that one thread reads, turns and writes whole, so
// that an output may be its input.  PAIRS: N values side by side.  HALVES: the
// first items hold N values of each half (their partners), the rest N values
// behind the turning ones.
template <int N, int LAYOUT>
struct RopeItem {
	int e0, e1;   // first value, and the partners' (HALVES: -1 behind rot)
	__device__ RopeItem(int i, int half)
	{
		const int pairs = LAYOUT == MOE_ROPE_HALVES ? half / N : 0;
		if (LAYOUT == MOE_ROPE_PAIRS) {
			e0 = i * N;
			e1 = -1;
		} else if (i < pairs) {
			e0 = i * N;
			e1 = half + i * N;
		} else {
			e0 = 2 * half + (i - pairs) * N;
			e1 = -1;
		}
	}
	__host__ __device__ static int per_head(int head_len, int half)
	{
		return LAYOUT == MOE_ROPE_PAIRS ? head_len / N : head_len / N - half / N;
	}
	__device__ void apply(float (&x)[N], float (&y)[N], const float2 *cs, int half) const
	{
		if (LAYOUT == MOE_ROPE_PAIRS) {
			if constexpr (N >= 2) {
#pragma unroll
				for (int k = 0; k < N; k += 2)
					if ((e0 + k) / 2 < half)
						turn(x[k], x[k + 1], cs[(e0 + k) / 2]);
			}
		} else if (e1 >= 0) {
#pragma unroll
			for (int k = 0; k < N; k++)
				turn(x[k], y[k], cs[e0 + k]);
		}
	}
};

}  // namespace moe
