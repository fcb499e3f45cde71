// kvcache.cu — the paged key/value cache in 4 bits (moe_kv_*): handles,
// append with the rotation on the way, read-back, and the row moves of the
// whole model's cache rotation.  The layout of a page is described in
// moe_b200.h; kvattn.cu reads it.
#include "kv.cuh"

namespace moe {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendBatch = 2;   // items of a thread whose loads are in flight together

// address of a KV head's record of a page: K codes, K scales, V codes, V scales
struct PageArgs {
	uint8_t *pages;
	int64_t page_bytes;
	int KVH, head_len, page_log2;
};

PageArgs page_args(const moe_kv_cache *c)
{
	PageArgs a;
	a.pages = c->pages;
	a.page_bytes = (int64_t)c->page_bytes;
	a.KVH = (int)c->d.n_kv_heads;
	a.head_len = (int)c->d.head_len;
	a.page_log2 = c->page_log2;
	return a;
}

__device__ __forceinline__ uint8_t *record(const PageArgs &a, int page, int head, int which)
{
	const int64_t half = ((int64_t)a.head_len / 2 + a.head_len / 16) << a.page_log2;
	return a.pages + page * a.page_bytes + (2 * head + which) * half;
}

template <typename T>
struct AppendArgs {
	BatchArgs b;
	PageArgs p;
	RopeArgs r;
	const int32_t *pos;   // or NULL: the cache rows
	Heads<T> q, k, v;     // k, v: inputs only; q.n 0: none
};

// A lane's N values of a 32-value block, N / 32 of it in consecutive lanes:
// the block's scale and codes (moe_kv_desc), two 4-bit codes to a byte with
// the lane that holds the values 16 further on.  Lanes of the lower half
// return the block's bytes sub * N .. sub * N + N - 1.
template <int N>
__device__ __forceinline__ void quantize_block(const float (&x)[N], __half &scale,
					       uint32_t (&by)[N / 4])
{
	constexpr int L = 32 / N;
	float hi = x[0], lo = x[0];
	bool bad = false;
#pragma unroll
	for (int k = 0; k < N; k++) {
		hi = fmaxf(hi, x[k]);
		lo = fminf(lo, x[k]);
		bad |= !(fabsf(x[k]) <= 3.402823466e38f);
	}
#pragma unroll
	for (int o = 1; o < L; o *= 2) {
		hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
		lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
	}
	const unsigned any = __ballot_sync(0xffffffffu, bad);
	bad = (any >> (threadIdx.x % 32 / L * L)) & ((1u << L) - 1);
	// the value of the largest magnitude takes code 0 (-8): a step of m / 8
	// where a symmetric code would have m / 7
	const float m = hi >= -lo ? hi : lo;
	scale = __float2half_rn(fminf(fmaxf(__fmul_rn(m, -0.125f), -65504.0f), 65504.0f));
	const float d = __half2float(scale);
	const float inv = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
	if (d == 0.0f || bad)   // one zero: which zero m is depends on the order of its zeros
		scale = __ushort_as_half(bad ? 0x7fff : 0);
#pragma unroll
	for (int w = 0; w < N / 4; w++) {
		uint32_t c = 0;
#pragma unroll
		for (int k = 0; k < 4; k++) {
			const int code = min(max(__float2int_rn(__fmul_rn(x[4 * w + k], inv)), -8), 7) + 8;
			c |= (uint32_t)(bad ? 8 : code) << (8 * k);
		}
		by[w] = c | __shfl_xor_sync(0xffffffffu, c, L / 2) << 4;
	}
}

// grid (token, slice of its items): per token the query heads are turned
// and written, then the key heads turned and quantized, the value heads
// quantized; a warp has items of one sort.  Bound by bytes for prompts (q, k, v
// in, q and 0.5625 bytes a value out) and by latency for decode batches:
// the rows leave for the registers first, then come the sequence (a search
// of two rounds), the angles and the page, each a dependent load.
template <typename T, bool VEC, int LAYOUT>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(AppendArgs<T> a)
{
	constexpr int N = kVec<T>, L = 32 / N;
	constexpr int QN = VEC ? N : LAYOUT == MOE_ROPE_PAIRS ? 2 : 1;   // q's item
	extern __shared__ float2 cs[];
	const int t = blockIdx.x;
	const int D = a.p.head_len, half = a.r.half, nb = D / 32;
	const int per_q = RopeItem<QN, LAYOUT>::per_head(D, half);
	const int nq = a.q.n * per_q, nq32 = (nq + 31) / 32 * 32;
	const int per = D / N, nkv = a.p.KVH * per;   // items of the keys, and of the values
	const int total = nq32 + 2 * nkv;
	const int step = gridDim.y * kAppendThreads;
	TokenRow row;
	int pos = 0;
	bool ready = false;
	for (int i0 = blockIdx.y * kAppendThreads + threadIdx.x; __syncthreads_or(i0 < total);
	     i0 += kAppendBatch * step) {
		float x[kAppendBatch][N], y[kAppendBatch][N];
#pragma unroll
		for (int u = 0; u < kAppendBatch; u++) {
			const int i = i0 + u * step;
			if (i < nq) {
				const RopeItem<QN, LAYOUT> it(i % per_q, half);
				const T *p = a.q.in + t * a.q.in_ts + (i / per_q) * a.q.in_hs;
				float f[QN];
				load_n<T, QN, VEC>(p + it.e0, f);
#pragma unroll
				for (int k = 0; k < QN; k++)
					x[u][k] = f[k];
				if (LAYOUT == MOE_ROPE_HALVES && it.e1 >= 0) {
					load_n<T, QN, VEC>(p + it.e1, f);
#pragma unroll
					for (int k = 0; k < QN; k++)
						y[u][k] = f[k];
				}
			} else if (i >= nq32 && i < total) {
				const int j = i - nq32, isv = j >= nkv, jj = isv ? j - nkv : j;
				const Heads<T> &h = isv ? a.v : a.k;
				const int e0 = jj % per * N;
				const T *p = h.in + t * h.in_ts + (jj / per) * h.in_hs;
				load_n<T, N, VEC>(p + e0, x[u]);
				if (LAYOUT == MOE_ROPE_HALVES && !isv && e0 < 2 * half) {
					// the partners of a key's values: in the other half
					if constexpr (VEC) {
						load_n<T, N, VEC>(p + (e0 < half ? e0 + half : e0 - half), y[u]);
					} else {
#pragma unroll
						for (int k = 0; k < N; k++) {
							const int e = e0 + k;
							y[u][k] = e < half ? to_f32(p[e + half])
								  : e < 2 * half ? to_f32(p[e - half]) : 0.0f;
						}
					}
				}
			}
		}
		if (!ready) {
			if (!find_row(a.b, t, row))
				return;   // the whole CTA: t is its own
			pos = a.pos ? a.pos[t] : row.row;
			if (half) {
				if (pos < 0 || pos >= a.r.max_position) {
					if (threadIdx.x == 0)
						atomicOr(a.b.err, kKvErrPos);
					return;
				}
				rope_angles(a.r, pos, cs);
			}
			__syncthreads();
			ready = true;
		}
#pragma unroll
		for (int u = 0; u < kAppendBatch; u++) {
			const int i = i0 + u * step;
			if (i < nq32) {
				if (i < nq) {
					const RopeItem<QN, LAYOUT> it(i % per_q, half);
					float f[QN], g[QN];
#pragma unroll
					for (int k = 0; k < QN; k++) {
						f[k] = x[u][k];
						g[k] = y[u][k];
					}
					it.apply(f, g, cs, half);
					T *p = a.q.out + t * a.q.out_ts + (i / per_q) * a.q.out_hs;
					store_n<T, QN, VEC>(p + it.e0, f);
					if (LAYOUT == MOE_ROPE_HALVES && it.e1 >= 0)
						store_n<T, QN, VEC>(p + it.e1, g);
				}
				continue;   // the whole warp: nq32 is a multiple of 32
			}
			const bool in = i < total;   // a block's lanes are in together
			const int j = in ? i - nq32 : 0, isv = j >= nkv, jj = isv ? j - nkv : j;
			const int head = jj / per, e0 = jj % per * N;
			if (!in) {
#pragma unroll
				for (int k = 0; k < N; k++)
					x[u][k] = 0.0f;
			}
			if (!isv && in) {
				if (LAYOUT == MOE_ROPE_PAIRS) {
#pragma unroll
					for (int k = 0; k < N; k += 2)
						if ((e0 + k) / 2 < half)
							turn(x[u][k], x[u][k + 1], cs[(e0 + k) / 2]);
				} else {
#pragma unroll
					for (int k = 0; k < N; k++) {
						const int e = e0 + k;
						if (e < half)
							turn(x[u][k], y[u][k], cs[e]);
						else if (e < 2 * half)
							turn(y[u][k], x[u][k], cs[e - half]);
					}
				}
			}
			__half scale;
			uint32_t by[N / 4];
			quantize_block<N>(x[u], scale, by);
			if (!in)
				continue;
			const int b = e0 / 32, sub = e0 % 32 / N;
			uint8_t *rec = record(a.p, row.page, head, isv);
			if (sub == 0)
				reinterpret_cast<__half *>(rec + ((D / 2) << a.p.page_log2))[row.at * nb + b] = scale;
			if (sub < L / 2) {
				uint8_t *dst = rec + row.at * (D / 2);
#pragma unroll
				for (int w = 0; w < N / 4; w++) {
					const int k4 = sub * (N / 4) + w;   // bytes 4 k4 .. of the block
					if (!isv) {
						*reinterpret_cast<uint32_t *>(dst + k4 * 4 * nb + 4 * b) = by[w];
					} else {
						uint16_t *d2 = reinterpret_cast<uint16_t *>(dst + 2 * k4 * 2 * nb + 2 * b);
						d2[0] = (uint16_t)by[w];
						d2[nb] = (uint16_t)(by[w] >> 16);
					}
				}
			}
		}
	}
}

template <typename T>
struct GatherArgs {
	BatchArgs b;
	PageArgs p;
	Heads<T> k, v;   // outputs only; n 0: none
};

// grid (token, slice): the values of the token's rows, code by code
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) gather_kernel(GatherArgs<T> a)
{
	constexpr int N = kVec<T>;
	const int t = blockIdx.x, D = a.p.head_len, nb = D / 32;
	const int per = D / N, nk = a.k.n * per, total = nk + a.v.n * per;
	TokenRow row;
	if (!find_row(a.b, t, row))
		return;
	for (int i = blockIdx.y * kAppendThreads + threadIdx.x; i < total;
	     i += gridDim.y * kAppendThreads) {
		const int isv = i >= nk, j = isv ? i - nk : i;
		const int head = j / per, e0 = j % per * N;
		const int b = e0 / 32, k0 = e0 % 16, up = e0 % 32 >= 16;
		const uint8_t *rec = record(a.p, row.page, head, isv);
		const float d = __half2float(
			reinterpret_cast<const __half *>(rec + ((D / 2) << a.p.page_log2))[row.at * nb + b]);
		const uint8_t *src = rec + row.at * (D / 2);
		float f[N];
#pragma unroll
		for (int w = 0; w < N / 4; w++) {
			const int k4 = k0 / 4 + w;
			uint32_t by;
			if (!isv) {
				by = *reinterpret_cast<const uint32_t *>(src + k4 * 4 * nb + 4 * b);
			} else {
				const uint16_t *s2 = reinterpret_cast<const uint16_t *>(src + 2 * k4 * 2 * nb + 2 * b);
				by = s2[0] | (uint32_t)s2[nb] << 16;
			}
			by = up ? by >> 4 : by;
#pragma unroll
			for (int k = 0; k < 4; k++)
				f[4 * w + k] = __fmul_rn((float)((int)(by >> (8 * k) & 15) - 8), d);
		}
		const Heads<T> &h = isv ? a.v : a.k;
		store_n<T, N, VEC>(h.out + t * h.out_ts + head * h.out_hs + e0, f);
	}
}

// slices of a token's items: enough CTAs for few tokens, one for many
unsigned slices(int64_t items, int64_t n_tokens)
{
	int64_t y = (items + kAppendThreads - 1) / kAppendThreads;
	const int64_t fill = (4 * (int64_t)sm_count() + n_tokens - 1) / n_tokens;
	y = y < fill ? y : fill;
	return (unsigned)(y < 1 ? 1 : y < 65535 ? y : 65535);
}

template <typename T, bool VEC, int LAYOUT>
cudaError_t launch_append_as(const AppendArgs<T> &a, cudaStream_t st)
{
	constexpr int N = kVec<T>, QN = VEC ? N : LAYOUT == MOE_ROPE_PAIRS ? 2 : 1;
	const int64_t items = (int64_t)a.q.n * RopeItem<QN, LAYOUT>::per_head(a.p.head_len, a.r.half) +
			      31 + 2 * (int64_t)a.p.KVH * (a.p.head_len / N);
	append_kernel<T, VEC, LAYOUT><<<dim3((unsigned)a.b.T, slices(items, a.b.T)), kAppendThreads,
					(a.r.half ? a.r.half : 1) * sizeof(float2), st>>>(a);
	return cudaGetLastError();
}

template <typename T>
cudaError_t launch_append(const AppendArgs<T> &a, int layout, bool vec, cudaStream_t st)
{
	if (layout == MOE_ROPE_PAIRS)
		return vec ? launch_append_as<T, true, MOE_ROPE_PAIRS>(a, st)
			   : launch_append_as<T, false, MOE_ROPE_PAIRS>(a, st);
	return vec && a.r.half % kVec<T> == 0 ? launch_append_as<T, true, MOE_ROPE_HALVES>(a, st)
					      : launch_append_as<T, false, MOE_ROPE_HALVES>(a, st);
}

template <typename T>
cudaError_t launch_gather(const GatherArgs<T> &a, bool vec, cudaStream_t st)
{
	const int64_t items = (int64_t)(a.k.n + a.v.n) * (a.p.head_len / kVec<T>);
	const dim3 grid((unsigned)a.b.T, slices(items, a.b.T));
	if (vec)
		gather_kernel<T, true><<<grid, kAppendThreads, 0, st>>>(a);
	else
		gather_kernel<T, false><<<grid, kAppendThreads, 0, st>>>(a);
	return cudaGetLastError();
}

int page_log2_of(int64_t page_size)
{
	for (int i = 4; i <= 8; i++)
		if (page_size == (int64_t)1 << i)
			return i;
	return -1;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

size_t moe_kv_page_bytes(int64_t page_size, int64_t n_kv_heads, int64_t head_len, int qtype)
{
	if (page_log2_of(page_size) < 0 || n_kv_heads <= 0 || n_kv_heads > 4096 ||
	    (head_len != 64 && head_len != 128 && head_len != 256) || qtype != MOE_Q4_0)
		return 0;
	return (size_t)(2 * n_kv_heads * page_size * (head_len / 2 + head_len / 16));
}

int moe_kv_create(moe_kv_cache **out, const moe_kv_desc *desc)
{
	const char *what = "moe_kv_create";
	if (!out || !desc)
		return kv_fail(MOE_ERR_INVALID, "%s: null argument", what);
	*out = nullptr;
	const moe_kv_desc &d = *desc;
	if (d.qtype != MOE_Q4_0)
		return kv_fail(MOE_ERR_UNSUPPORTED, "%s: type %d (MOE_Q4_0 only)", what, d.qtype);
	const size_t pb = moe_kv_page_bytes(d.page_size, d.n_kv_heads, d.head_len, d.qtype);
	if (!pb || d.n_pages <= 0 || d.n_pages > 0x7fffffff)
		return kv_fail(MOE_ERR_INVALID, "%s: %lld pages of %lld rows, %lld KV heads of %lld values "
			       "(page_size 16 .. 256, a power of two; head_len 64, 128 or 256)", what,
			       (long long)d.n_pages, (long long)d.page_size, (long long)d.n_kv_heads,
			       (long long)d.head_len);
	if ((uintptr_t)d.pages % 16)
		return kv_fail(MOE_ERR_INVALID, "%s: pages are not 16-byte aligned", what);
	if (int rc = ensure_library())
		return rc;
	moe_kv_cache *c = new (std::nothrow) moe_kv_cache();
	if (!c)
		return kv_fail(MOE_ERR_NOMEM, "%s: host memory", what);
	c->d = d;
	c->page_log2 = page_log2_of(d.page_size);
	c->page_bytes = pb;
	c->pages = static_cast<uint8_t *>(d.pages);
	cudaError_t e = cudaGetDevice(&c->device);
	if (e == cudaSuccess)
		e = cudaMalloc(&c->err, 256);
	if (e == cudaSuccess)
		e = cudaMemset(c->err, 0, 256);
	if (e == cudaSuccess && !c->pages) {
		e = cudaMalloc(&c->pages, (size_t)d.n_pages * pb);
		c->owned = e == cudaSuccess;
		if (c->owned)
			e = cudaMemset(c->pages, 0, (size_t)d.n_pages * pb);
	}
	if (e == cudaSuccess)
		e = cudaDeviceSynchronize();   // the caller's first use may be on any stream
	if (e != cudaSuccess) {
		moe_kv_destroy(c);
		return kv_cuda(e, what);
	}
	*out = c;
	return MOE_OK;
}

int moe_kv_destroy(moe_kv_cache *c)
{
	if (!c)
		return MOE_OK;
	DeviceGuard g(c->device);
	cudaError_t e = g.e;
	if (e == cudaSuccess) {
		e = cudaFree(c->err);
		if (c->owned) {
			const cudaError_t e2 = cudaFree(c->pages);
			e = e == cudaSuccess ? e2 : e;
		}
	}
	delete c;
	return e == cudaSuccess ? MOE_OK : kv_cuda(e, "moe_kv_destroy");
}

void *moe_kv_pages(moe_kv_cache *cache)
{
	return cache ? cache->pages : nullptr;
}

int moe_kv_append(moe_kv_cache *cache, const moe_kv_batch *batch, const moe_rope *rope,
		  const int32_t *pos, const moe_rows *k, const moe_rows *v, const moe_rows *q,
		  const moe_rows *q_out, void *stream)
{
	const char *what = "moe_kv_append";
	if (!cache)
		return kv_fail(MOE_ERR_INVALID, "%s: null cache", what);
	int rc = check_batch(what, cache, batch);
	if (rc != MOE_OK)
		return rc;
	const int64_t T = batch->n_tokens, D = cache->d.head_len, KVH = cache->d.n_kv_heads;
	if (!k || !v || (!q) != (!q_out))
		return kv_fail(MOE_ERR_INVALID, "%s: k or v missing, or q without q_out", what);
	if (rope && rope->device != cache->device)
		return kv_fail(MOE_ERR_INVALID, "%s: rope and cache are on devices %d and %d", what,
			       rope->device, cache->device);
	if (rope && rope->rot > D)
		return kv_fail(MOE_ERR_INVALID, "%s: rot %lld above head_len %lld", what,
			       (long long)rope->rot, (long long)D);
	const int type = k->type;
	rc = check_rows(what, "k", k, T, D, type, KVH, false);
	if (rc == MOE_OK)
		rc = check_rows(what, "v", v, T, D, type, KVH, false);
	if (rc == MOE_OK && q)
		rc = check_rows(what, "q", q, T, D, type, 0, false);
	if (rc == MOE_OK && q)
		rc = check_rows(what, "q_out", q_out, T, D, type, q->n_heads, true);
	if (rc == MOE_OK && q && q->n_heads % KVH)
		rc = kv_fail(MOE_ERR_INVALID, "%s: %lld heads over %lld KV heads", what,
			     (long long)q->n_heads, (long long)KVH);
	if (rc != MOE_OK)
		return rc;
	if (T == 0 || batch->n_seqs == 0)
		return MOE_OK;
	cudaStream_t st;
	if ((rc = resolve_stream(what, cache->device, stream, &st)) != MOE_OK)
		return rc;
	DeviceGuard g(cache->device);
	KV_CK(what, g.e);
	const bool vec = rows_vec16(k) && rows_vec16(v) && (!q || (rows_vec16(q) && rows_vec16(q_out)));
	auto go = [&](auto z) -> cudaError_t {
		using T_ = decltype(z);
		AppendArgs<T_> a;
		a.b = batch_args(cache, batch);
		a.p = page_args(cache);
		a.r = rope_args(rope);
		a.pos = pos;
		a.q = heads_of<T_>(q, q_out);
		a.k = heads_of<T_>(k, nullptr);
		a.v = heads_of<T_>(v, nullptr);
		return launch_append<T_>(a, rope ? rope->layout : MOE_ROPE_PAIRS, vec, st);
	};
	KV_CK(what, type == MOE_F32 ? go(float()) : type == MOE_F16 ? go(__half()) : go(__nv_bfloat16()));
	return MOE_OK;
}

int moe_kv_gather(moe_kv_cache *cache, const moe_kv_batch *batch, const moe_rows *k_out,
		  const moe_rows *v_out, void *stream)
{
	const char *what = "moe_kv_gather";
	if (!cache)
		return kv_fail(MOE_ERR_INVALID, "%s: null cache", what);
	int rc = check_batch(what, cache, batch);
	if (rc != MOE_OK)
		return rc;
	if (!k_out && !v_out)
		return kv_fail(MOE_ERR_INVALID, "%s: k_out and v_out missing", what);
	const int64_t T = batch->n_tokens, D = cache->d.head_len, KVH = cache->d.n_kv_heads;
	const int type = k_out ? k_out->type : v_out->type;
	if (k_out)
		rc = check_rows(what, "k_out", k_out, T, D, type, KVH, true);
	if (rc == MOE_OK && v_out)
		rc = check_rows(what, "v_out", v_out, T, D, type, KVH, true);
	if (rc != MOE_OK)
		return rc;
	if (T == 0 || batch->n_seqs == 0)
		return MOE_OK;
	cudaStream_t st;
	if ((rc = resolve_stream(what, cache->device, stream, &st)) != MOE_OK)
		return rc;
	DeviceGuard g(cache->device);
	KV_CK(what, g.e);
	const bool vec = (!k_out || rows_vec16(k_out)) && (!v_out || rows_vec16(v_out));
	auto go = [&](auto z) -> cudaError_t {
		using T_ = decltype(z);
		GatherArgs<T_> a;
		a.b = batch_args(cache, batch);
		a.p = page_args(cache);
		a.k = heads_of<T_>(nullptr, k_out);
		a.v = heads_of<T_>(nullptr, v_out);
		a.k.n = k_out ? (int)KVH : 0;
		a.v.n = v_out ? (int)KVH : 0;
		return launch_gather<T_>(a, vec, st);
	};
	KV_CK(what, type == MOE_F32 ? go(float()) : type == MOE_F16 ? go(__half()) : go(__nv_bfloat16()));
	return MOE_OK;
}

int moe_kv_status(moe_kv_cache *cache)
{
	const char *what = "moe_kv_status";
	if (!cache)
		return kv_fail(MOE_ERR_INVALID, "%s: null cache", what);
	DeviceGuard g(cache->device);
	KV_CK(what, g.e);
	KV_CK(what, cudaDeviceSynchronize());
	int32_t e = 0;
	KV_CK(what, cudaMemcpy(&e, cache->err, 4, cudaMemcpyDeviceToHost));
	if (!e)
		return MOE_OK;
	KV_CK(what, cudaMemset(cache->err, 0, 4));
	return kv_fail(MOE_ERR_INVALID, "%s:%s%s%s", what,
		       e & kKvErrBatch ? " q_start or kv_len out of range;" : "",
		       e & kKvErrPage ? " page outside the cache;" : "",
		       e & kKvErrPos ? " position out of range;" : "");
}

}  // extern "C"
