// rope.cu — rotary positions (moe_rope_*): angle tables and the kernel that
// turns the heads of a packed batch of tokens.
//
// Pair i of a head turns by angle(p, i) = p * f_i.  Far positions make large
// angles, whose fp32 form would have lost the turn's fraction (2^20 positions:
// 2^-4 radians), so angles are formed on the host in 64 bits.  One table row
// per position would be rot * 4 bytes each (64 MB for 128 k positions of 128
// values); instead p is split into p / 1024 and p % 1024, each with a table of
// 64-bit cosines and sines, and the kernel multiplies the two as complex
// numbers: 2 MB for a million positions, which stays in L2.
#include "kv.cuh"

#include <cmath>
#include <vector>

namespace moe {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeBatch = 4;   // items of a thread whose loads are in flight together

template <typename T>
struct RopeKernelArgs {
	RopeArgs r;
	const int32_t *pos;
	Heads<T> q, k;
	int head_len;
	int32_t *err;
};

// grid (token, slice of its items): bound by the bytes of q and k, read once
// and written once.  A thread's first loads leave before the position and the
// angles, which stand two dependent loads away, are known.
template <typename T, int N, bool VEC, int LAYOUT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeKernelArgs<T> a)
{
	extern __shared__ float2 cs[];
	const int t = blockIdx.x;
	const int per = RopeItem<N, LAYOUT>::per_head(a.head_len, a.r.half);
	const int nq = a.q.n * per, total = nq + a.k.n * per;
	const int step = gridDim.y * kRopeThreads;
	const int pos = a.pos[t];
	bool ready = false;
	for (int i0 = blockIdx.y * kRopeThreads + threadIdx.x; __syncthreads_or(i0 < total);
	     i0 += kRopeBatch * step) {
		float x[kRopeBatch][N], y[kRopeBatch][N];
#pragma unroll
		for (int u = 0; u < kRopeBatch; u++) {
			const int i = i0 + u * step;
			if (i < total) {
				const bool isq = i < nq;
				const Heads<T> &h = isq ? a.q : a.k;
				const int j = isq ? i : i - nq;
				const RopeItem<N, LAYOUT> it(j % per, a.r.half);
				const T *p = h.in + t * h.in_ts + (j / per) * h.in_hs;
				load_n<T, N, VEC>(p + it.e0, x[u]);
				if (LAYOUT == MOE_ROPE_HALVES && it.e1 >= 0)
					load_n<T, N, VEC>(p + it.e1, y[u]);
			}
		}
		if (!ready) {
			if (pos < 0 || pos >= a.r.max_position) {
				if (threadIdx.x == 0)
					atomicOr(a.err, kKvErrPos);
				return;   // the whole CTA: pos is the token's
			}
			rope_angles(a.r, pos, cs);
			__syncthreads();
			ready = true;
		}
#pragma unroll
		for (int u = 0; u < kRopeBatch; u++) {
			const int i = i0 + u * step;
			if (i < total) {
				const bool isq = i < nq;
				const Heads<T> &h = isq ? a.q : a.k;
				const int j = isq ? i : i - nq;
				const RopeItem<N, LAYOUT> it(j % per, a.r.half);
				it.apply(x[u], y[u], cs, a.r.half);
				T *p = h.out + t * h.out_ts + (j / per) * h.out_hs;
				store_n<T, N, VEC>(p + it.e0, x[u]);
				if (LAYOUT == MOE_ROPE_HALVES && it.e1 >= 0)
					store_n<T, N, VEC>(p + it.e1, y[u]);
			}
		}
	}
}

template <typename T, int N, bool VEC, int LAYOUT>
cudaError_t launch_rope_as(const RopeKernelArgs<T> &a, int64_t n_tokens, cudaStream_t st)
{
	const int per = RopeItem<N, LAYOUT>::per_head(a.head_len, a.r.half);
	const int64_t total = (int64_t)(a.q.n + a.k.n) * per;
	// few tokens: a token's items over several CTAs, each thread one item
	int64_t y = (total + kRopeThreads - 1) / kRopeThreads;
	const int64_t fill = (4 * (int64_t)sm_count() + n_tokens - 1) / n_tokens;
	y = y < fill ? y : fill;
	y = y < 65535 ? y : 65535;
	rope_kernel<T, N, VEC, LAYOUT>
		<<<dim3((unsigned)n_tokens, (unsigned)y), kRopeThreads, a.r.half * sizeof(float2), st>>>(a);
	return cudaGetLastError();
}

template <typename T>
cudaError_t launch_rope(const RopeKernelArgs<T> &a, int layout, bool vec, int64_t n_tokens,
			cudaStream_t st)
{
	constexpr int V = kVec<T>;
	if (layout == MOE_ROPE_PAIRS) {
		if (vec && a.head_len % V == 0)
			return launch_rope_as<T, V, true, MOE_ROPE_PAIRS>(a, n_tokens, st);
		return launch_rope_as<T, 2, false, MOE_ROPE_PAIRS>(a, n_tokens, st);
	}
	if (vec && a.head_len % V == 0 && a.r.half % V == 0)
		return launch_rope_as<T, V, true, MOE_ROPE_HALVES>(a, n_tokens, st);
	return launch_rope_as<T, 1, false, MOE_ROPE_HALVES>(a, n_tokens, st);
}

// radians a position of every pair (moe_rope_desc's definitions)
int frequencies(const moe_rope_desc &d, std::vector<double> &f)
{
	const double pi2 = 6.283185307179586476925;
	const int64_t half = d.rot / 2;
	f.resize((size_t)half);
	const double bf = d.beta_fast == 0 && d.beta_slow == 0 ? 32.0 : d.beta_fast;
	const double bs = d.beta_fast == 0 && d.beta_slow == 0 ? 1.0 : d.beta_slow;
	double low = 0, high = 0;
	if (d.scaling == MOE_ROPE_PARTS) {
		auto pair = [&](double turns) {
			return (double)d.rot * std::log(d.orig_context / (turns * pi2)) /
			       (2.0 * std::log(d.theta));
		};
		low = std::fmax(std::floor(pair(bf)), 0.0);
		high = std::fmin(std::ceil(pair(bs)), (double)d.rot - 1.0);
	}
	for (int64_t i = 0; i < half; i++) {
		double v = std::pow(d.theta, -2.0 * (double)i / (double)d.rot);
		if (d.freq_divisors) {
			const double q = d.freq_divisors[i];
			if (!std::isfinite(q) || q <= 0)
				return kv_fail(MOE_ERR_INVALID, "moe_rope_create: frequency divisor %lld is %g",
					       (long long)i, q);
			v /= q;
		}
		if (d.scaling == MOE_ROPE_LINEAR) {
			v /= d.factor;
		} else if (d.scaling == MOE_ROPE_PARTS) {
			const double r = std::fmin(std::fmax(((double)i - low) / std::fmax(high - low, 0.001),
							     0.0), 1.0);
			v = v / d.factor * r + v * (1.0 - r);
		} else if (d.scaling == MOE_ROPE_BANDS) {
			const double turns = d.orig_context * v / pi2;
			const double s = std::fmin(std::fmax((turns - d.low_freq) / (d.high_freq - d.low_freq),
							     0.0), 1.0);
			v = (1.0 - s) * v / d.factor + s * v;
		}
		f[(size_t)i] = v;
	}
	return MOE_OK;
}

int create_rope(moe_rope **out, const moe_rope_desc &d)
{
	if (d.rot <= 0 || d.rot % 2 || d.rot > 4096 || d.max_position <= 0 ||
	    d.max_position > (1 << 24))
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: rot %lld (even, up to 4096), "
			       "max_position %lld (up to 2^24)", (long long)d.rot,
			       (long long)d.max_position);
	if (d.layout != MOE_ROPE_PAIRS && d.layout != MOE_ROPE_HALVES)
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: layout %d", d.layout);
	if (d.scaling < MOE_ROPE_NONE || d.scaling > MOE_ROPE_BANDS)
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: scaling %d", d.scaling);
	if (!std::isfinite(d.theta) || d.theta <= 1.0)
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: theta %g", d.theta);
	if (d.scaling != MOE_ROPE_NONE && (!std::isfinite(d.factor) || d.factor < 1.0))
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: factor %g", d.factor);
	if (d.scaling >= MOE_ROPE_PARTS && (!std::isfinite(d.orig_context) || d.orig_context < 1.0))
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: orig_context %g", d.orig_context);
	if (d.scaling == MOE_ROPE_PARTS && !(d.beta_fast == 0 && d.beta_slow == 0) &&
	    !(d.beta_slow > 0 && d.beta_fast >= d.beta_slow && std::isfinite(d.beta_fast)))
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: beta_fast %g, beta_slow %g", d.beta_fast,
			       d.beta_slow);
	if (d.scaling == MOE_ROPE_BANDS &&
	    !(d.low_freq >= 0 && d.high_freq > d.low_freq && std::isfinite(d.high_freq)))
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: low_freq %g, high_freq %g", d.low_freq,
			       d.high_freq);
	if (!std::isfinite(d.magnitude) || d.magnitude < 0)
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: magnitude %g", d.magnitude);
	std::vector<double> f;
	if (int rc = frequencies(d, f))
		return rc;
	const double mag = d.magnitude != 0 ? d.magnitude
			   : d.scaling == MOE_ROPE_PARTS ? 0.1 * std::log(d.factor) + 1.0 : 1.0;
	const int64_t half = d.rot / 2, rows = (d.max_position + kRopeLow - 1) / kRopeLow;
	std::vector<double2> tab((size_t)((kRopeLow + rows) * half));
	for (int64_t p = 0; p < kRopeLow + rows; p++)
		for (int64_t i = 0; i < half; i++) {
			const bool low = p < kRopeLow;
			const double angle = (double)(low ? p : (p - kRopeLow) * kRopeLow) * f[(size_t)i];
			const double m = low ? 1.0 : mag;
			tab[(size_t)(p * half + i)] = make_double2(std::cos(angle) * m, std::sin(angle) * m);
		}
	if (int rc = ensure_library())
		return rc;
	moe_rope *r = new moe_rope();
	r->rot = d.rot;
	r->max_position = d.max_position;
	r->layout = d.layout;
	const size_t bytes = tab.size() * sizeof(double2);
	void *p = nullptr;
	cudaError_t e = cudaGetDevice(&r->device);
	if (e == cudaSuccess)
		e = cudaMalloc(&p, bytes + 256);
	r->lo = static_cast<double2 *>(p);
	if (e == cudaSuccess)
		e = cudaMemcpy(p, tab.data(), bytes, cudaMemcpyHostToDevice);
	if (e == cudaSuccess)
		e = cudaMemset(static_cast<uint8_t *>(p) + bytes, 0, 256);
	if (e == cudaSuccess)
		e = cudaDeviceSynchronize();   // the caller's first use may be on any stream
	if (e != cudaSuccess) {
		cudaFree(p);
		delete r;
		return kv_cuda(e, "moe_rope_create");
	}
	r->hi = r->lo + kRopeLow * half;
	r->err = reinterpret_cast<int32_t *>(static_cast<uint8_t *>(p) + bytes);
	*out = r;
	return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_rope_create(moe_rope **out, const moe_rope_desc *desc)
{
	if (!out || !desc)
		return kv_fail(MOE_ERR_INVALID, "moe_rope_create: null argument");
	*out = nullptr;
	try {
		return create_rope(out, *desc);
	} catch (const std::bad_alloc &) {
		return kv_fail(MOE_ERR_NOMEM, "moe_rope_create: host memory");
	}
}

int moe_rope_destroy(moe_rope *rope)
{
	if (!rope)
		return MOE_OK;
	DeviceGuard g(rope->device);
	const cudaError_t e = g.e == cudaSuccess ? cudaFree(rope->lo) : g.e;
	delete rope;
	return e == cudaSuccess ? MOE_OK : kv_cuda(e, "moe_rope_destroy");
}

int moe_rope_forward(moe_rope *rope, int64_t n_tokens, int64_t head_len, const int32_t *pos,
		     const moe_rows *q, const moe_rows *q_out, const moe_rows *k,
		     const moe_rows *k_out, void *stream)
{
	const char *what = "moe_rope_forward";
	if (!rope)
		return kv_fail(MOE_ERR_INVALID, "%s: null rope", what);
	if (n_tokens < 0 || n_tokens > 0x7fffffff || head_len < rope->rot || head_len > 4096 ||
	    head_len % 2)
		return kv_fail(MOE_ERR_INVALID, "%s: %lld tokens, head_len %lld (even, at least rot %lld, "
			       "up to 4096)", what, (long long)n_tokens, (long long)head_len,
			       (long long)rope->rot);
	if (!q || (!k) != (!k_out))
		return kv_fail(MOE_ERR_INVALID, "%s: q missing, or k without k_out", what);
	const int type = q->type;
	int rc = check_rows(what, "q", q, n_tokens, head_len, type, 0, false);
	if (rc == MOE_OK)
		rc = check_rows(what, "q_out", q_out, n_tokens, head_len, type, q->n_heads, true);
	if (rc == MOE_OK && k)
		rc = check_rows(what, "k", k, n_tokens, head_len, type, 0, false);
	if (rc == MOE_OK && k)
		rc = check_rows(what, "k_out", k_out, n_tokens, head_len, type, k->n_heads, true);
	if (rc != MOE_OK)
		return rc;
	if (n_tokens == 0)
		return MOE_OK;
	if (!pos)
		return kv_fail(MOE_ERR_INVALID, "%s: positions missing", what);
	cudaStream_t st;
	if ((rc = resolve_stream(what, rope->device, stream, &st)) != MOE_OK)
		return rc;
	DeviceGuard g(rope->device);
	KV_CK(what, g.e);
	const bool vec = rows_vec16(q) && rows_vec16(q_out) &&
			 (!k || (rows_vec16(k) && rows_vec16(k_out)));
	auto go = [&](auto z) -> cudaError_t {
		using T = decltype(z);
		RopeKernelArgs<T> a;
		a.r = rope_args(rope);
		a.pos = pos;
		a.q = heads_of<T>(q, q_out);
		a.k = heads_of<T>(k, k_out);
		a.head_len = (int)head_len;
		a.err = rope->err;
		return launch_rope<T>(a, rope->layout, vec, n_tokens, st);
	};
	KV_CK(what, type == MOE_F32 ? go(float()) : type == MOE_F16 ? go(__half()) : go(__nv_bfloat16()));
	return MOE_OK;
}

int moe_rope_status(moe_rope *rope)
{
	const char *what = "moe_rope_status";
	if (!rope)
		return kv_fail(MOE_ERR_INVALID, "%s: null rope", what);
	DeviceGuard g(rope->device);
	KV_CK(what, g.e);
	KV_CK(what, cudaDeviceSynchronize());
	int32_t e = 0;
	KV_CK(what, cudaMemcpy(&e, rope->err, 4, cudaMemcpyDeviceToHost));
	if (!e)
		return MOE_OK;
	KV_CK(what, cudaMemset(rope->err, 0, 4));
	return kv_fail(MOE_ERR_INVALID, "%s: a position was out of range", what);
}

}  // extern "C"
