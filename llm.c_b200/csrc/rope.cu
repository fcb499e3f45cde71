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
#include <type_traits>
#include <vector>

namespace moe {
namespace {

constexpr int kRopeThreads = 256, kRopeCtas = 4;

template <typename T>
struct RopeKernelArgs {
	RopeArgs r;
	const int32_t *pos;
	Heads<T> q, k;
	int n_tokens, head_len;
	TokenSplit cut;
	FastDiv half;          // pairs, to divide by
	int per_log2;          // rope_kernel: a row's lanes
	int rounds;            // a token's
	FastDiv per;           // rope_any_kernel: a head's items
	int32_t *err;
};

// the angles of the CTA's tokens, and whether their positions are in range
template <typename T>
__device__ __forceinline__ void token_angles(const RopeKernelArgs<T> &a, int t0, int nt, float2 *cs,
					     int *ok)
{
	const int half = a.r.half;
	for (int p = threadIdx.x; p < nt * half; p += kRopeThreads) {
		const int t = a.half.div(p), pos = a.pos[t0 + t];
		const bool in = pos >= 0 && pos < a.r.max_position;
		if (p == t * half) {
			ok[t] = in;
			if (!in)
				atomicOr(a.err, kKvErrPos);
		}
		if (in)
			cs[p] = rope_angle(a.r, pos, p - t * half);
	}
	__syncthreads();
}

// grid (token group, slice of a token's rounds): bound by the bytes of q and k, read
// once and written once.  A lane has 8 values of a row and the same place in every
// row it meets, so a token's angles stay in its registers.  The first loads leave
// before the positions and their angles, two dependent loads away, are known.
// 2048 tokens of 40 fp32 heads of 128: 17.2 us, 4.9 TB/s (rows at odd offsets, which are
// not streamed: 30.5); 16383 of 36 bf16 heads, half turning: 58.7 us, 5.1 TB/s, where
// conversions and addresses take 74 % of the issue slots.
template <typename T, bool VEC, int TURN>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) rope_kernel(const __grid_constant__ RopeKernelArgs<T> a)
{
	extern __shared__ uint4 smem[];
	__shared__ int ok[kGroupTokens];
	uint8_t *slots = reinterpret_cast<uint8_t *>(smem);
	float2 *cs = reinterpret_cast<float2 *>(   // [token][pair]
		slots + kRopeThreads / 32 * RowStream<T, VEC>::kWarpBytes);
	const int half = a.r.half, lane = threadIdx.x % 32;
	const int t0 = blockIdx.x * a.cut.tokens, nt = min(a.cut.tokens, a.n_tokens - t0);
	const int ml = 5 - a.per_log2;   // rows of a round, log2
	const int e0 = (lane & ((1 << a.per_log2) - 1)) * 8, sub = lane >> a.per_log2;
	const Rounds rr(a.cut, blockIdx.y);
	RowStream<T, VEC> stream(slots, 1 << a.per_log2);
	const int starts[2] = {rr.first, rr.start((a.q.n + (1 << ml) - 1) >> ml)};
	auto reader = [&](int s, int t) {
		const Heads<T> &h = s ? a.k : a.q;
		return RowReader<T, VEC>(stream, h, t0 + t, t < nt ? h.n : 0, ml, sub, e0, starts[s],
					 rr.step_log2);
	};
	// the first rows leave before the angles are known: of q, or of k in a warp
	// that has none of q
	const int early = reader(0, rr.token).w.left > 0 ? 0 : 1;
	{
		RowReader<T, VEC> first = early ? reader(1, rr.token) : reader(0, rr.token);
		first.begin();
	}
	token_angles(a, t0, nt, cs, ok);
	Turn8<TURN> tn(e0, half);
	for (int t = rr.token; t < nt; t += rr.token_step) {
		const bool good = ok[t];
		if (good)
			tn.angles(cs + t * half, e0, half);
#pragma unroll
		for (int s = 0; s < 2; s++) {
			const Heads<T> &h = s ? a.k : a.q;
			RowReader<T, VEC> in = reader(s, t);
			RowWalk<T> w = in.w;
			if (t == rr.token && s == early)
				in.skip_begun();
			else
				in.begin();
			T *out = h.out + (int64_t)(t0 + t) * h.out_ts + (int64_t)w.row * h.out_hs + e0;
			const int64_t d = (int64_t)w.step_rows * h.out_hs;
			for (; w.left > 0; w.left--, w.row += w.step_rows, out += d) {
				Raw<T, 8, VEC> x;
				stream.pop(x);
				float f[8];
				tn.apply(x, f);
				if (tn.turning)   // what does not turn keeps its bits
					x.set(f);
				stream.store(x, good && w.has() ? out : nullptr);
				in.next();
			}
		}
	}
	stream.finish();
}

// Rows that rope_kernel does not take: N = 2 values a thread where head_len is no
// multiple of 8, or its vectors no power of two up to 32; PairItems (TURN kTurnAny)
// where halves are no multiple of 8.  2048 tokens of 40 fp32 heads of 96: 24.6 us, 2.6 TB/s
// (in halves 27.8; 128 values with 100 turning in halves 41.6): bound by issue, an item's
// addresses for 8 bytes of it.
template <typename T, int TURN>
__global__ void __launch_bounds__(kRopeThreads) rope_any_kernel(const __grid_constant__ RopeKernelArgs<T> a)
{
	extern __shared__ float2 cs[];
	__shared__ int ok[kGroupTokens];
	const int half = a.r.half, lane = threadIdx.x % 32;
	const int t0 = blockIdx.x * a.cut.tokens, nt = min(a.cut.tokens, a.n_tokens - t0);
	const Rounds rr(a.cut, blockIdx.y);
	const int nq = a.q.n * a.per.n, items = nq + a.k.n * a.per.n;
	token_angles(a, t0, nt, cs, ok);
	for (int t = rr.token; t < nt; t += rr.token_step) {
		if (!ok[t])
			continue;
		for (int r = rr.first; r < a.rounds; r += rr.step()) {
			int j = r * 32 + lane;
			if (j >= items)
				break;
			const bool isq = j < nq;
			const Heads<T> &h = isq ? a.q : a.k;
			j -= isq ? 0 : nq;
			const int head = a.per.div(j), i = j - head * a.per.n;
			const T *in = h.in + (int64_t)(t0 + t) * h.in_ts + head * h.in_hs;
			T *out = h.out + (int64_t)(t0 + t) * h.out_ts + head * h.out_hs;
			if constexpr (TURN == kTurnAny) {
				PairItem<T> x;
				x.load(in, i, half);
				x.turn_store(out, i, cs + t * half, half);
			} else {
				Raw<T, 2, false> x;
				x.load(in + 2 * i);
				if (i < half) {
					float f[2];
					x.get(f);
					turn(f[0], f[1], cs[t * half + i]);
					x.set(f);
				}
				x.store(out + 2 * i);
			}
		}
	}
}

template <typename T>
cudaError_t launch_rope(RopeKernelArgs<T> a, int layout, bool vec, int64_t n_tokens, cudaStream_t st)
{
	const int turn = turn_of(layout, a.r.half), n8 = a.head_len / 8;
	// a row's vectors in lanes of one warp: 1, 2, 4 .. 32 of them
	const bool rows = turn != kTurnAny && a.head_len % 8 == 0 && n8 <= 32 && 32 % n8 == 0;
	a.n_tokens = (int)n_tokens;
	if (rows) {
		a.per_log2 = 0;
		while (1 << a.per_log2 < n8)
			a.per_log2++;
		const int m = 32 / n8;
		a.rounds = (a.q.n + m - 1) / m + (a.k.n + m - 1) / m;
	} else {
		const bool pairs = layout == MOE_ROPE_HALVES;
		a.per = FastDiv(pairs ? a.head_len - a.r.half : a.head_len / 2);
		a.rounds = ((a.q.n + a.k.n) * (int)a.per.n + 31) / 32;
	}
	const TokenSplit s = split_tokens(n_tokens, a.rounds, a.r.half);
	a.cut = s;
	a.half = FastDiv(a.r.half);
	const dim3 grid((unsigned)((n_tokens + s.tokens - 1) / s.tokens), 1u << s.slices_log2);
	const size_t angles = s.tokens * a.r.half * sizeof(float2);
	auto go = [&](auto kernel, size_t slots) -> cudaError_t {
		const size_t smem = angles + kRopeThreads / 32 * slots;
		if (cudaError_t e = ensure_smem(kernel, smem))
			return e;
		kernel<<<grid, kRopeThreads, smem, st>>>(a);
		return cudaGetLastError();
	};
	constexpr size_t slots = RowStream<T, true>::kWarpBytes;
	if (!rows)
		return layout == MOE_ROPE_HALVES ? go(rope_any_kernel<T, kTurnAny>, 0)
						 : go(rope_any_kernel<T, kTurnPairs>, 0);
	if (turn == kTurnPairs)
		return vec ? go(rope_kernel<T, true, kTurnPairs>, slots) : go(rope_kernel<T, false, kTurnPairs>, 0);
	return vec ? go(rope_kernel<T, true, kTurnHalves>, slots) : go(rope_kernel<T, false, kTurnHalves>, 0);
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
	if (n_tokens < 0 || n_tokens > (1 << 30) || head_len < rope->rot || head_len > 4096 ||
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
	if (!pos || (uintptr_t)pos % 4)
		return kv_fail(MOE_ERR_INVALID, "%s: positions missing or not aligned", what);
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
	KV_CK(what, cudaDeviceSynchronize());   // before a call on any stream records the next
	return kv_fail(MOE_ERR_INVALID, "%s: a position was out of range", what);
}

}  // extern "C"
