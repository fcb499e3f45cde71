// kvcache.cu — the paged key/value cache in 4 bits (moe_kv_*): handles,
// append with the rotation on the way, read-back, and the row moves of the
// whole model's cache rotation.  The layout of a page is described in
// moe_b200.h; kvattn.cu reads it.
#include "kv.cuh"

namespace moe {
namespace {

constexpr int kAppendThreads = 256, kAppendCtas = 4;
constexpr int kGatherBatch = 4;

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

__device__ __forceinline__ int64_t record_bytes(const PageArgs &a)   // of a head's K, or V
{
	return (a.head_len / 2 + a.head_len / 16) << a.page_log2;
}
__device__ __forceinline__ uint8_t *record(const PageArgs &a, uint8_t *page, int head, int which)
{
	return page + (2 * head + which) * record_bytes(a);
}

template <typename T>
struct AppendArgs {
	BatchArgs b;
	PageArgs p;
	RopeArgs r;
	const int32_t *pos;   // or NULL: the cache rows
	Heads<T> q, k, v;     // k, v: inputs only; q.n 0: none
	TokenSplit cut;
	FastDiv half;         // pairs, to divide by
	int per_log2;         // a row's lanes
	FastDiv per_q;        // kTurnAny: a query head's items
};

constexpr int kLanes = 4;   // of a 32-value block: 8 values each

// A lane's 8 values of a block whose 4 lanes stand side by side: the block's scale
// and codes (moe_kv_desc), two 4-bit codes to a byte with the lane that holds the
// values 16 further on.  The two lower lanes return the block's bytes 0 .. 7 and
// 8 .. 15.
__device__ __forceinline__ void quantize_block(const float (&x)[8], __half &scale, uint32_t (&by)[2])
{
	float hi = x[0], lo = x[0];
	bool bad = false;
#pragma unroll
	for (int k = 0; k < 8; k++) {
		hi = fmaxf(hi, x[k]);
		lo = fminf(lo, x[k]);
		bad |= !(fabsf(x[k]) <= 3.402823466e38f);
	}
#pragma unroll
	for (int o = 1; o < kLanes; o *= 2) {
		hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
		lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
	}
	const unsigned any = __ballot_sync(0xffffffffu, bad);
	bad = (any >> (threadIdx.x % 32 / kLanes * kLanes)) & ((1u << kLanes) - 1);
	// the value of the largest magnitude takes code 0 (-8): a step of m / 8
	// where a symmetric code would have m / 7
	const float m = hi >= -lo ? hi : lo;
	scale = __float2half_rn(fminf(fmaxf(__fmul_rn(m, -0.125f), -65504.0f), 65504.0f));
	const float d = __half2float(scale);
	const float inv = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
	if (d == 0.0f || bad)   // one zero: which zero m is depends on the order of its zeros
		scale = __ushort_as_half(bad ? 0x7fff : 0);
#pragma unroll
	for (int w = 0; w < 2; w++) {
		uint32_t c = 0;
#pragma unroll
		for (int k = 0; k < 4; k++) {
			const int code = min(max(__float2int_rn(__fmul_rn(x[4 * w + k], inv)), -8), 7) + 8;
			c |= (uint32_t)(bad ? 8 : code) << (8 * k);
		}
		by[w] = c | __shfl_xor_sync(0xffffffffu, c, kLanes / 2) << 4;
	}
}

// The layout's 4-byte words of a pair of blocks (2 b, 2 b + 1), whose 8 lanes stand
// side by side: a K word is 4 bytes of one block (word s of the lane's block, s the
// lane's place in it), a V word 2 bytes of each block (word p, p the lane's place in
// the pair).  So a row is written and read in whole words by neighbouring lanes.
__device__ __forceinline__ int row_word_at(int b, int nb, bool isv)
{
	const int p = threadIdx.x % (2 * kLanes), s = threadIdx.x % kLanes;
	return isv ? p * 2 * nb + 2 * (b & ~1) : s * 4 * nb + 4 * b;
}

// that word, out of the bytes that the blocks' lower lanes hold (8 each)
__device__ __forceinline__ uint32_t row_word(const uint32_t (&by)[2], bool isv)
{
	const int lane = threadIdx.x % 32, p = lane % (2 * kLanes), s = lane % kLanes;
	const int byte = isv ? 2 * p : 4 * s;
	const int src = (isv ? lane - p : lane - s) + byte / 8;
	const uint32_t x0 = __shfl_sync(0xffffffffu, by[0], src), x1 = __shfl_sync(0xffffffffu, by[1], src);
	const int two = (src + kLanes) & 31;   // a V word's other block
	const uint32_t y0 = __shfl_sync(0xffffffffu, by[0], two), y1 = __shfl_sync(0xffffffffu, by[1], two);
	const uint32_t x = byte & 4 ? x1 : x0, y = byte & 4 ? y1 : y0;
	return isv ? __byte_perm(x, y, byte & 2 ? 0x7632 : 0x5410) : x;
}

// the bytes that hold a lane's own 8 values out of the words
__device__ __forceinline__ void row_bytes(uint32_t word, int b, bool isv, uint32_t (&by)[2])
{
	const int lane = threadIdx.x % 32, p = lane % (2 * kLanes), s = lane % kLanes;
#pragma unroll
	for (int i = 0; i < 2; i++) {
		const int k4 = s % 2 * 2 + i;   // bytes 4 k4 .. of the block
		const int src = isv ? lane - p + 2 * k4 : lane - s + k4;
		const uint32_t x = __shfl_sync(0xffffffffu, word, src);
		const uint32_t y = __shfl_sync(0xffffffffu, word, (src + 1) & 31);
		by[i] = isv ? __byte_perm(x, y, b & 1 ? 0x7632 : 0x5410) : x;
	}
}

// grid (token group, slice of a token's rounds): per token the query heads are turned
// and written, then the key heads turned and quantized, the value heads quantized.
// Bound by bytes for prompts (q, k, v in, q and 0.5625 bytes a value out) and by
// latency for decode batches: the first rows leave for the registers, then come the
// tokens' sequences (a search of two rounds), angles and pages, each a dependent
// load.  A lane has 8 values of a row and the same place in every row it meets, so a
// token's angles stay in its registers (kTurnAny: halves that are no multiple of 8,
// value by value).  64 decode tokens 4.9 us; 512 fp32 tokens of 16 + 32 heads 10.3; 16383 ragged
// fp16 ones of 28 + 8 heads of 64 42.8 (72 % of the issue slots: maxima and bytes by
// shuffles, a rounding a value).
template <typename T, bool VEC, int TURN>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) append_kernel(const __grid_constant__ AppendArgs<T> a)
{
	extern __shared__ uint4 smem[];
	struct Token {
		int ok, pos, at;
		uint8_t *page;
	};
	__shared__ Token toks[kGroupTokens];
	uint8_t *slots = reinterpret_cast<uint8_t *>(smem);
	float2 *cs = reinterpret_cast<float2 *>(   // [token][pair]
		slots + kAppendThreads / 32 * RowStream<T, VEC>::kWarpBytes);
	const int half = a.r.half, D = a.p.head_len, nb = D / 32;
	const int t0 = blockIdx.x * a.cut.tokens, nt = min(a.cut.tokens, a.b.T - t0);
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	const int ml = 5 - a.per_log2;   // rows of a round, log2
	const int e0 = (lane & ((1 << a.per_log2) - 1)) * 8, sub = lane >> a.per_log2;
	const Rounds rr(a.cut, blockIdx.y);
	// (kTurnAny: the queries go by items of their own)
	constexpr int Q = TURN == kTurnAny ? 0 : 1;
	RowStream<T, VEC> stream(slots, 1 << a.per_log2);
	const int q_rounds = Q ? (a.q.n + (1 << ml) - 1) >> ml : 0;
	const int kv_rounds = (a.k.n + (1 << ml) - 1) >> ml;
	const int starts[3] = {rr.first, rr.start(q_rounds), rr.start(q_rounds + kv_rounds)};
	auto reader = [&](int s, int t) {
		const Heads<T> &h = s == 0 ? a.q : s == 1 ? a.k : a.v;
		const int n = t >= nt || (s == 0 && !Q) ? 0 : h.n;
		return RowReader<T, VEC>(stream, h, t0 + t, n, ml, sub, e0, starts[s], rr.step_log2);
	};
	// the first rows leave before the tokens' places are known: of the first sort
	// that the warp has rows of
	const int early = reader(0, rr.token).w.left > 0 ? 0 : reader(1, rr.token).w.left > 0 ? 1 : 2;
	{
		RowReader<T, VEC> first = early == 0   ? reader(0, rr.token)
					  : early == 1 ? reader(1, rr.token)
						       : reader(2, rr.token);
		first.begin();
	}
	if (warp == 0) {
		TokenRow row = find_rows(a.b, t0, nt);
		int pos = 0;
		if (row.ok) {
			pos = a.pos ? a.pos[t0 + lane] : row.row;
			if (half && (pos < 0 || pos >= a.r.max_position)) {
				row.ok = 0;
				atomicOr(a.b.err, kKvErrPos);
			}
		}
		if (lane < nt) {
			toks[lane].ok = row.ok;
			toks[lane].pos = pos;
			toks[lane].at = row.at;
			toks[lane].page = a.p.pages + (row.ok ? row.page * a.p.page_bytes : 0);
		}
	} else if (warp == 1 && blockIdx.x == 0 && blockIdx.y == 0) {
		check_sequences(a.b);
	}
	__syncthreads();
	if (half) {
		for (int p = threadIdx.x; p < nt * half; p += kAppendThreads) {
			const int u = a.half.div(p);
			if (toks[u].ok)
				cs[p] = rope_angle(a.r, toks[u].pos, p - u * half);
		}
		__syncthreads();
	}
	const int b = e0 / 32;
	const int64_t kv_bytes = record_bytes(a.p);
	Turn8<Q ? TURN : kTurnPairs> tn(e0, half);
	for (int t = rr.token; t < nt; t += rr.token_step) {
		const bool good = toks[t].ok;
		const int64_t tok = t0 + t;
		const float2 *tcs = cs + t * half;
		T *qo = a.q.out + tok * a.q.out_ts;
		if constexpr (Q) {
			if (good)
				tn.angles(tcs, e0, half);
			RowReader<T, VEC> q = reader(0, t);
			RowWalk<T> w = q.w;
			if (t == rr.token && early == 0)
				q.skip_begun();
			else
				q.begin();
			qo += e0 + (int64_t)w.row * a.q.out_hs;
			const int64_t d = (int64_t)w.step_rows * a.q.out_hs;
			for (; w.left > 0; w.left--, w.row += w.step_rows, qo += d) {
				Raw<T, 8, VEC> x;
				stream.pop(x);
				float f[8];
				tn.apply(x, f);
				if (tn.turning)   // what does not turn keeps its bits
					x.set(f);
				stream.store(x, good && w.has() ? qo : nullptr);
				q.next();
			}
		} else if (good) {
			const int items = a.q.n * a.per_q.n;
			for (int j = rr.first * 32 + lane; j < items; j += rr.step() * 32) {
				const int head = a.per_q.div(j), i = j - head * a.per_q.n;
				PairItem<T> x;
				x.load(a.q.in + tok * a.q.in_ts + head * a.q.in_hs, i, half);
				x.turn_store(qo + head * a.q.out_hs, i, tcs, half);
			}
		}
		const int at = toks[t].at;
		const int codes_at = at * (D / 2), scale_at = ((D / 2) << a.p.page_log2) + (at * nb + b) * 2;
#pragma unroll
		for (int isv = 0; isv < 2; isv++) {
			RowReader<T, VEC> in = reader(1 + isv, t);
			RowWalk<T> w = in.w;
			if (t == rr.token && early == 1 + isv)
				in.skip_begun();
			else
				in.begin();
			uint8_t *rec = toks[t].page + (2 * w.row + isv) * kv_bytes;
			const int64_t d = 2 * w.step_rows * kv_bytes;
			const int word_at = codes_at + row_word_at(b, nb, isv);
			for (; w.left > 0; w.left--, w.row += w.step_rows, rec += d) {
				Raw<T, 8, VEC> x;
				stream.pop(x);
				float f[8];
				if (Q && !isv)
					tn.apply(x, f);
				else
					x.get(f);
				in.next();
				if (!Q && !isv && good && e0 < 2 * half && w.has()) {
					const T *src = a.k.in + tok * a.k.in_ts + w.row * a.k.in_hs + e0;
#pragma unroll
					for (int i = 0; i < 8; i++) {
						const int e = e0 + i;
						if (e >= 2 * half)
							break;
						float g = to_f32(src[e < half ? i + half : i - half]);
						if (e < half)
							turn(f[i], g, tcs[e]);
						else
							turn(g, f[i], tcs[e - half]);
					}
				}
				__half scale;
				uint32_t by[2];
				quantize_block(f, scale, by);
				const uint32_t word = row_word(by, isv);
				if (good && w.has()) {
					if (lane % kLanes == 0)
						*reinterpret_cast<__half *>(rec + scale_at) = scale;
					*reinterpret_cast<uint32_t *>(rec + word_at) = word;
				}
			}
		}
	}
	stream.finish();
}

template <typename T>
struct GatherArgs {
	BatchArgs b;
	PageArgs p;
	Heads<T> k, v;   // outputs only; n 0: none
	TokenSplit cut;
	int per_log2, k_rounds, v_rounds;
};

// grid (token group, slice of a token's rounds): the values of the tokens' rows, code
// by code, kGatherBatch rounds in flight together.  16384 rows of 8 KV heads of 128 to bf16:
// 23 us, 3.7 TB/s of codes in and values out.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) gather_kernel(const __grid_constant__ GatherArgs<T> a)
{
	__shared__ uint8_t *page_of[kGroupTokens];
	__shared__ int row_of[kGroupTokens];
	const int D = a.p.head_len, nb = D / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	const int t0 = blockIdx.x * a.cut.tokens, nt = min(a.cut.tokens, a.b.T - t0);
	if (warp == 0) {
		const TokenRow row = find_rows(a.b, t0, nt);
		if (lane < nt) {
			page_of[lane] = row.ok ? a.p.pages + row.page * a.p.page_bytes : nullptr;
			row_of[lane] = row.at;
		}
	} else if (warp == 1 && blockIdx.x == 0 && blockIdx.y == 0) {
		check_sequences(a.b);
	}
	__syncthreads();
	const int rows = 32 >> a.per_log2;
	const int e0 = (lane & ((1 << a.per_log2) - 1)) * 8, sub = lane >> a.per_log2, b = e0 / 32;
	const Rounds rr(a.cut, blockIdx.y);
	const int n = a.k_rounds + a.v_rounds;
	for (int t = rr.token; t < nt; t += rr.token_step) {
		uint8_t *page = page_of[t];
		if (!page)
			continue;
		const int row = row_of[t];
		T *ko = a.k.out + (int64_t)(t0 + t) * a.k.out_ts + e0;
		T *vo = a.v.out + (int64_t)(t0 + t) * a.v.out_ts + e0;
		for (int r0 = rr.first; r0 < n; r0 += kGatherBatch * rr.step()) {
			uint32_t word[kGatherBatch];
			__half scale[kGatherBatch];
#pragma unroll
			for (int u = 0; u < kGatherBatch; u++) {
				const int r = r0 + u * rr.step();
				const bool isv = r >= a.k_rounds;
				const int head = (isv ? r - a.k_rounds : r) * rows + sub;
				word[u] = 0;
				scale[u] = __half();
				if (r >= n || head >= a.p.KVH)
					continue;
				const uint8_t *rec = record(a.p, page, head, isv);
				scale[u] = reinterpret_cast<const __half *>(
					rec + ((D / 2) << a.p.page_log2))[row * nb + b];
				word[u] = *reinterpret_cast<const uint32_t *>(rec + row * (D / 2) +
									      row_word_at(b, nb, isv));
			}
#pragma unroll
			for (int u = 0; u < kGatherBatch; u++) {
				const int r = r0 + u * rr.step();
				const bool isv = r >= a.k_rounds;
				const int head = (isv ? r - a.k_rounds : r) * rows + sub;
				uint32_t by[2];
				row_bytes(word[u], b, isv, by);
				if (r >= n || head >= a.p.KVH)
					continue;
				const float d = __half2float(scale[u]);
				float f[8];
#pragma unroll
				for (int w = 0; w < 2; w++) {
					const uint32_t x = e0 % 32 >= 16 ? by[w] >> 4 : by[w];
#pragma unroll
					for (int k = 0; k < 4; k++)
						f[4 * w + k] = __fmul_rn((float)((int)(x >> (8 * k) & 15) - 8), d);
				}
				Raw<T, 8, VEC> x;
				x.set(f);
				x.store(isv ? vo + head * a.v.out_hs : ko + head * a.k.out_hs);
			}
		}
	}
}

int log2_of(int n)
{
	int l = 0;
	while (1 << l < n)
		l++;
	return l;
}

template <typename T, bool VEC, int TURN>
cudaError_t launch_append_as(AppendArgs<T> a, cudaStream_t st)
{
	const int D = a.p.head_len, m = 32 / (D / 8);
	a.per_q = FastDiv(D - a.r.half);
	a.per_log2 = log2_of(D / 8);
	const int q_rounds = TURN == kTurnAny ? (a.q.n * (D - a.r.half) + 31) / 32 : (a.q.n + m - 1) / m;
	const TokenSplit s = split_tokens(a.b.T, q_rounds + 2 * ((a.p.KVH + m - 1) / m), a.r.half);
	a.cut = s;
	a.half = FastDiv(a.r.half ? a.r.half : 1);
	const size_t smem = (s.tokens * a.r.half) * sizeof(float2) +
			    kAppendThreads / 32 * RowStream<T, VEC>::kWarpBytes;
	if (cudaError_t e = ensure_smem(append_kernel<T, VEC, TURN>, smem))
		return e;
	append_kernel<T, VEC, TURN><<<dim3((unsigned)((a.b.T + s.tokens - 1) / s.tokens),
					   1u << s.slices_log2), kAppendThreads, smem, st>>>(a);
	return cudaGetLastError();
}

template <typename T>
cudaError_t launch_append(const AppendArgs<T> &a, int layout, bool vec, cudaStream_t st)
{
	switch (turn_of(layout, a.r.half)) {
	case kTurnPairs:
		return vec ? launch_append_as<T, true, kTurnPairs>(a, st)
			   : launch_append_as<T, false, kTurnPairs>(a, st);
	case kTurnHalves:
		return vec ? launch_append_as<T, true, kTurnHalves>(a, st)
			   : launch_append_as<T, false, kTurnHalves>(a, st);
	default:
		return vec ? launch_append_as<T, true, kTurnAny>(a, st)
			   : launch_append_as<T, false, kTurnAny>(a, st);
	}
}

template <typename T>
cudaError_t launch_gather(GatherArgs<T> a, bool vec, cudaStream_t st)
{
	const int m = 32 / (a.p.head_len / 8), rounds = (a.p.KVH + m - 1) / m;
	a.per_log2 = log2_of(a.p.head_len / 8);
	a.k_rounds = a.k.n ? rounds : 0;
	a.v_rounds = a.v.n ? rounds : 0;
	const TokenSplit s = split_tokens(a.b.T, a.k_rounds + a.v_rounds, 0);
	a.cut = s;
	const dim3 grid((unsigned)((a.b.T + s.tokens - 1) / s.tokens), 1u << s.slices_log2);
	if (vec)
		gather_kernel<T, true><<<grid, kAppendThreads, 0, st>>>(a);
	else
		gather_kernel<T, false><<<grid, kAppendThreads, 0, st>>>(a);
	return cudaGetLastError();
}

// grid (rows, KV heads, layers x K and V): a row's codes in 8-byte words, its scales in
// 2-byte ones (a full cache's rotation, once in half a context of decode steps)
__global__ void kv_move_q4_kernel(uint8_t *pages, int64_t layer_bytes, int64_t page_bytes, int HL,
				  int page_log2, int from, int to)
{
	const int64_t half = (int64_t)(HL / 2 + HL / 16) << page_log2;
	uint8_t *base = pages + (blockIdx.z / 2) * layer_bytes + (2 * blockIdx.y + blockIdx.z % 2) * half;
	auto at = [&](int r) { return base + (r >> page_log2) * page_bytes; };
	const int src = from + blockIdx.x, dst = to + blockIdx.x, mask = (1 << page_log2) - 1;
	const int words = HL / 16, scales = HL / 32;   // of a row
	const int sc = (HL / 2) << page_log2;
	if ((int)threadIdx.x < words)
		reinterpret_cast<uint64_t *>(at(dst) + (dst & mask) * (HL / 2))[threadIdx.x] =
			reinterpret_cast<const uint64_t *>(at(src) + (src & mask) * (HL / 2))[threadIdx.x];
	else if ((int)threadIdx.x < words + scales)
		reinterpret_cast<uint16_t *>(at(dst) + sc + (dst & mask) * scales * 2)[threadIdx.x - words] =
			reinterpret_cast<const uint16_t *>(at(src) + sc +
							   (src & mask) * scales * 2)[threadIdx.x - words];
}

int page_log2_of(int64_t page_size)
{
	for (int i = 4; i <= 8; i++)
		if (page_size == (int64_t)1 << i)
			return i;
	return -1;
}

}  // namespace

cudaError_t launch_kv_move_q4(uint8_t *pages, int64_t layer_bytes, int64_t page_bytes, int L,
			      int KVH, int HL, int page_log2, int from, int to, int rows,
			      cudaStream_t st)
{
	if (rows <= 0 || from == to)
		return cudaSuccess;
	kv_move_q4_kernel<<<dim3(rows, KVH, 2 * L), 32, 0, st>>>(pages, layer_bytes, page_bytes, HL,
								  page_log2, from, to);
	return cudaGetLastError();
}

int kv_create(moe_kv_cache **out, const moe_kv_desc *desc, int32_t *err)
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
	c->err = err;
	if (e == cudaSuccess && !err) {
		e = cudaMalloc(&c->err, 256);
		c->err_owned = e == cudaSuccess;
		if (c->err_owned)
			e = cudaMemset(c->err, 0, 256);
	}
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

int kv_status(const char *what, int32_t e)
{
	if (!e)
		return MOE_OK;
	if (e & kKvErrWait)
		return kv_fail(MOE_ERR_TIMEOUT, "%s: a bounded wait in the attention kernel expired", what);
	return kv_fail(MOE_ERR_INVALID, "%s:%s%s%s", what,
		       e & kKvErrBatch ? " q_start or kv_len out of range;" : "",
		       e & kKvErrPage ? " page outside the cache;" : "",
		       e & kKvErrPos ? " position out of range;" : "");
}

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
	return kv_create(out, desc, nullptr);
}

int moe_kv_destroy(moe_kv_cache *c)
{
	if (!c)
		return MOE_OK;
	DeviceGuard g(c->device);
	cudaError_t e = g.e;
	if (e == cudaSuccess) {
		if (c->err_owned)
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
	if ((uintptr_t)pos % 4)
		return kv_fail(MOE_ERR_INVALID, "%s: positions are not aligned", what);
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
	KV_CK(what, cudaDeviceSynchronize());   // before a call on any stream records the next
	return kv_status(what, e);
}

}  // extern "C"
