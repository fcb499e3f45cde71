// kvwide.cu — attention over the paged 4-bit cache for many queries (prompts, chunks): an
// item is a CTA's, 256 query rows (query token x head of the group) of a KV head and a
// run of 32-row key tiles, with the products on tcgen05.mma.
//
//   S   = Q K^T       Q as fp16 (a power of two a row); K = code * scale exactly, as two
//                     fp16 numbers (below), fp32 sums in tensor memory
//   O  += P V         P = exp2(S - max) in fp16, V = code * scale in fp16
//
// K: a scale's 11 bits are cut into 8 and 3, and a code (-8 .. 7) times either is an fp16
// number exactly, down to the smallest scale: two rows of B a key, whose scores the rows
// add.  (Codes alone, with a sum a block and its scale in fp32, cost the rows four times
// the tensor memory reads and a shared-memory read of 128 scales a tile: 148 us for a
// 2048-token prompt.)  From 2^13 on a product may not fit (-8 * 2^13 is above 65504): keys
// with such a scale take theirs times 2^-4, and their scores 2^4.
// V's scales are rounded in: a weight and a value are rounded to fp16 once each, as often
// as kvattn.cu rounds (weight, then weight * scale).  They are brought below 2 by a power
// of two a block, the largest so far to [1, 2).
//
// 19 warps: thread r of the first 256 has query row r and its softmax (two groups of 128,
// whose TMEM lanes and columns are their own), 128 take K's codes apart, 128 take V's
// apart, a warp a group issues its products, and one fetches the tiles.  What waits for
// what:
//
//   copier   tile j: for the stagers to be done with tile j - 4
//   stagers  tile j there; its K: for S of tile j - 2; V: for O += P V of tile j - 2 (K, V
//            and their barriers are double)
//   issuer   S of tile i + 1 (double too): for its K and the rows' reads of S of tile
//            i - 1, so it runs beside the softmax of tile i; then O += P V of tile i: for
//            P and V
//   rows     S of tile i to registers (and O += P V of tile i - 2, issued before it,
//            done); softmax; P (double) to shared memory; where the maximum or V's
//            factors move, O += P V of tile i - 1
//
// A barrier's next phase needs what follows a wait for this one, so none is missed.
// All operands are rows of 64 bytes (32 values) in the 64-byte swizzle, so a block is a
// slice.
#include "expert_core.cuh"
#include "kvattn.cuh"

#include <type_traits>

namespace moe {
using namespace kva;
namespace {

constexpr int kGroup = 128, kGroups = kWideRows / kGroup;   // rows of one MMA
constexpr int kStagers = 128;                               // of K, and as many of V
constexpr int kWideIssuer = kWideRows + 2 * kStagers, kWideCopier = kWideIssuer + 32 * kGroups;
constexpr int kWideThreads = kWideCopier + 32;
constexpr int kRing = 4, kAhead = 2;                        // tiles as they lie in the page; on their way

template <int HL>
struct WideLayout {
	static constexpr int NB = HL / 32;
	static constexpr int kQ = kGroup * 64;               // a block's slice of a group's Q
	static constexpr int kK = 2 * kAttnTile * 64;        // a block's rows of high parts, then low ones
	static constexpr int kV = HL * 64, kP = kGroup * 64;
	static constexpr int kOffK = kGroups * NB * kQ, kOffV = kOffK + 2 * NB * kK, kOffP = kOffV + 2 * kV;
	static constexpr int kOffRaw = kOffP + 2 * kGroups * kP;
	// a tile as it lies in the page; V's rows by fours with 16 bytes between, so that 8
	// lanes that read 4 rows each find them in banks of their own
	static constexpr int kCodes = kAttnTile * HL / 2, kScales = kAttnTile * NB * 2;
	static constexpr int kRawKS = kCodes, kRawV = kCodes + kScales;
	static constexpr int kRawVS = kRawV + kCodes + kAttnTile / 4 * 16, kRaw = kRawVS + kScales;
	static constexpr int kBytes = kOffRaw + kRing * kRaw, kSmem = kBytes + 1024;   // to align the base
	// columns: a group's two S (high parts' scores, then low ones') and its O
	static constexpr int kTmemS = 2 * kAttnTile, kTmemO = 2 * kTmemS, kTmemGroup = 256, kTmem = kGroups * kTmemGroup;
	static_assert(kRaw % 16 == 0 && kTmemO + HL <= kTmemGroup && kTmem <= 512, "sizes");
};

// rows of 64 bytes, 64-byte swizzle: start >> 4, 8 rows 512 bytes on, version 1, layout 4
__device__ __forceinline__ uint64_t slice_desc(uint32_t addr)
{
	return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)1 << 16) | ((uint64_t)(512 >> 4) << 32) |
	       ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
}
// byte of a slice where 16-byte chunk c of row r stands
__device__ __forceinline__ int slice_at(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }

// fp16 x fp16 -> fp32, both K-major, M 128
template <int N>
__device__ __forceinline__ void mma_slice(uint32_t d, uint32_t a, uint32_t b, bool first)
{
	constexpr uint32_t desc = (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kGroup >> 4) << 24);
#pragma unroll
	for (int k = 0; k < 2; k++)
		asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
			     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
			     "l"(slice_desc(a + 32 * k)), "l"(slice_desc(b + 32 * k)), "r"(desc),
			     "r"(k || !first ? 1u : 0u)
			     : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar)
{
	asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
			     smem_addr(bar))
		     : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

#define KV_R16(r, o)                                                                                       \
	"=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]),        \
		"=r"(r[o + 6]), "=r"(r[o + 7]), "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]),           \
		"=r"(r[o + 11]), "=r"(r[o + 12]), "=r"(r[o + 13]), "=r"(r[o + 14]), "=r"(r[o + 15])

// 16 columns at a (and, in the same wait, at a + step)
__device__ __forceinline__ void tmem_two(uint32_t a, uint32_t b, uint32_t (&r)[32])
{
	asm volatile(
		"tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
		"tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
		"tcgen05.wait::ld.sync.aligned;"
		: KV_R16(r, 0), KV_R16(r, 16)
		: "r"(a), "r"(b));
}
__device__ __forceinline__ void tmem_one(uint32_t a, uint32_t (&r)[16])
{
	asm volatile(
		"tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
		"tcgen05.wait::ld.sync.aligned;"
		: KV_R16(r, 0)
		: "r"(a));
}
__device__ __forceinline__ void tmem_store16(uint32_t a, const uint32_t *r)
{
	asm volatile(
		"tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
		"r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
		"r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(a)
		: "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two fp32 multiply-adds
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
	float2 d;
	asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
	    "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
	    : "=f"(d.x), "=f"(d.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
	return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
	float2 d;
	asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
	    "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
	    : "=f"(d.x), "=f"(d.y)
	    : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
	return d;
}

// a pair of codes less 8, exact: from low nibbles of bytes 0 and 2 (1024 + c in fp16), from
// high ones (1024 + 16 c)
__device__ __forceinline__ __half2 pair_low(uint32_t w)
{
	return __hadd2(bits_h2((w & 0x000f000fu) | 0x64006400u), bits_h2(0xe408e408u));   // - 1032
}
__device__ __forceinline__ __half2 pair_high(uint32_t w)
{
	return __hfma2(bits_h2((w & 0x00f000f0u) | 0x64006400u), bits_h2(0x2c002c00u),    // / 16
		       bits_h2(0xd480d480u));                                             // - 72
}

template <int NW>
__device__ __forceinline__ void words_of(const uint8_t *p, uint32_t (&w)[NW])
{
	if constexpr (NW == 4) {
		const uint4 v = *reinterpret_cast<const uint4 *>(p);
		w[0] = v.x;
		w[1] = v.y;
		w[2] = v.z;
		w[3] = v.w;
	} else if constexpr (NW == 2) {
		const uint2 v = *reinterpret_cast<const uint2 *>(p);
		w[0] = v.x;
		w[1] = v.y;
	} else {
		w[0] = *reinterpret_cast<const uint32_t *>(p);
	}
}

// grid: the plan's items.  A 2048-token prompt (32 heads on 8, 34 GFLOP) takes 128 us, 268
// TFLOP/s (kvattn.cu's kernel: 193).  A tile of 256 x 32 scores takes 2600 clocks: its
// products are 700 of the tensor cores', the rest is latency, of which the rows' steps
// (a wait that finds its barrier done 200 to 300, scores 360, softmax 860, the hand-over
// of P 330) and the issue of small products one after the other (120 each) are the most.
template <typename T, int HL, bool FOLD>
__global__ void __launch_bounds__(kWideThreads, 1) kv_wide_kernel(const __grid_constant__ AttnArgs a)
{
	using WL = WideLayout<HL>;
	constexpr int NB = WL::NB;
	extern __shared__ uint8_t smem_raw[];
	__shared__ uint64_t bar_s[kGroups][2], p_ready[kGroups][2], bar_o[kGroups][2], s_free[kGroups][2];
	__shared__ uint64_t k_ready[2], v_ready[2], k_free[2], v_free[2], raw_ready[kRing], raw_free[kRing];
	__shared__ int have_s[kRing];   // halves of a tile that are there
	__shared__ uint32_t tmem_at;
	// what the stagers found in a tile's V scales: factors for the sums so far, keys whose
	// scale of a block is not finite; and the factors that the sums have by now
	struct Found {
		int have;         // halves of the tile that are there; 4: of its keys some are large
		uint32_t large;   // those whose K is held times 2^-4
		uint32_t shrinks, bads;
		float shrink[NB];
		uint32_t bad[NB];
		float unit[NB];   // (tiles where sums move to the record) v_unit as of the tile
	};
	__shared__ Found found_s[2];
	__shared__ float v_unit[NB];
	uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
	const uint32_t sa = smem_addr(sm);
	const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
	const int tid = threadIdx.x % 128;   // of a group's rows, or the stagers of K or V
	const bool row_warp = threadIdx.x < kWideRows, copier = threadIdx.x >= kWideCopier;
	const bool issuer = threadIdx.x >= kWideIssuer && !copier;
	const bool k_stager = !row_warp && threadIdx.x < kWideRows + kStagers;

	griddep_launch_dependents();
	Item it;
	if (!cta_item<kWideRows, true>(a, blockIdx.x, it))
		return;
	const int groups = (it.rows + kGroup - 1) / kGroup;   // that have rows
	if (threadIdx.x == 0) {
		for (int b = 0; b < 2; b++) {
			mbar_init(&k_ready[b], kStagers / 32);
			mbar_init(&v_ready[b], kStagers / 32);
			mbar_init(&k_free[b], groups);
			mbar_init(&v_free[b], groups);
		}
		for (int b = 0; b < kRing; b++) {
			mbar_init(&raw_ready[b], 1);
			mbar_init(&raw_free[b], 2 * kStagers / 32);
		}
		for (int g = 0; g < kGroups; g++) {
			for (int b = 0; b < 2; b++) {
				mbar_init(&bar_s[g][b], 1);
				mbar_init(&p_ready[g][b], kGroup / 32);
				mbar_init(&bar_o[g][b], 1);
				mbar_init(&s_free[g][b], kGroup / 32);
			}
		}
		fence_mbar_init();
	}
	if (threadIdx.x < NB)   // (rows of an item without tiles wait for nothing but the barrier below)
		v_unit[threadIdx.x] = 1.0f / 32768.0f;
	if (warp == 0) {
		asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
				     smem_addr(&tmem_at)),
			     "r"(WL::kTmem));
		asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
	}

	// ---- the key tiles t0, t0 + 1, ..: lane l of the copier keeps the pages of the next
	// 32 of them (two where a page is half a tile)
	const int ntile = it.t1 - it.t0;
	const int32_t *table = a.b.table + it.b * a.b.table_stride;
	const int P = 1 << a.b.page_log2;
	const bool small = P < kAttnTile;
	auto key0 = [&](int i) { return (it.t0 + i) * kAttnTile; };
	// which halves of a tile hold rows that the item sees
	auto needs = [&](int k0) -> int {
		return (k0 < it.hi && k0 + 16 > it.lo ? 1 : 0) | (k0 + 16 < it.hi && k0 + 32 > it.lo ? 2 : 0);
	};
	int page_a = -1, page_b = -1;   // of tile (i & ~31) + lane
	auto load_pages = [&](int i) {
		page_a = page_b = -1;
		if (i + lane < ntile) {
			const int k0 = key0(i + lane), need = needs(k0);
			const bool wa = need & (small ? 1 : 3), wb = small && (need & 2);
			if (wa)
				page_a = table[k0 >> a.b.page_log2];
			if (wb)
				page_b = table[(k0 + 16) >> a.b.page_log2];
			const bool ba = (unsigned)page_a >= (unsigned)a.b.n_pages;
			const bool bb = (unsigned)page_b >= (unsigned)a.b.n_pages;
			if ((wa && ba) || (wb && bb))
				atomicOr(a.b.err, kKvErrPage);
			page_a = ba ? -1 : page_a;
			page_b = bb ? -1 : page_b;
		}
	};
	const int half_rec = (HL / 2 + HL / 16) << a.b.page_log2;
	const uint8_t *head_pages = a.pages + 2 * (int64_t)it.kvh * half_rec;
	// tile i's bytes on their way to its place in the ring, 16 bytes a lane and copy
	constexpr int CH = WL::kCodes / 16, CR = HL / 32;   // chunks of a tile's codes, of a row's
	constexpr int SC = WL::kScales / 16;                // of its scales
	auto issue = [&](int i) {
		if ((i & 31) == 0)
			load_pages(i);
		const int k0 = key0(i);
		const int pa = __shfl_sync(0xffffffffu, page_a, i & 31);
		const int pb = small ? __shfl_sync(0xffffffffu, page_b, i & 31) : pa;
		const int have = needs(k0) & ((pa >= 0 ? 1 : 0) | (pb >= 0 ? 2 : 0));
		const uint32_t st = sa + WL::kOffRaw + i % kRing * WL::kRaw;
		const int r0 = k0 & (P - 1);
#pragma unroll
		for (int h = 0; h < 2; h++) {
			if (!(have >> h & 1))
				continue;
			// the half's first row: in the tile's page, or another page's first
			const int at = small ? 0 : r0 + 16 * h;
			const uint8_t *k = head_pages + (int64_t)(h ? pb : pa) * a.page_bytes;
			const uint8_t *codes = k + at * (HL / 2) + lane * 16;
			const uint8_t *scales = k + ((HL / 2) << a.b.page_log2) + at * NB * 2;
#pragma unroll
			for (int x = 0; x < CH / 64; x++) {
				const int j = h * (CH / 2) + 32 * x + lane, row = j / CR;
				copy16(st + j * 16, codes + 512 * x);
				copy16(st + WL::kRawV + row / 4 * 16 + j * 16, codes + 512 * x + half_rec);
			}
			const int isv = lane >= SC / 2, j = lane - isv * (SC / 2);
			if (lane < SC)
				copy16(st + (isv ? WL::kRawVS : WL::kRawKS) + (h * (SC / 2) + j) * 16,
				       scales + isv * half_rec + j * 16);
		}
		return have;
	};
	const int group = row_warp ? threadIdx.x / kGroup : issuer ? warp - kWideIssuer / 32 : 0;
	const int row = group * kGroup + tid;
	// ---- the row's query: block b's values in the order that the codes come apart in
	const bool row_used = row_warp && row < it.rows;
	const int qi = row_used ? a.by_g.div(it.r0 + row) : 0;
	const int row_pos = it.kv - it.n + qi;   // the cache row at which it stands
	float qs = 0.0f;                         // scores to exponents of 2
	if (row_warp) {
		const T *p = static_cast<const T *>(a.q) + (it.s0 + qi) * a.q_ts +
			     (it.kvh * (int64_t)a.G + (it.r0 + row - qi * a.G)) * a.q_hs;
		auto four = [&](int e, float (&x)[4]) {
			if (!row_used) {
				x[0] = x[1] = x[2] = x[3] = 0.0f;
			} else if (a.q_vec) {
				const uint2 v = *reinterpret_cast<const uint2 *>(p + e);
				const T *t = reinterpret_cast<const T *>(&v);
#pragma unroll
				for (int k = 0; k < 4; k++)
					x[k] = to_f32(t[k]);
			} else {
#pragma unroll
				for (int k = 0; k < 4; k++)
					x[k] = to_f32(p[e + k]);
			}
		};
		// the largest magnitude, by its bits: an infinity or a NaN is above all
		uint32_t bits = 0;
#pragma unroll 8
		for (int e = 0; e < HL; e += 4) {
			float x[4];
			four(e, x);
#pragma unroll
			for (int k = 0; k < 4; k++)
				bits = max(bits, __float_as_uint(x[k]) & 0x7fffffffu);
		}
		const bool bad = bits >= 0x7f800000u;
		const int e2 = bits == 0 || bad ? 0 : 13 - ilogbf(__uint_as_float(bits));   // -114 .. 162
		const float up = __int_as_float((127 + min(e2, 127)) << 23);
		const float up2 = e2 > 127 ? __int_as_float(e2 << 23) : 1.0f;
		// a query with an infinity or a NaN has no finite scores: NaN
		qs = bad ? __int_as_float(0x7fffffff) : scalbnf(a.scale2, -e2);
#pragma unroll
		for (int b = 0; b < NB; b++)
#pragma unroll
			for (int c = 0; c < 4; c++) {
				float x[4], y[4];
				four(32 * b + 4 * c, x);
				four(32 * b + 16 + 4 * c, y);
#pragma unroll
				for (int k = 0; k < 4; k++) {
					x[k] = bad ? 0.0f : x[k] * up2 * up;
					y[k] = bad ? 0.0f : y[k] * up2 * up;
				}
				*reinterpret_cast<uint4 *>(sm + (group * NB + b) * WL::kQ + slice_at(tid, c)) =
					make_uint4(pack_h2(x[0], x[2]), pack_h2(x[1], x[3]),
						   pack_h2(y[0], y[2]), pack_h2(y[1], y[3]));
			}
	}
	// rows of the cache that it sees
	const int see_lo = row_used && a.window ? max(0, row_pos - a.window + 1) : 0;
	const int see_hi = !row_used ? 0 : a.causal ? min(it.kv, row_pos + 1) : it.kv;
	// rows that every query of the item sees
	const int first_row = it.kv - it.n + a.by_g.div(it.r0);
	const int last_row = it.kv - it.n + a.by_g.div(it.r0 + it.rows - 1);
	const int all_lo = a.window ? max(it.lo, last_row - a.window + 1) : it.lo;
	const int all_hi = a.causal ? min(it.kv, first_row + 1) : it.kv;

	// ---- codes to operands
	// whether a key's scales have one of 2^13 or more: a matter of its own row, so what the
	// others hold (behind the sequence's end, or behind a query) counts for nothing
	auto k_is_large = [&](const uint32_t (&d)[NB / 2]) -> bool {
		bool large = false;
#pragma unroll
		for (int k = 0; k < NB / 2; k++)
			large |= !__hble2(__habs2(bits_h2(d[k])), bits_h2(0x6fff6fffu));
		return large;
	};
	auto stage_k = [&](int i) {
		const uint8_t *raw = sm + WL::kOffRaw + i % kRing * WL::kRaw;
		const int j = tid / 4, c = tid % 4;   // key row, 16-byte chunk of its slices
		uint32_t w[NB], d[NB / 2];
		words_of<NB>(raw + j * (HL / 2) + c * 4 * NB, w);
		words_of<NB / 2>(raw + WL::kRawKS + j * NB * 2, d);
		if (k_is_large(d))
#pragma unroll
			for (int k = 0; k < NB / 2; k++)
				d[k] = h2_bits(__hmul2(bits_h2(d[k]), bits_h2(0x2c002c00u)));   // 2^-4
		uint8_t *kd = sm + WL::kOffK + (i & 1) * NB * WL::kK + slice_at(j, c);
#pragma unroll
		for (int b = 0; b < NB; b++) {
			const uint32_t top = d[b / 2] & 0xfff8fff8u;   // 8 bits of each
			const __half2 rest = __hsub2(bits_h2(d[b / 2]), bits_h2(top));   // 3 bits
			const __half2 hi = b & 1 ? __high2half2(bits_h2(top)) : __low2half2(bits_h2(top));
			const __half2 lo = b & 1 ? __high2half2(rest) : __low2half2(rest);
			const __half2 x[4] = {pair_low(w[b]), pair_low(w[b] >> 8), pair_high(w[b]), pair_high(w[b] >> 8)};
			uint32_t h[4], l[4];
#pragma unroll
			for (int k = 0; k < 4; k++) {
				h[k] = h2_bits(__hmul2(x[k], hi));
				l[k] = h2_bits(__hmul2(x[k], lo));
			}
			*reinterpret_cast<uint4 *>(kd + b * WL::kK) = make_uint4(h[0], h[1], h[2], h[3]);
			*reinterpret_cast<uint4 *>(kd + b * WL::kK + WL::kK / 2) = make_uint4(l[0], l[1], l[2], l[3]);
		}
	};
	// V's factors, a power of two a block, two to a word, and the largest scales that
	// they hold below 2 (2 over the factor).  Every stager's warp has the same ones: a lane
	// looks at a key's scales
	uint32_t v_fac[NB / 2], v_top[NB / 2];
#pragma unroll
	for (int k = 0; k < NB / 2; k++) {
		v_fac[k] = 0x78007800u;   // 2^15
		v_top[k] = 0x04000400u;   // 2^-14
	}
	auto stage_v = [&](int i, int have) {
		const uint8_t *raw = sm + WL::kOffRaw + i % kRing * WL::kRaw;
		const int k0 = key0(i);
		uint32_t bad[NB];   // keys whose scale of a block is not finite
		bool any_bad = false;
		uint32_t use;   // keys with rows that some query sees: the others may hold anything
		{
			uint32_t w[NB / 2];
			words_of<NB / 2>(raw + WL::kRawVS + lane * NB * 2, w);
			const bool in = (have >> (lane / 16) & 1) && k0 + lane >= it.lo && k0 + lane < it.hi;
			use = __ballot_sync(0xffffffffu, in);
			bool grow = false;
#pragma unroll
			for (int k = 0; k < NB / 2; k++)
				grow |= !__hble2(__habs2(bits_h2(w[k])), bits_h2(v_top[k]));
			if (__any_sync(0xffffffffu, grow && in)) {
				const bool tell = tid == 0;
				Found &f = found_s[i & 1];
				uint32_t bads = 0;
				float shrink[NB];
#pragma unroll
				for (int b = 0; b < NB; b++) {
					const float v = fabsf(half_of(w[b / 2], b & 1));
					const bool not_finite = in && !(v <= 65504.0f);
					bad[b] = __ballot_sync(0xffffffffu, not_finite);
					bads |= bad[b];
					const float top = warp_max(in && !not_finite ? v : 0.0f);
					const float had = half_of(v_fac[b / 2], b & 1);
					shrink[b] = 1.0f;
					if (top * had > 2.0f) {
						const float r = scalbnf(1.0f, -min(ilogbf(top), 15));
						shrink[b] = r / had;
						v_fac[b / 2] = set_half(v_fac[b / 2], b & 1, r);
						v_top[b / 2] = set_half(v_top[b / 2], b & 1, 2.0f / r);
						if (tell)
							v_unit[b] = 1.0f / r;
					}
					if (tell) {
						f.shrink[b] = shrink[b];
						f.bad[b] = bad[b];
					}
				}
				any_bad = bads != 0;
				if (tell) {
					f.shrinks = 1;
					f.bads = bads;
				}
			} else if (tid == 0) {
				found_s[i & 1].shrinks = found_s[i & 1].bads = 0;
			}
			if (FOLD && i % kFold == 0 && tid == 0)
#pragma unroll
				for (int b = 0; b < NB; b++)
					found_s[i & 1].unit[b] = 1.0f / half_of(v_fac[b / 2], b & 1);
		}
		// 4 keys x 8 values: byte (block b0 or b0 + 1, value k or k + 1, and 16 further on)
		const int g = lane % 8, w = tid / 8;
		if (w >= HL / 8)
			return;
		constexpr int H2 = NB / 2;
		const int k = w / H2 * 2, b0 = w % H2 * 2;
		const uint8_t *vp = raw + WL::kRawV + 4 * g * (HL / 2) + g * 16 + 4 * w;
		uint32_t x[4], s[4];
#pragma unroll
		for (int j = 0; j < 4; j++) {
			x[j] = *reinterpret_cast<const uint32_t *>(vp + j * (HL / 2));
			s[j] = *reinterpret_cast<const uint32_t *>(raw + WL::kRawVS + (4 * g + j) * NB * 2 + b0 * 2);
		}
		const uint32_t mine = use >> (4 * g) & 15;
		if (mine != 15 || any_bad) {
#pragma unroll
			for (int j = 0; j < 4; j++) {
				uint32_t keep = mine >> j & 1 ? 0xffffffffu : 0u;
#pragma unroll
				for (int b = 0; b < NB; b++)
					if (any_bad && (bad[b] >> (4 * g + j) & 1) && b / 2 == b0 / 2)
						keep &= b & 1 ? 0x0000ffffu : 0xffff0000u;
				s[j] &= keep;
			}
		}
		uint32_t fac = v_fac[0];
		if (NB == 4)
			fac = b0 ? v_fac[NB / 2 - 1] : v_fac[0];
#pragma unroll
		for (int j = 0; j < 4; j++)
			s[j] = h2_bits(__hmul2(bits_h2(s[j]), bits_h2(fac)));
		uint8_t *vd = sm + WL::kOffV + (i & 1) * WL::kV + g % 2 * 8;
		const int odd = lane / 8 & 1;   // the lanes of two words store odd and even rows in turn
#pragma unroll
		for (int tt = 0; tt < 4; tt++) {
			const int blk = tt / 2, t = tt ^ odd;   // byte of the words: block b0 + blk
			const uint32_t sel = t | (4 + t) << 8;
			const __half2 s01 = bits_h2(__byte_perm(s[0], s[1], blk ? 0x7632 : 0x5410));
			const __half2 s23 = bits_h2(__byte_perm(s[2], s[3], blk ? 0x7632 : 0x5410));
			const uint32_t x01 = __byte_perm(x[0], x[1], sel), x23 = __byte_perm(x[2], x[3], sel);
			const int n = 32 * (b0 + blk) + k + (t & 1);
			*reinterpret_cast<uint2 *>(vd + slice_at(n, g / 2)) =
				make_uint2(h2_bits(__hmul2(pair_low(x01), s01)), h2_bits(__hmul2(pair_low(x23), s23)));
			*reinterpret_cast<uint2 *>(vd + slice_at(n + 16, g / 2)) =
				make_uint2(h2_bits(__hmul2(pair_high(x01), s01)),
					   h2_bits(__hmul2(pair_high(x23), s23)));
		}
	};

	bool failed = false;
	auto wait = [&](uint64_t *bar, int phase) {
		if (!failed && !mbar_wait(bar, (uint32_t)phase & 1)) {
			failed = true;
			atomicOr(a.b.err, kKvErrWait);
		}
	};
	// what the warp wrote (and read of tensor memory) is the tensor cores'
	auto give = [&](uint64_t *bar) {
		fence_proxy_async();   // generic writes before the tensor cores' reads
		fence_before();
		__syncwarp();
		if (lane == 0)
			mbar_arrive(bar);
	};
	uint32_t tg = 0;   // the group's columns
	auto issue_s = [&](int i) {
#pragma unroll
		for (int b = 0; b < NB; b++)
			mma_slice<2 * kAttnTile>(tg + (i & 1) * WL::kTmemS, sa + (group * NB + b) * WL::kQ,
						 sa + WL::kOffK + ((i & 1) * NB + b) * WL::kK, b == 0);
		mma_commit(&bar_s[group][i & 1]);
		mma_commit(&k_free[i & 1]);
	};

	fence_proxy_async();   // Q
	fence_before();
	__syncthreads();
	fence_after();
	const uint32_t tmem = tmem_at;
	tg = tmem + group * WL::kTmemGroup;

	float bias = kNoMax, l = 0.0f;   // kLift - the largest score so far, and the weights' sum
	uint32_t poison = 0;             // blocks of V of which the row has seen a NaN
	const uint32_t tq = tg + ((uint32_t)(32 * (warp % 4)) << 16);   // the warp's lanes
	if (copier) {
		for (int j = 0; j < ntile + kAhead; j++) {
			if (j < ntile) {
				if (j >= kRing)
					wait(&raw_free[j % kRing], j / kRing - 1);
				const int have = issue(j);
				if (lane == 0)
					have_s[j % kRing] = have;
			}
			copies_commit();
			copies_wait<kAhead>();   // tile j - kAhead is there
			__syncwarp();
			if (j >= kAhead && lane == 0)
				mbar_arrive(&raw_ready[(j - kAhead) % kRing]);
		}
	} else if (issuer) {
		if (lane == 0 && ntile > 0 && group < groups) {
			wait(&k_ready[0], 0);
			fence_after();
			if (!failed)
				issue_s(0);
			for (int i = 0; i < ntile; i++) {
				if (i + 1 < ntile) {
					wait(&k_ready[(i + 1) & 1], (i + 1) / 2);
					if (i > 0)
						wait(&s_free[group][(i - 1) & 1], (i - 1) / 2);
					fence_after();
					if (!failed)
						issue_s(i + 1);
				}
				wait(&v_ready[i & 1], i / 2);
				wait(&p_ready[group][i & 1], i / 2);
				fence_after();
				if (!failed) {
					mma_slice<HL>(tg + WL::kTmemO, sa + WL::kOffP + (2 * group + (i & 1)) * WL::kP,
						      sa + WL::kOffV + (i & 1) * WL::kV, i == 0);
					mma_commit(&bar_o[group][i & 1]);
					mma_commit(&v_free[i & 1]);
				}
			}
		}
	} else if (!row_warp) {
#pragma unroll 1
		for (int j = 0; j < ntile; j++) {
			wait(&raw_ready[j % kRing], j / kRing);
			if (j >= 2)
				wait(k_stager ? &k_free[j & 1] : &v_free[j & 1], j / 2 - 1);
			if (k_stager) {
				stage_k(j);
			} else {
				const int have = have_s[j % kRing];
				stage_v(j, have);
				if (tid / 32 == 0) {
					uint32_t d[NB / 2];
					words_of<NB / 2>(sm + WL::kOffRaw + j % kRing * WL::kRaw + WL::kRawKS + lane * NB * 2, d);
					const uint32_t large = __ballot_sync(0xffffffffu, k_is_large(d));
					if (tid == 0) {
						found_s[j & 1].have = have | (large ? 4 : 0);
						found_s[j & 1].large = large;
					}
				}
			}
			give(k_stager ? &k_ready[j & 1] : &v_ready[j & 1]);
			if (lane == 0)
				mbar_arrive(&raw_free[j % kRing]);
		}
	} else if (group < groups) {
		// sums so far by a factor of the row's own, and of the blocks'
		auto rescale = [&](float f, const float *blocks) {
#pragma unroll 1
			for (int b = 0; b < NB; b++) {
				uint32_t r[32];
				const uint32_t at = tq + WL::kTmemO + 32 * b;
				tmem_two(at, at + 16, r);
				const float fb = blocks ? blocks[b] : f;
#pragma unroll
				for (int k = 0; k < 32; k++)
					r[k] = __float_as_uint(__uint_as_float(r[k]) * fb);
				tmem_store16(at, r);
				tmem_store16(at + 16, r + 16);
			}
			tmem_store_wait();
		};
		// the row's record: sums in true size, bias, weights' sum
		float *pp = a.part + ((int64_t)blockIdx.x * a.part_rows + row) * (HL + 4);
		// the sums of the tiles before to it, on top of what is there (!first): times f and the
		// blocks' factors, in true size
		auto fold = [&](bool first, float f, const float *blocks, const float *unit) {
			float g = 0.0f;
			if (!first && row_used) {
				g = ex2(bias - pp[HL]);   // (the maximum only rises)
				l = fmaf(pp[HL + 1], g, l);
			}
			if (row_used)
				*reinterpret_cast<float2 *>(pp + HL) = make_float2(bias, l);
			l = 0.0f;
#pragma unroll 1
			for (int e = 0; e < HL; e += 16) {
				uint32_t r[16];
				const uint32_t at = tq + WL::kTmemO + e;
				tmem_one(at, r);
				const float u = f * unit[e / 32] * (blocks ? blocks[e / 32] : 1.0f);
				if (row_used) {
#pragma unroll
					for (int k = 0; k < 16; k += 4) {
						float4 *d = reinterpret_cast<float4 *>(pp + e + k);
						const float4 w = first ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : *d;
						*d = make_float4(fmaf(w.x, g, __uint_as_float(r[k]) * u),
								 fmaf(w.y, g, __uint_as_float(r[k + 1]) * u),
								 fmaf(w.z, g, __uint_as_float(r[k + 2]) * u),
								 fmaf(w.w, g, __uint_as_float(r[k + 3]) * u));
					}
				}
#pragma unroll
				for (int k = 0; k < 16; k++)
					r[k] = 0;
				tmem_store16(at, r);
			}
			tmem_store_wait();
		};
		const float none = -__int_as_float(0x7f800000);
		auto tile = [&](auto full_c, const float2 (&s)[kAttnTile / 2], int i, uint32_t seen) {
			constexpr bool FULL = decltype(full_c)::value;   // every row sees all of it
			const Found &fd = found_s[i & 1];
			// ---- weights, times 2^kLift over the largest so far
			float2 t[kAttnTile / 2];
			auto weigh = [&]() {
#pragma unroll
				for (int j = 0; j < kAttnTile / 2; j++) {
					t[j] = fma2(s[j], make_float2(qs, qs), make_float2(bias, bias));
					if (!FULL) {
						t[j].x = seen >> (2 * j) & 1 ? t[j].x : none;
						t[j].y = seen >> (2 * j + 1) & 1 ? t[j].y : none;
					}
				}
			};
			weigh();
			float m[4] = {none, none, none, none};
#pragma unroll
			for (int j = 0; j < kAttnTile / 2; j++)
				m[j % 4] = fmaxf(fmaxf(m[j % 4], t[j].x), t[j].y);
			m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
			const bool raise = __any_sync(0xffffffffu, m[0] > kLift + kLag);
			float f = 1.0f;
			if (raise) {
				float top = none;
#pragma unroll
				for (int j = 0; j < kAttnTile / 2; j++) {
					top = fmaxf(top, FULL || (seen >> (2 * j) & 1) ? s[j].x * qs : none);
					top = fmaxf(top, FULL || (seen >> (2 * j + 1) & 1) ? s[j].y * qs : none);
				}
				const float next = fminf(bias, kLift - top);
				f = ex2(next - bias);
				bias = next;
				l *= f;
				weigh();
			}
			uint32_t w[kAttnTile / 2];
			float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
			for (int j = 0; j < kAttnTile / 2; j++) {
				const float2 p = make_float2(ex2(t[j].x), ex2(t[j].y));
				sum[j % 2] = add2(sum[j % 2], p);
				w[j] = pack_h2(p.x, p.y);
			}
			sum[0] = add2(sum[0], sum[1]);
			l += sum[0].x + sum[0].y;
			// (P's place is free: S of this tile came after O += P V of tile i - 2)
			const bool folds = FOLD && i > 0 && i % kFold == 0;
			if (i > 0 && (raise || fd.shrinks || folds)) {
				wait(&bar_o[group][(i - 1) & 1], (i - 1) / 2);
				fence_after();
				if (folds) {
					fold(i == kFold, f, fd.shrinks ? fd.shrink : nullptr, fd.unit);
				} else {
					if (fd.shrinks)   // V's factors of this tile
						rescale(1.0f, fd.shrink);
					if (raise)
						rescale(f, nullptr);
				}
			}
			if (fd.bads)
#pragma unroll
				for (int b = 0; b < NB; b++)
					poison |= seen & fd.bad[b] ? 1u << b : 0u;
#pragma unroll
			for (int c = 0; c < 4; c++)
				*reinterpret_cast<uint4 *>(sm + WL::kOffP + (2 * group + (i & 1)) * WL::kP + slice_at(tid, c)) =
					make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
			give(&p_ready[group][i & 1]);
		};
#pragma unroll 1
		for (int i = 0; i < ntile; i++) {
			// ---- scores
			float2 s[kAttnTile / 2];
			wait(&bar_s[group][i & 1], i / 2);
			fence_after();
			{
				const uint32_t at = tq + (i & 1) * WL::kTmemS;
				uint32_t r[32], q[32];
				tmem_two(at, at + 16, r);
				tmem_two(at + kAttnTile, at + kAttnTile + 16, q);
#pragma unroll
				for (int j = 0; j < kAttnTile / 2; j++)
					s[j] = add2(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])),
						    make_float2(__uint_as_float(q[2 * j]), __uint_as_float(q[2 * j + 1])));
			}
			fence_before();
			__syncwarp();
			if (lane == 0)
				mbar_arrive(&s_free[group][i & 1]);
			wait(&v_ready[i & 1], i / 2);   // what was found in the tile
			const int k0 = key0(i), have = found_s[i & 1].have;
			if (have == 3 && k0 >= all_lo && k0 + kAttnTile <= all_hi) {
				tile(std::true_type{}, s, i, 0xffffffffu);
			} else {
				const uint32_t large = have & 4 ? found_s[i & 1].large : 0;
				if (large)
#pragma unroll
					for (int j = 0; j < kAttnTile / 2; j++) {
						s[j].x *= large >> (2 * j) & 1 ? 16.0f : 1.0f;
						s[j].y *= large >> (2 * j + 1) & 1 ? 16.0f : 1.0f;
					}
				const int from = min(max(see_lo - k0, 0), 32), to = min(max(see_hi - k0, 0), 32);
				const uint32_t range = to > from ? 0xffffffffu >> (32 - (to - from)) << from : 0u;
				tile(std::false_type{}, s, i,
				     range & ((have & 1 ? 0xffffu : 0u) | (have & 2 ? 0xffff0000u : 0u)));
			}
		}
		// ---- out of tensor memory: a thread has its row
		if (ntile > 0)
			wait(&bar_o[group][(ntile - 1) & 1], (ntile - 1) / 2);
		fence_after();
		const bool folded = FOLD && ntile > kFold;
		float f = 0.0f;
		if (folded && row_used) {
			f = ex2(bias - pp[HL]);
			l = fmaf(pp[HL + 1], f, l);
		}
		const RowOut<T> out(a, it, row, bias, l);
#pragma unroll 1
		for (int b = 0; b < NB; b++) {
			uint32_t r[32];
			if (ntile > 0) {
				tmem_two(tq + WL::kTmemO + 32 * b, tq + WL::kTmemO + 32 * b + 16, r);
			} else {
#pragma unroll
				for (int k = 0; k < 32; k++)
					r[k] = 0;
			}
			const float iv = poison >> b & 1 ? __int_as_float(0x7fffffff) : v_unit[b];
			if (!row_used)
				continue;
#pragma unroll
			for (int e = 0; e < 32; e += 8) {
				float v[8];
#pragma unroll
				for (int k = 0; k < 8; k++)
					v[k] = __uint_as_float(r[e + k]) * iv;
				float4 *d = reinterpret_cast<float4 *>(pp + 32 * b + e);
				if (folded) {
					const float4 x = d[0], y = d[1];
					const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
					for (int k = 0; k < 8; k++)
						v[k] = fmaf(w[k], f, v[k]);
				}
				if (it.runs > 1) {
					d[0] = make_float4(v[0], v[1], v[2], v[3]);
					d[1] = make_float4(v[4], v[5], v[6], v[7]);
				} else {
					out.eight(32 * b + e, v);
				}
			}
		}
		if (row_used) {
			if (it.runs > 1)
				*reinterpret_cast<float2 *>(pp + HL) = make_float2(bias, l);
			else
				out.lse();
		}
	}
	fence_before();
	__syncthreads();
	if (warp == 0) {
		fence_after();
		asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(WL::kTmem));
	}
}

template <typename T, int HL>
cudaError_t launch_wide_as(const AttnArgs &a, const Plan &p, cudaStream_t st)
{
	constexpr int smem = WideLayout<HL>::kSmem;
	auto kernel = p.folds ? kv_wide_kernel<T, HL, true> : kv_wide_kernel<T, HL, false>;
	if (cudaError_t e = ensure_smem(kernel, smem))
		return e;
	kernel<<<(unsigned)p.items, kWideThreads, smem, st>>>(a);
	if (cudaError_t e = cudaGetLastError())
		return e;
	return launch_merge<T, HL, kWideRows>(a, p, st);
}

}  // namespace

namespace kva {

cudaError_t launch_wide(const AttnArgs &a, const Plan &p, int type, int HL, cudaStream_t st)
{
	if (type == MOE_F16)
		return HL == 64 ? launch_wide_as<__half, 64>(a, p, st) : launch_wide_as<__half, 128>(a, p, st);
	return HL == 64 ? launch_wide_as<__nv_bfloat16, 64>(a, p, st)
			: launch_wide_as<__nv_bfloat16, 128>(a, p, st);
}

}  // namespace kva
}  // namespace moe
