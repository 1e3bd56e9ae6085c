// What the losses on the scores of a vocabulary (nnf_vocab_loss.cu) share: rows of fp32, bf16 or fp16 that start and end anywhere,
// the running maximum and sum of a softmax, and their exchange across a thread-block cluster.
#pragma once

#include "nnf_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nnf
{
	// The elements of 16 bytes, as floats and back. Rounding to 16 bits happens once, to nearest, when a gradient is stored.
	template <class T> struct piece;

	template <> struct piece<float>
	{
		static constexpr int N = 4;
		static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[N])
		{
			f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
		}
		static __device__ __forceinline__ uint4 pack(const float (&f)[N])
		{
			return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
		}
		static __device__ __forceinline__ float value(const float * p) { return *p; }
		static __device__ __forceinline__ void store(float * p, float v) { *p = v; }
		static constexpr uint32_t kNothing = 0xff800000u;   // -infinity, in every element of the word
		template <int K> static __device__ __forceinline__ float maximum(const uint4 (&v)[K])
		{
			float m = -INFINITY;
			#pragma unroll
			for (int j = 0; j < K; ++j)
				m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[j].x), __uint_as_float(v[j].y)), fmaxf(__uint_as_float(v[j].z), __uint_as_float(v[j].w))));
			return m;
		}
	};

	template <> struct piece<__nv_bfloat16>
	{
		static constexpr int N = 8;
		static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[N])
		{
			const uint32_t w[4] = {v.x, v.y, v.z, v.w};
			#pragma unroll
			for (int i = 0; i < 4; ++i)
			{
				f[2 * i] = __uint_as_float(w[i] << 16);
				f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
			}
		}
		static __device__ __forceinline__ uint4 pack(const float (&f)[N])
		{
			uint32_t w[4];
			#pragma unroll
			for (int i = 0; i < 4; ++i)
			{
				const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			}
			return make_uint4(w[0], w[1], w[2], w[3]);
		}
		static __device__ __forceinline__ float value(const __nv_bfloat16 * p) { return __bfloat162float(*p); }
		static __device__ __forceinline__ void store(__nv_bfloat16 * p, float v) { *p = __float2bfloat16_rn(v); }
		static constexpr uint32_t kNothing = 0xff80ff80u;
		// two elements at a time; NaN is passed over, as fmaxf does
		template <int K> static __device__ __forceinline__ float maximum(const uint4 (&v)[K])
		{
			auto two = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162 *>(&w); };
			__nv_bfloat162 m = __hmax2(__hmax2(two(v[0].x), two(v[0].y)), __hmax2(two(v[0].z), two(v[0].w)));
			#pragma unroll
			for (int j = 1; j < K; ++j)
				m = __hmax2(m, __hmax2(__hmax2(two(v[j].x), two(v[j].y)), __hmax2(two(v[j].z), two(v[j].w))));
			return fmaxf(__bfloat162float(m.x), __bfloat162float(m.y));
		}
	};

	template <> struct piece<__half>
	{
		static constexpr int N = 8;
		static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[N])
		{
			const uint32_t w[4] = {v.x, v.y, v.z, v.w};
			#pragma unroll
			for (int i = 0; i < 4; ++i)
			{
				const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
				f[2 * i] = t.x;
				f[2 * i + 1] = t.y;
			}
		}
		static __device__ __forceinline__ uint4 pack(const float (&f)[N])
		{
			uint32_t w[4];
			#pragma unroll
			for (int i = 0; i < 4; ++i)
			{
				const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
				w[i] = *reinterpret_cast<const uint32_t *>(&h);
			}
			return make_uint4(w[0], w[1], w[2], w[3]);
		}
		static __device__ __forceinline__ float value(const __half * p) { return __half2float(*p); }
		static __device__ __forceinline__ void store(__half * p, float v) { *p = __float2half_rn(v); }
		static constexpr uint32_t kNothing = 0xfc00fc00u;
		// two elements at a time; NaN is passed over, as fmaxf does
		template <int K> static __device__ __forceinline__ float maximum(const uint4 (&v)[K])
		{
			auto two = [](uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); };
			__half2 m = __hmax2(__hmax2(two(v[0].x), two(v[0].y)), __hmax2(two(v[0].z), two(v[0].w)));
			#pragma unroll
			for (int j = 1; j < K; ++j)
				m = __hmax2(m, __hmax2(__hmax2(two(v[j].x), two(v[j].y)), __hmax2(two(v[j].z), two(v[j].w))));
			return fmaxf(__half2float(m.x), __half2float(m.y));
		}
	};

	// The 16-byte frame of a row of `cols` elements that starts anywhere: every aligned piece that holds one of its elements. Only the
	// first and the last piece can be partial; their elements are read and written one by one, the neighbouring rows' stay untouched.
	template <class T>
	struct row_frame
	{
		static constexpr int N = piece<T>::N;
		T * at;            // the row's first element
		int shift;         // elements of the first piece in front of it
		int pieces;
		int cols;

		__device__ __forceinline__ row_frame(T * row, int cols) : at(row), cols(cols)
		{
			shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
			pieces = (shift + cols + N - 1) / N;
		}
		__device__ __forceinline__ bool whole(int i) const { return (i > 0 || shift == 0) && (i + 1) * N - shift <= cols; }
		__device__ __forceinline__ uint4 * address(int i) const { return reinterpret_cast<uint4 *>(at - shift) + i; }
		__device__ __forceinline__ bool has(int i, int k) const { const int e = i * N - shift + k; return e >= 0 && e < cols; }
	};

	// maximum and sum of exp2((x - maximum) * k) of some elements; nothing: (-infinity, 0)
	struct softmax_part
	{
		float m, s;
	};

	__device__ __forceinline__ float exp2_of(float x)
	{
		float e;
		asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
		return e;
	}

	// two fp32 operations in one instruction, each rounded as by itself
	__device__ __forceinline__ unsigned long long pair_of(float a, float b)
	{
		unsigned long long r;
		asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
		return r;
	}
	__device__ __forceinline__ void pair_apart(unsigned long long p, float& a, float& b)
	{
		asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
	}
	__device__ __forceinline__ unsigned long long pair_fma(unsigned long long a, unsigned long long b, unsigned long long c)
	{
		unsigned long long r;
		asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
		return r;
	}
	__device__ __forceinline__ unsigned long long pair_add(unsigned long long a, unsigned long long b)
	{
		unsigned long long r;
		asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
		return r;
	}

	// What a part's exponentials are multiplied with when the maximum becomes m. A part without a maximum (-infinity) keeps its sum: 0, or
	// NaN where an element was NaN, which no maximum shows.
	__device__ __forceinline__ float rescale(float part_m, float m, float k)
	{
		return part_m == m ? 1.0F : exp2_of((part_m - m) * k);
	}

	// the same with what k leaves out (rest > 0)
	__device__ __forceinline__ float rescale(float part_m, float m, float k, float rest)
	{
		const float gap = part_m - m;
		return part_m == m ? 1.0F : exp2_of(__fmaf_rn(gap, k, gap * rest));
	}

	// From here on an argument leaves the fused form: x*k - mk is off by what mk was rounded by, 0.03 at this size.
	constexpr float kFused = 1.0e6F;

	// Sum of exp2(x*k - mk) over some pieces, with one fused operation for the argument. REST: k is rounded down and `rest`, above 0, is what
	// that leaves out, which is then added to each argument: left out of every term it is a bias of the sum (1e-7 of it for scores a
	// few tau apart), small against the rounding of one log probability, but not in a sequence's sum of them.
	template <class T, int K, bool REST>
	__device__ __forceinline__ float sum_of_fused(const uint4 (&v)[K], float mk, float k, float rest)
	{
		constexpr int N = piece<T>::N;
		const unsigned long long kk = pair_of(k, k), mm = pair_of(-mk, -mk), rr = pair_of(rest, rest);
		unsigned long long both = pair_of(0.0F, 0.0F);
		#pragma unroll
		for (int j = 0; j < K; ++j)
		{
			float f[N];
			piece<T>::unpack(v[j], f);
			#pragma unroll
			for (int e = 0; e < N; e += 2)
			{
				float a, b;
				const unsigned long long x = pair_of(f[e], f[e + 1]);
				pair_apart(REST ? pair_fma(x, rr, pair_fma(x, kk, mm)) : pair_fma(x, kk, mm), a, b);
				both = pair_add(both, pair_of(exp2_of(a), exp2_of(b)));
			}
		}
		float s[2];
		pair_apart(both, s[0], s[1]);
		return s[0] + s[1];
	}

	// Sum of exp2((x - base)*k), the difference first: for scores beyond kFused (a row of nothing but the type's lowest value).
	template <class T, int K>
	__device__ __forceinline__ float sum_of_apart(const uint4 (&v)[K], float base, float k)
	{
		constexpr int N = piece<T>::N;
		float s[2] = {0.0F, 0.0F};
		#pragma unroll
		for (int j = 0; j < K; ++j)
		{
			float f[N];
			piece<T>::unpack(v[j], f);
			#pragma unroll
			for (int e = 0; e < N; ++e)
				s[e & 1] += exp2_of((f[e] - base) * k);
		}
		return s[0] + s[1];
	}

	// Sum of exp2((x - m)*k) over some pieces whose maximum is at most m; m = -infinity: of 0 (or NaN). rest: as above, 0 without.
	template <class T, int K, bool REST = false>
	__device__ __forceinline__ float sum_of_exp(const uint4 (&v)[K], float m, float k, float rest = 0.0F)
	{
		const float base = m == -INFINITY ? 0.0F : m;
		const float mk = base * k;
		if (fabsf(mk) < kFused)
		{
			// mk is m*k rounded: the fused sum is against 2^mk, and what mk is off by (2^-24 of it: 1e-6 for scores of 10) is put right on the sum
			const float off = __fmaf_rn(base, k, -mk);
			return sum_of_fused<T, K, REST>(v, mk, k, rest) * exp2_of(REST ? -__fmaf_rn(base, rest, off) : -off);
		}
		return sum_of_apart<T, K>(v, base, k);
	}

	// The gradient's c*exp2((x - m)*k) over a row. As in sum_of_exp the argument is one fused operation, and what m*k rounded is off by goes
	// into c; fp32 results take the product with c, 16-bit ones have it in the argument (log2 |c| - m*k, rounded, is off by 2^-24 of
	// at most 400: 1.7e-5 of the result, against the 2^-9 or 2^-12 of their own rounding) and their sign in the packed words.
	template <class T>
	struct row_gradient
	{
		float m, k, c, mk, offset;
		uint32_t sign;

		__device__ __forceinline__ row_gradient(float m, float k, float c) : m(m), k(k), c(c), mk(m * k)
		{
			const float put_right = c * exp2_of(-__fmaf_rn(m, k, -mk));
			offset = sizeof(T) == 4 ? put_right : __log2f(fabsf(put_right)) - mk;
			sign = c < 0.0F ? 0x80008000u : 0u;
		}
		__device__ __forceinline__ bool near() const { return fabsf(mk) < (sizeof(T) == 4 ? kFused : 256.0F); }

		template <bool NEAR> __device__ __forceinline__ uint4 whole(const uint4& v) const
		{
			constexpr int N = piece<T>::N;
			float f[N];
			piece<T>::unpack(v, f);
			const unsigned long long kk = pair_of(k, k), add = sizeof(T) == 4 ? pair_of(-mk, -mk) : pair_of(offset, offset);
			#pragma unroll
			for (int e = 0; e < N; e += 2)
			{
				if (NEAR)
				{
					float a, b;
					pair_apart(pair_fma(pair_of(f[e], f[e + 1]), kk, add), a, b);
					f[e] = sizeof(T) == 4 ? exp2_of(a) * offset : exp2_of(a);
					f[e + 1] = sizeof(T) == 4 ? exp2_of(b) * offset : exp2_of(b);
				}
				else
				{
					f[e] = exp2_of((f[e] - m) * k) * c;
					f[e + 1] = exp2_of((f[e + 1] - m) * k) * c;
				}
			}
			uint4 w = piece<T>::pack(f);
			if (NEAR && sizeof(T) == 2)
				w = make_uint4(w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign);
			return w;
		}
	};

	__device__ __forceinline__ softmax_part part_of(float x)
	{
		return {fmaxf(x, -INFINITY), x == -INFINITY ? 0.0F : x - x + 1.0F};   // (infinity and NaN: NaN)
	}

	// the elements of some pieces join a part
	template <class T, int K>
	__device__ __forceinline__ void add_part(softmax_part& part, const uint4 (&v)[K], float k)
	{
		const float m = fmaxf(part.m, piece<T>::template maximum<K>(v));
		part.s = part.s * rescale(part.m, m, k) + sum_of_exp<T, K>(v, m, k);
		part.m = m;
	}

	// The same over as many steps as a row has (512 where a warp takes a row of 1 MiB), no worse for their number: the sum carries what
	// its roundings lose (confident rows, 1 and a hundred thousand small terms: off by up to 44*2^-24 without), and its reference moves only
	// when the maximum is more than a factor of two above it, so that scores in ascending order do not multiply it with an approximate
	// power at every step (20*2^-24 short, in the mean, over 131072). The reference stays an element: a row that is nearly one
	// score has that score's own term exact.
	struct running_part
	{
		float m;         // the maximum
		float against;   // the reference, an element that is at most 1/k below the maximum; the sum is against it, or
		float mk;        // against 2^mk where that is below kFused (against*k, rounded; 0 where there is no reference)
		float s, lost;   // the sum, and what its roundings have added to it
	};

	__device__ __forceinline__ running_part running_none() { return {-INFINITY, -INFINITY, 0.0F, 0.0F, 0.0F}; }

	// exponent of what the sum is against, less m*k (both with what k leaves out)
	__device__ __forceinline__ float running_gap(const running_part& part, float m, float k, float rest)
	{
		if (fabsf(part.mk) < kFused)
			return -__fmaf_rn(m, rest, __fmaf_rn(m, k, -part.mk));
		const float gap = part.against - m;
		return __fmaf_rn(gap, k, gap * rest);
	}

	// the part's sum against m, which is at least its maximum; without a reference it is 0, or NaN
	__device__ __forceinline__ float running_sum(const running_part& part, float m, float k, float rest)
	{
		const float s = part.s - part.lost;
		return part.against == -INFINITY ? s : s * exp2_of(running_gap(part, m, k, rest));
	}

	__device__ __forceinline__ void running_raise(running_part& part, float k, float rest)
	{
		const float mk = part.m * k;
		if (part.against != -INFINITY)
		{
			float gap = running_gap(part, part.m, k, rest);
			if (fabsf(mk) < kFused)
				gap += __fmaf_rn(part.m, rest, __fmaf_rn(part.m, k, -mk));
			const float share = exp2_of(gap);
			part.s *= share;
			part.lost *= share;
		}
		part.against = part.m;
		part.mk = mk;
	}

	template <class T, int K>
	__device__ __forceinline__ void add_running(running_part& part, const uint4 (&v)[K], float k, float rest)
	{
		part.m = fmaxf(part.m, piece<T>::template maximum<K>(v));
		if ((part.m - part.against) * k > 1.0F)   // (both infinite: no)
			running_raise(part, k, rest);
		const float terms = fabsf(part.mk) < kFused ? sum_of_fused<T, K, true>(v, part.mk, k, rest) : sum_of_apart<T, K>(v, part.against, k);
		const float more = terms - part.lost, s = part.s + more;
		part.lost = (s - part.s) - more;
		part.s = s;
	}

	// what a single element (none: -infinity) adds to a sum against m, which is at least it
	__device__ __forceinline__ float edge_term(float x, float m, float k, float rest)
	{
		return x == -INFINITY ? 0.0F : (x - x + 1.0F) * rescale(x, m, k, rest);   // (infinity and NaN: NaN)
	}

	// ex2.approx.ftz is below 2^x by 0.83*2^-24 of it in the mean (measured over -20..0; 2.3*2^-24 at most; for x = 0, as in the maximum's own
	// term, it is exact). A term has two of them, its own and its part's: what a sum against its maximum is short of, for the reason given
	// at sum_of_fused.
	__device__ __forceinline__ float lifted(float s) { return s > 1.0F ? __fmaf_rn(s - 1.0F, 9.9e-8F, s) : s; }

	__device__ __forceinline__ float vocab_warp_max(float v)
	{
		float r;
		asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
		return r;
	}

	__device__ __forceinline__ float vocab_warp_sum(float v)
	{
		#pragma unroll
		for (int o = 16; o > 0; o >>= 1)
			v += __shfl_xor_sync(0xffffffffu, v, o);
		return v;
	}

	// ---- thread-block clusters -----------------------------------------------------------------------
	__device__ __forceinline__ uint32_t vocab_cluster_rank()
	{
		uint32_t r;
		asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
		return r;
	}

	__device__ __forceinline__ void vocab_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
	__device__ __forceinline__ void vocab_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

	// a store into the shared memory of another CTA of the cluster, at the address that `p` has in this one
	__device__ __forceinline__ void vocab_cluster_store(const softmax_part * p, uint32_t rank, softmax_part v)
	{
		uint32_t a;
		asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
		asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" :: "r"(a), "f"(v.m), "f"(v.s) : "memory");
	}

	// the same, counted by a barrier of that CTA
	__device__ __forceinline__ void vocab_cluster_send(const softmax_part * p, const uint64_t * bar, uint32_t rank, softmax_part v)
	{
		uint32_t a, b;
		asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
		asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(rank));
		asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
			:: "r"(a), "f"(v.m), "f"(v.s), "r"(b) : "memory");
	}
}
