// Losses on the scores of a vocabulary: log probabilities of given tokens (forward and backward), the clipped policy loss with a KL
// term, the loss of paired sequences, and distillation from a teacher's top logits. Logits are rows of fp32, bf16 or fp16, one for each
// token, and the targets are indices: what softmax + negative log likelihood (nnf_loss.cu) is for the classes of an image, with dense
// targets and stored probabilities, these are where a row has 1e3..1e5 scores.
//
//   M = max_j x_j,  S = sum_j exp((x_j - M)/tau),  p_j = exp((x_j - M)/tau)/S,  logp = (x_a - M)/tau - ln S
//   every gradient is  dx_j = (what the targets hold at j) - c*p_j,  c one number for the row: the direction in which the loss falls,
//   as the library's backward passes have it and its optimiser step adds it.
//
// HBM bounds them: an element is 2 or 4 bytes in (and as many out), and takes one or two exponentials. So a row is read once and stays
// on chip between its sum and its gradient, in one of three places:
//   short rows (up to 256 pieces of 16 bytes): a warp's registers, row after row (vocab_short_kernel)
//   longer ones: the shared memory of a CTA, or of a thread-block cluster whose CTAs exchange maxima and sums (vocab_held_kernel)
//   log probabilities alone need not be held (vocab_score_kernel, vocab_score_warp_kernel); their backward pass reads the row again
//   (vocab_bwd_kernel), as does the loss of paired sequences, whose gradient needs the sums over all rows of a pair.
// Rows of 16-bit scores are next to being bound by instructions too: per element an unpacking, a fused multiply-add, an exponential, a
// sum and half a maximum, and for the gradient the first three again and half a rounding; fp32 arithmetic goes in pairs (f32x2). Maximum,
// sum and everything behind them are fp32; a gradient is rounded once, when it is stored.
#include "nnf_vocab.cuh"

#include <math.h>

#include <type_traits>

namespace nnf
{
	namespace
	{
		constexpr int kVocabCluster = 8;         // most CTAs of a row (the portable cluster size)
		constexpr int64_t kMaxPieces = 65536;    // of a row: 1 MiB
		constexpr int kMaxKept = 1024;           // most logits that are kept of a teacher's row

		enum { kScore = 0, kPolicy = 1, kDistill = 2 };

		struct vocab_params
		{
			const void * x;
			void * dx;                 // gradient, or null
			int64_t ldx, lddx;
			int64_t rows;
			int cols;
			int add;                   // the gradient is added to what dx holds
			float tau, inv_tau, k;     // k = log2(e)/tau
			float k_down, k_rest;      // the same, rounded down, and what that leaves out
			float inv_rest;            // 1/tau less inv_tau
			int cluster;               // CTAs of a row
			// targets
			const void * tokens;
			int tokens_wide;           // 64-bit indices
			const float * mask;
			float scale;
			float * loss;
			float * logp;
			float * saved;             // [2][rows]: M, S
			// score: only the rows in [offsets[0], offsets[sequences]) are written, or null
			const void * offsets;
			int offsets_wide;
			int64_t sequences;
			// policy
			const float * old_logp, * advantages, * ref_logp;
			float * kl;
			float low, high, kl_coef;
			// distillation
			const void * ids, * teacher;
			int64_t ld_ids, ld_teacher;
			int ids_wide, teacher_type, kept;
		};

		__device__ __forceinline__ int64_t index_at(const void * p, int wide, int64_t i)
		{
			return wide ? __ldg(static_cast<const long long *>(p) + i) : (int64_t)__ldg(static_cast<const int *>(p) + i);
		}

		__device__ __forceinline__ float value_at(const void * p, int type, int64_t i)
		{
			if (type == NNF_BF16)
				return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
			if (type == NNF_F16)
				return __half2float(static_cast<const __half *>(p)[i]);
			return __ldg(static_cast<const float *>(p) + i);
		}

		__device__ __forceinline__ int64_t within(int64_t row, int64_t rows) { return row < 0 ? 0 : row > rows ? rows : row; }

		// the rows that the packed sequences cover
		__device__ __forceinline__ void covered_rows(const vocab_params& p, int64_t& begin, int64_t& end)
		{
			begin = index_at(p.offsets, p.offsets_wide, 0);
			end = index_at(p.offsets, p.offsets_wide, p.sequences);
			begin = within(begin, p.rows);
			end = within(end, p.rows);
		}

		// a piece of a gradient that is nothing: at once where it is whole and starts at its 16 bytes, else element by element
		template <class T>
		__device__ __forceinline__ void clear_piece(const row_frame<T>& x, T * dx, bool aligned, int i)
		{
			const int first = i * piece<T>::N - x.shift;
			if (aligned && x.whole(i))
				__stcs(reinterpret_cast<uint4 *>(dx + first), make_uint4(0, 0, 0, 0));
			else
			{
				#pragma unroll 1
				for (int e = 0; e < piece<T>::N; ++e)
					if (x.has(i, e))
						piece<T>::store(dx + first + e, 0.0F);
			}
		}

		// (xa - M)/tau - ln S, rounded once: what a reciprocal that is rounded to 32 bits loses has one sign in every row (1.4*2^-24 in the mean
		// at a temperature of 1.7), which a sequence's sum gathers
		__device__ __forceinline__ float logp_of(const vocab_params& p, float xa, float m, float s)
		{
			const float gap = xa - m, ln = -logf(s), h = gap * p.inv_tau;
			const float lost = __fmaf_rn(gap, p.inv_rest, __fmaf_rn(gap, p.inv_tau, -h));   // of h
			const float sum = __fadd_rn(h, ln), back = sum - h;
			const float less = (h - (sum - back)) + (ln - back);                           // of the sum
			return h == -INFINITY ? h + ln : sum + (lost + less);
		}

		// what a policy's row comes to
		struct policy_row
		{
			float logp, kl, loss;
			float c, at_token;   // the gradient: c*exp2((x_j - M)*k), and at the token
		};

		__device__ __forceinline__ policy_row policy_of(const vocab_params& p, float xa, const softmax_part& total, float weight, float old_logp, float a, float ref_logp, bool on)
		{
			policy_row r = {0.0F, 0.0F, 0.0F, 0.0F, 0.0F};
			if (!on)
				return r;
			r.logp = (xa - total.m) * p.inv_tau - logf(total.s);
			const float ratio = expf(r.logp - old_logp);
			const float free = ratio * a, held = fminf(fmaxf(ratio, p.low), p.high) * a;
			// min() that keeps a NaN
			float loss = -(free <= held ? free : held < free ? held : free + held);
			float g = held < free ? 0.0F : free;
			if (p.ref_logp)
			{
				const float gap = ref_logp - r.logp, grown = expm1f(gap);
				r.kl = grown - gap;
				if (p.kl_coef != 0.0F)   // (0 * infinity is no number)
				{
					loss += p.kl_coef * r.kl;
					g += p.kl_coef * grown;
				}
			}
			g = weight != 0.0F ? g * weight * p.inv_tau : 0.0F;
			r.loss = weight != 0.0F ? loss * weight : 0.0F;
			r.c = -g / total.s;
			r.at_token = -g * expm1f(r.logp);   // g * (1 - p)
			return r;
		}

		// of a row's partial pieces an element a lane: the first piece's in the lower half of the warp, the last one's in the upper
		template <class T>
		__device__ __forceinline__ float edge_of(const row_frame<T>& x, int lane)
		{
			const int at = lane < 16 ? 0 : x.pieces - 1, e = lane & 15;
			const bool there = e < piece<T>::N && !x.whole(at) && (lane < 16 || x.pieces > 1) && x.has(at, e);
			return there ? piece<T>::value(x.at + at * piece<T>::N - x.shift + e) : -INFINITY;
		}

		struct distill_shared
		{
			int * id;         // -1: the entry does not count
			float * q;        // the teacher's logit
			float * x;        // the student's score
			float * old;      // what the gradient held (it is added to)
			uint32_t * seen;  // a bit for each of this CTA's columns
		};

		constexpr unsigned long long kWaitNs = 5000000000ull;

		__device__ __forceinline__ uint32_t shared_address(const void * p) { return (uint32_t)__cvta_generic_to_shared(p); }

		__device__ __forceinline__ void mbar_init(uint64_t * b, int count)
		{
			asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(shared_address(b)), "r"(count) : "memory");
		}
		__device__ __forceinline__ void mbar_arrive_expect(uint64_t * b, uint32_t bytes)
		{
			asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(shared_address(b)), "r"(bytes) : "memory");
		}
		__device__ __forceinline__ bool mbar_try(uint64_t * b, uint32_t phase)
		{
			uint32_t done;
			asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
				: "=r"(done) : "r"(shared_address(b)), "r"(phase), "r"(1000000u) : "memory");   // suspended for up to a millisecond
			return done != 0;
		}
		// Bounded: when the limit runs out the error word is raised and the caller carries on, without waiting any more for what this flag
		// stands for; every loop has its number of turns from the start, so that all threads still meet at the same barriers and leave. The
		// row's sum is then made NaN, which its results show, and what has not come is waited for once more, since it would be written
		// into the shared memory of a CTA that has left. Nothing covers what takes longer than both waits.
		__device__ __forceinline__ void mbar_wait(uint64_t * b, uint32_t phase, bool& gave_up, int * error)
		{
			if (gave_up || mbar_try(b, phase))
				return;
			unsigned long long start, now;
			asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
			while (!mbar_try(b, phase))
			{
				asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
				if (now - start > kWaitNs)
				{
					gave_up = true;
					if (error)
						*error = 4;
					return;
				}
			}
		}

		__device__ __forceinline__ void copy_bulk(void * to, const void * from, uint32_t bytes, uint64_t * bar)
		{
			asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
				:: "r"(shared_address(to)), "l"(from), "r"(bytes), "r"(shared_address(bar)) : "memory");
		}

		// ---- long rows: held in shared memory ----------------------------------------------------------------------------
		// A CTA per row (a cluster, where the row is split), several of them on an SM. Bulk copies bring the row in, chunk by chunk; each
		// chunk's exponentials are summed against the thread's running maximum as it arrives; the gradient is computed from shared memory.
		// What an SM has in flight are the rows of its other CTAs: the bytes that a row takes up decide how many those are, so a
		// quarter of a long row is held in registers (four CTAs of 64 KB instead of three: 8192x32000 bf16 198 -> 178 us when it came; not for
		// shorter rows, of which shared memory has room for more CTAs than registers do: 16384x12000 146 -> 154).
		//
		// One B200, policy loss, us (bytes at the copy rate of 6.55 TB/s): bf16 8192x32000 172 (160), 16384x12000 136 (120), 2048x131072 195 (164);
		// fp32 8192x16000 157 (160), 1024x131072 181 (164). bf16 3000x32000 under the profiler: issue slots 60 %, exponentials (XU) 70 %, DRAM 54 %
		// (writes still in L2 at the end not counted), 4 CTAs an SM. Twice the scores for the same bytes are why bf16 lies behind fp32; of a row
		// that is split each CTA waits for the slowest of its cluster. Distillation of 64 kept logits takes 208 us for 8192x32000: the teacher's row,
		// the loss and the kept columns lengthen a CTA's 10 us by 2.
		//
		// Measured and not kept: a persistent CTA an SM with the exponentials in registers and a ring of rows filled ahead of it (one row's
		// chain of latencies at a time: 1.5 times the time), the gradient's exponentials by polynomial (issue slots are as short as the
		// XU), warps of their own for the teacher's row (better for 16 kept logits, worse from 64 on), that row in front of
		// the sums (its latency then keeps them from following the chunks: 4096x32000 with 64 kept logits 107 us against 104).
		constexpr int kHeldThreads = 256, kHeldChunk = 4, kHeldChunks = 40;   // kHeldChunk: pieces of a chunk that a thread takes

		// kAnyRow: gradients that are added, or whose rows start elsewhere in their 16 bytes than the logits'; the loss alone.
		// kAlignedRow: whole pieces are stored at once. kRegisterRow: and the second chunk is held in registers.
		enum { kAnyRow = 0, kAlignedRow = 1, kRegisterRow = 2 };

		struct held_params
		{
			vocab_params v;
			int slots;                 // pieces of a CTA in shared memory
			int * error;
		};

		struct held_result             // what the row comes to, found by the first warp
		{
			float m, s, c, at_token, share;
			float t_max, t_sum;        // of the teacher's logits
			int on;
		};

		template <class T, int OP, int ROW>
		__global__ void __launch_bounds__(kHeldThreads, 4) vocab_held_kernel(const held_params hp)
		{
			constexpr int N = piece<T>::N;
			extern __shared__ __align__(128) unsigned char s_held[];
			__shared__ softmax_part s_part[kVocabCluster * (kHeldThreads / 32)];
			__shared__ uint64_t s_bar[kHeldChunks];
			__shared__ uint64_t s_exchanged;
			__shared__ held_result s_result;
			__shared__ softmax_part s_teacher[kHeldThreads / 32];
			__shared__ float s_number[2][32];
			const vocab_params& p = hp.v;
			const uint32_t split = (uint32_t)p.cluster;
			const uint32_t rank = split > 1 ? vocab_cluster_rank() : 0;
			const int tid = (int)threadIdx.x, step = (int)blockDim.x, lane = tid & 31, warp = tid >> 5, warps = step >> 5;
			const int64_t row = blockIdx.x / split;
			if (split > 1)
			{
				if (tid == 0)
				{
					mbar_init(&s_exchanged, 1);
					asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
					mbar_arrive_expect(&s_exchanged, split * (uint32_t)warps * (uint32_t)sizeof(softmax_part));
				}
				vocab_cluster_arrive();   // waited for before the first store into another CTA
			}
			const row_frame<T> x(const_cast<T *>(static_cast<const T *>(p.x)) + row * p.ldx, p.cols);
			T * const dx = p.dx ? static_cast<T *>(p.dx) + row * p.lddx : nullptr;
			const int per = split > 1 ? (x.pieces + (int)split - 1) / (int)split : x.pieces;
			const int from = (int)rank * per, count = max(min(per, x.pieces - from), 0);   // this CTA's pieces
			const int chunk = step * kHeldChunk;
			const int away = ROW == kRegisterRow && count > 2 * chunk ? chunk : 0;         // of those, in registers: [chunk, 2*chunk)
			const int kept = count - away, chunks = (kept + chunk - 1) / chunk;            // in shared memory, in their order
			const int lo = count > 0 && !x.whole(from) ? 1 : 0, hi = count > lo && !x.whole(from + count - 1) ? count - 1 : count;   // whole pieces
			uint4 * const held = reinterpret_cast<uint4 *>(s_held);
			T * const held_at = reinterpret_cast<T *>(s_held);
			if (tid == 0)
			{
				for (int i = 0; i < chunks; ++i)
					mbar_init(s_bar + i, 1);
				asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
			}
			pdl_begin();

			// a thread's first entry of the teacher's row: on its way before anything is waited for
			int64_t id_first = -1;
			float t_first = -INFINITY;
			if (OP == kDistill && tid < p.kept)
			{
				id_first = index_at(p.ids, p.ids_wide, row * p.ld_ids + tid);
				t_first = value_at(p.teacher, p.teacher_type, row * p.ld_teacher + tid);
			}
			const float w = p.mask ? p.mask[row] : 1.0F;
			int token = 0;
			bool on = w != 0.0F;
			if (OP == kPolicy)
			{
				const int64_t t = index_at(p.tokens, p.tokens_wide, row);
				on = on && t >= 0 && t < p.cols;
				token = on ? (int)t : 0;
			}
			const float weight = p.scale * w;
			// this CTA's elements: [begin, begin + elements) of the row
			const int begin = max(from * N - x.shift, 0), elements = max(min((from + count) * N - x.shift, p.cols) - begin, 0);
			auto nothing = [&]()
			{
				if (ROW == kAnyRow)
				{
					if (dx && !p.add)
						for (int e = tid; e < elements; e += step)
							piece<T>::store(dx + begin + e, 0.0F);
					return;
				}
				uint4 * const out = reinterpret_cast<uint4 *>(dx - x.shift) + from;
				for (int i = tid + lo; i < hi; i += step)
					__stcs(out + i, make_uint4(0, 0, 0, 0));
				if (tid < 2 * N)
				{
					const int i = tid < N ? 0 : count - 1;
					if ((tid < N ? lo > 0 : hi < count) && x.has(from + i, tid % N))
						piece<T>::store(dx + (from + i) * N - x.shift + tid % N, 0.0F);
				}
			};
			if (!on)   // the same in every CTA of the cluster
			{
				if (rank == 0 && tid == 0)
				{
					p.loss[row] = 0.0F;
					if (OP == kPolicy)
					{
						p.logp[row] = 0.0F;
						if (p.kl)
							p.kl[row] = 0.0F;
					}
				}
				nothing();
				if (split > 1)
					vocab_cluster_wait();
				return;
			}
			if (tid == 0)
			{
				for (int i = 0; i < chunks; ++i)
				{
					const int skip = i > 0 ? away : 0;
					const int a = max(i * chunk, lo), b = min((i + 1) * chunk, hi - away);
					const uint32_t bytes = b > a ? (uint32_t)(b - a) * 16 : 0;
					mbar_arrive_expect(s_bar + i, bytes);
					if (bytes)
						copy_bulk(held + a, x.address(from + a + skip), bytes, s_bar + i);
				}
			}
			uint4 own[kHeldChunk];
			if (ROW == kRegisterRow)
			{
				#pragma unroll
				for (int j = 0; j < kHeldChunk; ++j)
					own[j] = away ? __ldcs(x.address(from + chunk + j * step + tid))
						: make_uint4(piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing);
			}
			// the partial pieces, an element a thread
			if (tid < 2 * N)
			{
				const int i = tid < N ? 0 : count - 1, e = tid % N;
				if (tid < N ? lo > 0 : hi < count)
					held_at[(tid < N ? 0 : kept - 1) * N + e] = x.has(from + i, e) ? x.at[(from + i) * N - x.shift + e] : T(-INFINITY);
			}
			// what a policy's row comes to besides its sums, in the first warp: the token's score, and a number a lane (a load for all of them)
			float xa = 0.0F, number = 0.0F;
			if (OP == kPolicy && warp == 0)
			{
				xa = piece<T>::value(x.at + token);
				number = (lane == 0 || (lane != 1 && !p.ref_logp) ? p.old_logp : lane == 1 ? p.advantages : p.ref_logp)[row];
			}
			distill_shared d = {};
			// the score at a column of this CTA, in shared memory; elsewhere it was fetched with the teacher's row
			auto place = [&](int id) { const int e = id + x.shift - from * N; return away && e >= 2 * chunk * N ? e - chunk * N : e; };
			auto present = [&](int id)
			{
				const int e = id + x.shift - from * N;
				return e >= 0 && e < count * N && !(away && e >= chunk * N && e < 2 * chunk * N);
			};
			if (OP == kDistill)
			{
				d.id = reinterpret_cast<int *>(held + hp.slots);
				d.q = reinterpret_cast<float *>(d.id + p.kept);
				d.x = d.q + p.kept;
				d.seen = reinterpret_cast<uint32_t *>(d.x + p.kept);
				d.old = reinterpret_cast<float *>(d.seen + (per * N + 31) / 32);   // kAnyRow
			}
			__syncthreads();   // the barriers and the partial pieces are there

			// ---- maximum and sum, against the thread's running maximum ----
			softmax_part part = {-INFINITY, 0.0F};
			bool gave_up = false;
			for (int i = 0; i < chunks; ++i)
			{
				mbar_wait(s_bar + i, 0, gave_up, hp.error);
				uint4 v[kHeldChunk];
				#pragma unroll
				for (int j = 0; j < kHeldChunk; ++j)
				{
					const int at = i * chunk + j * step + tid;
					v[j] = at < kept ? held[at] : make_uint4(piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing);
				}
				add_part<T, kHeldChunk>(part, v, p.k);
			}
			if (ROW == kRegisterRow && away)
				add_part<T, kHeldChunk>(part, own, p.k);
			if (gave_up)
			{
				bool again = false;
				for (int i = 0; i < chunks; ++i)
					mbar_wait(s_bar + i, 0, again, hp.error);
				part.s = NAN;
			}
			if (OP == kDistill && warp * 32 < p.kept)
			{
				// the teacher's entries of this warp; its logits' maximum and sum are joined as the student's are
				softmax_part teacher = {-INFINITY, 0.0F};
				for (int e = tid; e < p.kept; e += step)
				{
					const int64_t id = e == tid ? id_first : index_at(p.ids, p.ids_wide, row * p.ld_ids + e);
					const bool in = id >= 0 && id < p.cols, mine = in && id >= begin && id < begin + elements;
					const float l = !in ? -INFINITY : e == tid ? t_first : value_at(p.teacher, p.teacher_type, row * p.ld_teacher + e);
					d.id[e] = in ? (int)id : -1;
					d.q[e] = l;
					if (mine)
						d.seen[((int)id - begin) >> 5] = 0;
					if (ROW == kAnyRow && p.add && mine)
						d.old[e] = piece<T>::value(dx + id);
					if (in && (mine || rank == 0) && !present((int)id))   // (the first CTA finds the loss)
						d.x[e] = piece<T>::value(x.at + id);
					const float m = fmaxf(teacher.m, l);
					teacher.s = teacher.s * rescale(teacher.m, m, p.k) + part_of(l).s * rescale(l, m, p.k);
					teacher.m = m;
				}
				const float m = vocab_warp_max(teacher.m);
				teacher.s = vocab_warp_sum(teacher.s * rescale(teacher.m, m, p.k));
				if (lane == 0)
					s_teacher[warp] = {m, teacher.s};
			}
			{
				const float m = vocab_warp_max(part.m);
				part.s = vocab_warp_sum(part.s * rescale(part.m, m, p.k));
				part.m = m;
			}
			// The first warp of every CTA gets every warp's part (and the CTA leaves only then). Once the other CTAs have this
			// one's parts, they may write over what it still reads: the token's score, where the gradient takes the scores' place, and the
			// row's numbers, where an output takes an input's (logp that of old_logp). They must be here by then.
			bool late = false;   // another CTA's parts
			if (split > 1)
			{
				vocab_cluster_wait();
				if (OP == kPolicy && warp == 0)
				{
					asm volatile("st.shared.f32 [%0], %1;" :: "r"(shared_address(s_number[0] + lane)), "f"(xa) : "memory");   // (waits for it)
					asm volatile("st.shared.f32 [%0], %1;" :: "r"(shared_address(s_number[1] + lane)), "f"(number) : "memory");
					__syncwarp();
				}
				if (lane < (int)split)
					vocab_cluster_send(s_part + rank * warps + warp, &s_exchanged, lane, part);
				if (warp == 0)
				{
					mbar_wait(&s_exchanged, 0, late, hp.error);
					if (late)
					{
						bool again = false;
						mbar_wait(&s_exchanged, 0, again, hp.error);
					}
					__syncwarp();
				}
				if (OP == kDistill)
					__syncthreads();   // the teacher's parts
			}
			else
			{
				if (lane == 0)
					s_part[warp] = part;
				__syncthreads();
			}
			if (warp == 0)
			{
				softmax_part total = {-INFINITY, late ? NAN : 0.0F};
				for (int i = lane; i < (int)split * warps; i += 32)
					total.m = fmaxf(total.m, s_part[i].m);
				total.m = vocab_warp_max(total.m);
				for (int i = lane; i < (int)split * warps; i += 32)
					total.s += s_part[i].s * rescale(s_part[i].m, total.m, p.k);
				total.s = vocab_warp_sum(total.s);
				on = total.s != 0.0F;   // NaN counts; a row of nothing but -infinity does not
				held_result r = {total.m, total.s, 0.0F, 0.0F, 0.0F, 0.0F, 0.0F, on};
				if (OP == kPolicy)
				{
					auto of_lane = [&](int l) { return __shfl_sync(0xffffffffu, number, l); };
					const float old_logp = of_lane(0), advantage = of_lane(1), ref_logp = of_lane(2);
					const policy_row l = policy_of(p, xa, total, weight, old_logp, advantage, ref_logp, on);
					r.c = l.c;
					r.at_token = l.at_token;
					r.on = l.c != 0.0F || l.at_token != 0.0F;
					if (rank == 0 && lane == 0)
					{
						p.loss[row] = l.loss;
						p.logp[row] = l.logp;
						if (p.kl)
							p.kl[row] = l.kl;
					}
				}
				else
				{
					const softmax_part mine = lane < min(warps, (p.kept + 31) / 32) ? s_teacher[lane] : softmax_part{-INFINITY, 0.0F};
					const float top = vocab_warp_max(mine.m);
					r.t_max = top == -INFINITY ? 0.0F : top;
					r.t_sum = vocab_warp_sum(mine.s * rescale(mine.m, top, p.k));
					r.on = on && r.t_sum != 0.0F && weight != 0.0F;
					r.c = r.on ? -weight * p.tau / total.s : 0.0F;
					r.share = r.on ? weight * p.tau / r.t_sum : 0.0F;
				}
				if (lane == 0)
					s_result = r;
			}
			__syncthreads();
			const held_result r = s_result;
			if (OP == kDistill && rank == 0 && warp == warps - 1)
			{
				// the loss, while the other warps are at the gradient
				float sum = 0.0F;
				if (r.on)
				{
					const float ln = logf(r.s), t_ln = logf(r.t_sum);
					for (int e = lane; e < p.kept; e += 32)
					{
						const float q = exp2_of((d.q[e] - r.t_max) * p.k);
						if (q != 0.0F)
						{
							const float xe = present(d.id[e]) ? piece<T>::value(held_at + place(d.id[e])) : d.x[e];
							sum += q * (((d.q[e] - r.t_max) * p.inv_tau - t_ln) - ((xe - r.m) * p.inv_tau - ln));
						}
					}
					sum = vocab_warp_sum(sum) * (weight * p.tau * p.tau / r.t_sum);
				}
				if (lane == 0)
					p.loss[row] = sum;
			}
			if (!dx)
				return;
			if (!r.on)
			{
				nothing();
				return;
			}
			const row_gradient<T> gradient(r.m, p.k, r.c);
			if (ROW == kAnyRow)
			{
				for (int e = tid; e < elements; e += step)
				{
					const int id = begin + e;
					float g = exp2_of((piece<T>::value(held_at + id + x.shift - from * N) - r.m) * p.k) * r.c;
					if (OP == kPolicy && id == token)
						g = r.at_token;
					piece<T>::store(dx + id, p.add ? piece<T>::value(dx + id) + g : g);
				}
			}
			else
			{
				uint4 * const out = reinterpret_cast<uint4 *>(dx - x.shift) + from;
				auto pieces = [&](auto near)
				{
					for (int i = 0; i < chunks; ++i)
					{
						const int at = i * chunk + tid, skip = i > 0 ? away : 0;
						#pragma unroll
						for (int j = 0; j < kHeldChunk; ++j)
							if (at + j * step >= lo && at + j * step < hi - away)
								__stcs(out + (at + skip + j * step), gradient.template whole<near.value>(held[at + j * step]));
					}
					if (ROW == kRegisterRow && away)
					{
						#pragma unroll
						for (int j = 0; j < kHeldChunk; ++j)
							__stcs(out + (chunk + j * step + tid), gradient.template whole<near.value>(own[j]));
					}
				};
				if (gradient.near())
					pieces(std::true_type());
				else
					pieces(std::false_type());
				if (tid < 2 * N)
				{
					const int i = tid < N ? 0 : count - 1, e = tid % N, id = (from + i) * N - x.shift + e;
					if ((tid < N ? lo > 0 : hi < count) && x.has(from + i, e) && !(OP == kPolicy && id == token))
						piece<T>::store(dx + id, exp2_of((piece<T>::value(held_at + (tid < N ? 0 : kept - 1) * N + e) - r.m) * p.k) * r.c);
				}
				if (OP == kPolicy && token >= begin && token < begin + elements)
				{
					// behind the token's piece, by the thread that has just written it
					const int i = (token + x.shift) / N - from;
					if (tid == i % step)
						piece<T>::store(dx + token, r.at_token);
				}
			}
			if (OP == kDistill)
			{
				// The columns that the teacher kept: c*(q - p), written over -c*p. An index that is there twice holds the sum of both; the
				// first of its entries writes it. `seen` shows whether there is one at all.
				bool twice = false;
				for (int e = tid; e < p.kept; e += step)
				{
					const int at = d.id[e] - begin;
					if (d.id[e] >= 0 && at >= 0 && at < elements)
					{
						const uint32_t bit = 1u << (at & 31);
						twice = twice || (atomicOr(d.seen + (at >> 5), bit) & bit);
					}
				}
				twice = __syncthreads_or(twice);   // also: the pieces above are written
				for (int e = tid; e < p.kept; e += step)
				{
					const int id = d.id[e];
					if (id < begin || id >= begin + elements)
						continue;
					float q = exp2_of((d.q[e] - r.t_max) * p.k);
					bool leads = true;
					if (twice)
					{
						q = 0.0F;
						for (int o = 0; o < p.kept; ++o)
							if (d.id[o] == id)
							{
								leads = leads && o >= e;
								q += exp2_of((d.q[o] - r.t_max) * p.k);
							}
					}
					if (leads)
					{
						const float xe = present(id) ? piece<T>::value(held_at + place(id)) : d.x[e];
						const float g = exp2_of((xe - r.m) * p.k) * r.c + r.share * q;
						piece<T>::store(dx + id, ROW == kAnyRow && p.add ? d.old[e] + g : g);
					}
				}
			}
		}

		// ---- log probabilities alone: nothing to be held -----------------------------------------------------------------
		// A CTA per row (a cluster, where there are few rows); a thread's next pieces are on their way while it sums the current ones.
		// One B200, bf16, us (bytes at the copy rate): 8192x32000 87 (80), 2048x131072 86 (82), 64x32000 4.5 (a launch). XU 72 %, issue slots 68 %, DRAM 69 %:
		// what is left is the chain at either end of a row (token, first piece; sums, result).
		constexpr int kScoreThreads = 256, kScorePieces = 4;

		template <class T>
		__global__ void __launch_bounds__(kScoreThreads, 4) vocab_score_kernel(const vocab_params p)
		{
			constexpr int N = piece<T>::N;
			__shared__ softmax_part s_part[kVocabCluster * (kScoreThreads / 32)];
			const uint32_t split = (uint32_t)p.cluster;
			const uint32_t rank = split > 1 ? vocab_cluster_rank() : 0;
			const int tid = (int)threadIdx.x, step = (int)blockDim.x, lane = tid & 31, warp = tid >> 5, warps = step >> 5;
			const int64_t row = blockIdx.x / split;
			if (split > 1)
				vocab_cluster_arrive();
			const row_frame<T> x(const_cast<T *>(static_cast<const T *>(p.x)) + row * p.ldx, p.cols);
			const int per = split > 1 ? (x.pieces + (int)split - 1) / (int)split : x.pieces;
			const int from = (int)rank * per, to = min(from + per, x.pieces);
			const int lo = from + (from < to && !x.whole(from)), hi = to - (to > lo && !x.whole(to - 1));   // whole pieces
			pdl_begin();
			bool inside = true;
			if (p.offsets)
			{
				int64_t begin, end;
				covered_rows(p, begin, end);
				inside = row >= begin && row < end;
			}
			const int64_t token = inside ? index_at(p.tokens, p.tokens_wide, row) : -1;
			if (token < 0 || token >= p.cols)   // the same in every CTA of the cluster
			{
				if (inside && rank == 0 && tid == 0)
				{
					p.logp[row] = 0.0F;
					if (p.saved)
						p.saved[row] = p.saved[p.rows + row] = 0.0F;
				}
				if (split > 1)
					vocab_cluster_wait();
				return;
			}
			const uint4 nothing = make_uint4(piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing);
			const uint4 * const in = x.address(0);
			uint4 v[kScorePieces], next[kScorePieces];
			#pragma unroll
			for (int j = 0; j < kScorePieces; ++j)
			{
				const int at = lo + j * step + tid;
				v[j] = at < hi ? __ldg(in + at) : nothing;
			}
			float xa = 0.0F;
			running_part own = running_none();
			float at_edge = -INFINITY;
			if (rank == 0 && tid == 0)
				xa = piece<T>::value(x.at + token);
			if (tid < 2 * N && from < to)
			{
				// the partial pieces, an element a thread
				const int at = tid < N ? from : to - 1, e = tid % N;
				if ((tid < N ? lo > from : hi < to) && x.has(at, e))
					at_edge = piece<T>::value(x.at + at * N - x.shift + e);
			}
			for (int i = lo; i < hi; i += kScorePieces * step)
			{
				#pragma unroll
				for (int j = 0; j < kScorePieces; ++j)
				{
					const int at = i + (kScorePieces + j) * step + tid;
					next[j] = at < hi ? __ldg(in + at) : nothing;
				}
				add_running<T, kScorePieces>(own, v, p.k_down, p.k_rest);
				#pragma unroll
				for (int j = 0; j < kScorePieces; ++j)
					v[j] = next[j];
			}
			softmax_part part;
			part.m = vocab_warp_max(fmaxf(own.m, at_edge));
			part.s = vocab_warp_sum(running_sum(own, part.m, p.k_down, p.k_rest) + edge_term(at_edge, part.m, p.k_down, p.k_rest));
			if (split > 1)
			{
				// the first CTA gets every warp's part
				vocab_cluster_wait();
				if (lane == 0)
					vocab_cluster_store(s_part + rank * warps + warp, 0, part);
				vocab_cluster_arrive();
				vocab_cluster_wait();
			}
			else
			{
				if (lane == 0)
					s_part[warp] = part;
				__syncthreads();
			}
			if (rank == 0 && warp == 0)
			{
				softmax_part total = {-INFINITY, 0.0F};
				for (int i = lane; i < (int)split * warps; i += 32)
					total.m = fmaxf(total.m, s_part[i].m);
				total.m = vocab_warp_max(total.m);
				for (int i = lane; i < (int)split * warps; i += 32)
					total.s += s_part[i].s * rescale(s_part[i].m, total.m, p.k_down, p.k_rest);
				total.s = lifted(vocab_warp_sum(total.s));
				if (lane == 0)
				{
					const bool on = total.s != 0.0F;   // NaN counts; a row of nothing but -infinity does not
					p.logp[row] = on ? logp_of(p, xa, total.m, total.s) : 0.0F;
					if (p.saved)
					{
						p.saved[row] = on ? total.m : 0.0F;
						p.saved[p.rows + row] = on ? total.s : 0.0F;
					}
				}
			}
		}

		// The same for many rows: a warp takes row after row, and a row's first pieces are asked for while the one before it ends. Lane l
		// keeps the token of the l-th of the warp's next 32 rows, so that rows that count for nothing cost no time. bf16, us (bytes at the
		// copy rate; a CTA per row): 16384x12000 70 (60; 75), 32768x4096 52 (41; 85), 65536x1000 36 (20; 47; issue slots 66 %, XU 47 %, DRAM 41 %:
		// what a row costs besides its scores, and its latencies).
		constexpr int kRowWarps = 8;   // of a CTA

		template <class T>
		__global__ void __launch_bounds__(kRowWarps * 32, 4) vocab_score_warp_kernel(const vocab_params p)
		{
			constexpr int K = kScorePieces;
			const int lane = (int)threadIdx.x & 31;
			const int warps = (int)gridDim.x * kRowWarps;   // of the launch: no more than are resident
			const uint4 nothing = make_uint4(piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing);
			pdl_begin();
			int64_t begin = 0, end = p.rows;
			if (p.offsets)
				covered_rows(p, begin, end);
			int64_t base = begin + (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5) - 32 * (int64_t)warps;   // the first of 32 rows, `warps` apart
			uint32_t ahead = 0;          // those of them that count and are still to come
			int token = 0;

			// the row that comes next: its first pieces, its token's score, and of its partial pieces an element a lane
			row_frame<T> x(nullptr, 0);
			int64_t row = -1;
			int lo = 0, hi = 0;
			float xa = 0.0F, edge = -INFINITY;
			uint4 next[K];
			auto fetch = [&](int i, auto first)
			{
				#pragma unroll
				for (int j = 0; j < K; ++j)
				{
					const int at = i + j * 32 + lane;
					next[j] = (!first.value || at >= lo) && at < hi ? __ldg(x.address(at)) : nothing;
				}
			};
			auto advance = [&]()
			{
				row = -1;
				while (ahead == 0)
				{
					base += 32 * warps;
					if (base >= end)
						return;
					const int64_t r = base + (int64_t)lane * warps;
					const int64_t wide = r < end ? index_at(p.tokens, p.tokens_wide, r) : -1;
					const bool on = wide >= 0 && wide < p.cols;
					token = (int)wide;
					if (!on && r < end)
					{
						p.logp[r] = 0.0F;
						if (p.saved)
							p.saved[r] = p.saved[p.rows + r] = 0.0F;
					}
					ahead = __ballot_sync(0xffffffffu, on);
				}
				const int l = __ffs((int)ahead) - 1;
				ahead &= ahead - 1;
				row = base + (int64_t)l * warps;
				x = row_frame<T>(const_cast<T *>(static_cast<const T *>(p.x)) + row * p.ldx, p.cols);
				lo = x.whole(0) ? 0 : 1;
				hi = x.whole(x.pieces - 1) ? x.pieces : x.pieces - 1;
				fetch(0, std::true_type());
				xa = piece<T>::value(x.at + __shfl_sync(0xffffffffu, token, l));
				if (lo > 0 || hi < x.pieces)
					edge = edge_of(x, lane);
			};
			for (advance(); row >= 0;)
			{
				running_part part = running_none();
				const bool steps = hi > K * 32, ragged = lo > 0 || hi < x.pieces;
				uint4 v[K];
				for (int i = K * 32; i < hi; i += K * 32)
				{
					#pragma unroll
					for (int j = 0; j < K; ++j)
						v[j] = next[j];
					fetch(i, std::false_type());
					add_running<T, K>(part, v, p.k_down, p.k_rest);
				}
				#pragma unroll
				for (int j = 0; j < K; ++j)
					v[j] = next[j];
				const int64_t done = row;
				const float its_xa = xa, at_edge = ragged ? edge : -INFINITY;
				advance();
				// the last step, and the only one of a short row: against the row's maximum at once
				const float m = vocab_warp_max(fmaxf(fmaxf(part.m, at_edge), piece<T>::template maximum<K>(v)));
				float sum = sum_of_exp<T, K, true>(v, m, p.k_down, p.k_rest);
				if (ragged)
					sum += edge_term(at_edge, m, p.k_down, p.k_rest);
				if (steps)
					sum += running_sum(part, m, p.k_down, p.k_rest);
				const float s = lifted(vocab_warp_sum(sum));
				if (lane == 0)
				{
					const bool on = s != 0.0F;   // NaN counts; a row of nothing but -infinity does not
					p.logp[done] = on ? logp_of(p, its_xa, m, s) : 0.0F;
					if (p.saved)
					{
						p.saved[done] = on ? m : 0.0F;
						p.saved[p.rows + done] = on ? s : 0.0F;
					}
				}
			}
		}

		// ---- short rows, with their gradient: a warp has a row in registers ---------------------------------------------------
		// As above a warp takes row after row, and asks for the next one before it works on the one it has. NP: pieces of a lane. Policy loss,
		// us (bytes at the copy rate; the row in a CTA's shared memory): bf16 65536x1000 68 (40; 150), 32768x2000 61 (40; 80), fp32 65536x1000
		// 96 (80; 140). Bound by latencies: at 65536x1000 issue slots are busy 63 %, XU 56 %, DRAM 36 %; in 80 registers five warps a scheduler are
		// resident, each of which has an instruction ready every 8 cycles, so that a third of the cycles have none. A row takes 700.
		template <class T, int OP, int NP, bool ANY>
		__global__ void __launch_bounds__(kRowWarps * 32, NP > 4 ? 2 : 3) vocab_short_kernel(const vocab_params p)
		{
			constexpr int N = piece<T>::N;
			extern __shared__ __align__(16) unsigned char s_short[];
			const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
			const int64_t warps = (int64_t)gridDim.x * kRowWarps;
			const uint4 nothing = make_uint4(piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing, piece<T>::kNothing);
			distill_shared d = {};
			if (OP == kDistill)
			{
				constexpr int words = NP * 32 * N / 32 + 1;
				d.id = reinterpret_cast<int *>(s_short) + (size_t)warp * (4 * p.kept + words);
				d.q = reinterpret_cast<float *>(d.id + p.kept);
				d.x = d.q + p.kept;
				d.old = d.x + p.kept;
				d.seen = reinterpret_cast<uint32_t *>(d.old + p.kept);
				for (int i = lane; i < words; i += 32)
					d.seen[i] = 0;
			}
			pdl_begin();
			int64_t base = (int64_t)blockIdx.x * kRowWarps + warp - 32 * warps;   // the first of 32 rows, `warps` apart
			uint32_t ahead = 0;          // those of them that count and are still to come
			int token = 0;               // of the lane's row, as the following
			float weight = 0.0F, old_logp = 0.0F, advantage = 0.0F, ref_logp = 0.0F;

			row_frame<T> x(nullptr, 0);  // the row that comes next
			int64_t row = -1;
			float xa = 0.0F, edge = -INFINITY, its_weight = 0.0F, its_old = 0.0F, its_advantage = 0.0F, its_ref = 0.0F;
			int its_token = 0;
			uint4 next[NP];
			auto empty_row = [&](int64_t r)   // its gradient is nothing
			{
				const row_frame<T> e(const_cast<T *>(static_cast<const T *>(p.x)) + r * p.ldx, p.cols);
				T * const dx = static_cast<T *>(p.dx) + r * p.lddx;
				for (int i = lane; i < e.pieces; i += 32)
					clear_piece<T>(e, dx, !ANY, i);
			};
			auto advance = [&]()
			{
				row = -1;
				while (ahead == 0)
				{
					base += 32 * warps;
					if (base >= p.rows)
						return;
					const int64_t r = base + lane * warps;
					const bool there = r < p.rows;
					const float w = !there ? 0.0F : p.mask ? p.mask[r] : 1.0F;
					bool on = w != 0.0F;
					weight = p.scale * w;
					if (OP == kPolicy && there)
					{
						const int64_t wide = index_at(p.tokens, p.tokens_wide, r);
						on = on && wide >= 0 && wide < p.cols;
						token = (int)wide;
						old_logp = p.old_logp[r];
						advantage = p.advantages[r];
						ref_logp = p.ref_logp ? p.ref_logp[r] : 0.0F;
					}
					if (!on && there)
					{
						p.loss[r] = 0.0F;
						if (OP == kPolicy)
						{
							p.logp[r] = 0.0F;
							if (p.kl)
								p.kl[r] = 0.0F;
						}
					}
					ahead = __ballot_sync(0xffffffffu, on);
					if (p.dx && !p.add)
						for (uint32_t off = __ballot_sync(0xffffffffu, !on && there); off; off &= off - 1)
							empty_row(base + (__ffs((int)off) - 1) * warps);
				}
				const int l = __ffs((int)ahead) - 1;
				ahead &= ahead - 1;
				row = base + l * warps;
				x = row_frame<T>(const_cast<T *>(static_cast<const T *>(p.x)) + row * p.ldx, p.cols);
				const int lo = x.whole(0) ? 0 : 1, hi = x.whole(x.pieces - 1) ? x.pieces : x.pieces - 1;
				#pragma unroll
				for (int j = 0; j < NP; ++j)
				{
					const int at = j * 32 + lane;
					next[j] = at >= lo && at < hi ? __ldcs(x.address(at)) : nothing;
				}
				its_weight = __shfl_sync(0xffffffffu, weight, l);
				if (OP == kPolicy)
				{
					its_token = __shfl_sync(0xffffffffu, token, l);
					xa = piece<T>::value(x.at + its_token);
					its_old = __shfl_sync(0xffffffffu, old_logp, l);
					its_advantage = __shfl_sync(0xffffffffu, advantage, l);
					its_ref = __shfl_sync(0xffffffffu, ref_logp, l);
				}
				edge = edge_of(x, lane);
			};
			for (advance(); row >= 0;)
			{
				const row_frame<T> y = x;
				const int64_t done = row;
				const float w = its_weight, at_edge = edge, score = xa, o = its_old, a = its_advantage, f = its_ref;
				const int tok = its_token;
				uint4 v[NP];
				#pragma unroll
				for (int j = 0; j < NP; ++j)
					v[j] = next[j];
				T * const dx = p.dx ? static_cast<T *>(p.dx) + done * p.lddx : nullptr;
				float t_max = 0.0F, t_sum = 0.0F;
				if (OP == kDistill)
				{
					float m = -INFINITY;
					for (int e = lane; e < p.kept; e += 32)
					{
						const int64_t id = index_at(p.ids, p.ids_wide, done * p.ld_ids + e);
						const bool in = id >= 0 && id < p.cols;
						const float t = in ? value_at(p.teacher, p.teacher_type, done * p.ld_teacher + e) : -INFINITY;
						d.id[e] = in ? (int)id : -1;
						d.q[e] = t;
						d.x[e] = in ? piece<T>::value(y.at + id) : 0.0F;
						if (ANY && p.add && in)
							d.old[e] = piece<T>::value(dx + id);
						m = fmaxf(m, t);
					}
					m = vocab_warp_max(m);
					t_max = m == -INFINITY ? 0.0F : m;
					for (int e = lane; e < p.kept; e += 32)
						t_sum += exp2_of((d.q[e] - t_max) * p.k);
					t_sum = vocab_warp_sum(t_sum);
				}
				advance();

				softmax_part total;
				total.m = vocab_warp_max(fmaxf(piece<T>::template maximum<NP>(v), at_edge));
				total.s = vocab_warp_sum(sum_of_exp<T, NP>(v, total.m, p.k) + (at_edge == -INFINITY ? 0.0F : exp2_of((at_edge - total.m) * p.k)));
				bool on = total.s != 0.0F;   // NaN counts; a row of nothing but -infinity does not
				float c = 0.0F, at_token = 0.0F;
				if (OP == kPolicy)
				{
					const policy_row l = policy_of(p, score, total, w, o, a, f, on);
					c = l.c;
					at_token = l.at_token;
					if (lane == 0)
					{
						p.loss[done] = l.loss;
						p.logp[done] = l.logp;
						if (p.kl)
							p.kl[done] = l.kl;
					}
					on = c != 0.0F || at_token != 0.0F;
				}
				else
				{
					on = on && t_sum != 0.0F && w != 0.0F;
					c = on ? -w * p.tau / total.s : 0.0F;
					float sum = 0.0F;
					if (on)
					{
						const float ln = logf(total.s), t_ln = logf(t_sum);
						for (int e = lane; e < p.kept; e += 32)
						{
							const float q = exp2_of((d.q[e] - t_max) * p.k);
							if (q != 0.0F)
								sum += q * (((d.q[e] - t_max) * p.inv_tau - t_ln) - ((d.x[e] - total.m) * p.inv_tau - ln));
						}
						sum = vocab_warp_sum(sum) * (w * p.tau * p.tau / t_sum);
					}
					if (lane == 0)
						p.loss[done] = sum;
				}
				if (!dx)
				{
					__syncwarp();
					continue;
				}
				if (!on)
				{
					if (!p.add)
						empty_row(done);
					__syncwarp();
					continue;
				}
				const int lo = y.whole(0) ? 0 : 1, hi = y.whole(y.pieces - 1) ? y.pieces : y.pieces - 1;
				const row_gradient<T> gradient(total.m, p.k, c);
				if (ANY)
				{
					#pragma unroll
					for (int j = 0; j < NP; ++j)
					{
						const int at = j * 32 + lane;
						if (at >= lo && at < hi)
						{
							float g[N];
							piece<T>::unpack(v[j], g);
							#pragma unroll
							for (int e = 0; e < N; ++e)
							{
								const int col = at * N - y.shift + e;
								const float t = OP == kPolicy && col == tok ? at_token : exp2_of((g[e] - total.m) * p.k) * c;
								piece<T>::store(dx + col, p.add ? piece<T>::value(dx + col) + t : t);
							}
						}
					}
				}
				else
				{
					uint4 * const out = reinterpret_cast<uint4 *>(dx - y.shift);
					if (gradient.near())
					{
						#pragma unroll
						for (int j = 0; j < NP; ++j)
							if (j * 32 + lane >= lo && j * 32 + lane < hi)
								__stcs(out + j * 32 + lane, gradient.template whole<true>(v[j]));
					}
					else
					{
						#pragma unroll
						for (int j = 0; j < NP; ++j)
							if (j * 32 + lane >= lo && j * 32 + lane < hi)
								__stcs(out + j * 32 + lane, gradient.template whole<false>(v[j]));
					}
				}
				if (lo > 0 || hi < y.pieces)
				{
					const int at = lane < 16 ? 0 : y.pieces - 1, e = lane & 15, col = at * N - y.shift + e;
					if (e < N && !y.whole(at) && (lane < 16 || y.pieces > 1) && y.has(at, e))
					{
						const float t = ANY && OP == kPolicy && col == tok ? at_token : exp2_of((at_edge - total.m) * p.k) * c;
						piece<T>::store(dx + col, p.add ? piece<T>::value(dx + col) + t : t);
					}
				}
				__syncwarp();   // what lies under the target's columns is written
				if (!ANY && OP == kPolicy && lane == 0)
					piece<T>::store(dx + tok, at_token);
				if (OP == kDistill)
				{
					// the columns that the teacher kept, as in the kernel for long rows
					bool twice = false;
					for (int e = lane; e < p.kept; e += 32)
						if (d.id[e] >= 0)
						{
							const uint32_t bit = 1u << (d.id[e] & 31);
							twice = twice || (atomicOr(d.seen + (d.id[e] >> 5), bit) & bit);
						}
					twice = __any_sync(0xffffffffu, twice);
					__syncwarp();
					const float share = w * p.tau / t_sum;
					for (int e = lane; e < p.kept; e += 32)
					{
						const int id = d.id[e];
						if (id < 0)
							continue;
						d.seen[id >> 5] = 0;
						float q = exp2_of((d.q[e] - t_max) * p.k);
						bool leads = true;
						if (twice)
						{
							q = 0.0F;
							for (int i = 0; i < p.kept; ++i)
								if (d.id[i] == id)
								{
									leads = leads && i >= e;
									q += exp2_of((d.q[i] - t_max) * p.k);
								}
						}
						if (leads)
						{
							const float g = exp2_of((d.x[e] - total.m) * p.k) * c + share * q;
							piece<T>::store(dx + id, ANY && p.add ? d.old[e] + g : g);
						}
					}
					__syncwarp();
				}
			}
		}

		// ---- backward of the log probabilities: one pass, nothing to be found first ------------------------
		struct vocab_bwd_params
		{
			const void * x;
			void * dx;
			int64_t ldx, lddx;
			int64_t rows;
			int cols;
			int add;
			float inv_tau, k;
			const void * tokens;
			int tokens_wide;
			const float * dlogp, * saved;
			const void * offsets;      // as for the score, or null
			int offsets_wide;
			int64_t sequences;
			int slices;                // CTAs of a row
			int64_t last;              // the last row of this launch, which comes first
		};

		constexpr int kBwdThreads = 256, kBwdPieces = 4;

		// ALIGNED: whole pieces are stored at once (the gradient is not added, and its rows start where the logits' do in their 16 bytes).
		// The last row comes first: the end of the logits is what the forward pass before has left in L2 (8192x32000 bf16, forward and backward,
		// 265 -> 252 us when it came). HBM bounds it: 8192x32000 with 30 % of the rows out moves 891 MB in 132 us, 6.8 TB/s with what comes from L2.
		template <class T, bool ALIGNED>
		__global__ void __launch_bounds__(kBwdThreads) vocab_bwd_kernel(const vocab_bwd_params p)
		{
			constexpr int N = piece<T>::N;
			pdl_begin();
			const int64_t row = p.last - blockIdx.x / p.slices;
			if (p.offsets)
			{
				vocab_params q = {};
				q.offsets = p.offsets; q.offsets_wide = p.offsets_wide; q.sequences = p.sequences; q.rows = p.rows;
				int64_t begin, end;
				covered_rows(q, begin, end);
				if (row < begin || row >= end)
					return;
			}
			const row_frame<T> x(const_cast<T *>(static_cast<const T *>(p.x)) + row * p.ldx, p.cols);
			T * const dx = static_cast<T *>(p.dx) + row * p.lddx;
			const int64_t token = index_at(p.tokens, p.tokens_wide, row);
			const float g = __ldg(p.dlogp + row) * p.inv_tau, m = __ldg(p.saved + row), s = __ldg(p.saved + p.rows + row);
			const bool on = token >= 0 && token < p.cols && s != 0.0F && g != 0.0F;
			const int step = (int)blockDim.x, from = (int)(blockIdx.x % p.slices) * step * kBwdPieces + (int)threadIdx.x;
			const int lo = x.whole(0) ? 0 : 1, hi = x.pieces > lo && !x.whole(x.pieces - 1) ? x.pieces - 1 : x.pieces;   // whole pieces
			if (!on)
			{
				if (!p.add)
					for (int j = 0, i = from; j < kBwdPieces && i < x.pieces; ++j, i += step)
						clear_piece<T>(x, dx, ALIGNED, i);
				return;
			}
			const row_gradient<T> gradient(m, p.k, -g / s);
			auto at = [&](int col)   // one element
			{
				const float score = piece<T>::value(x.at + col);
				const float t = col == (int)token ? -g * expm1f((score - m) * p.inv_tau - logf(s)) : exp2_of((score - m) * p.k) * gradient.c;
				return p.add ? piece<T>::value(dx + col) + t : t;
			};
			if (ALIGNED && gradient.near())
			{
				uint4 v[kBwdPieces];
				#pragma unroll
				for (int j = 0; j < kBwdPieces; ++j)
					if (from + j * step >= lo && from + j * step < hi)
						v[j] = __ldcs(x.address(from + j * step));
				float at_token = 0.0F;
				const int token_piece = (int)(token + x.shift) / N;
				const bool mine = token_piece >= from && token_piece < from + kBwdPieces * step && (token_piece - from) % step == 0;
				if (mine)
					at_token = at((int)token);   // before it is written over, should the gradient take the scores' place
				uint4 * const out = reinterpret_cast<uint4 *>(dx - x.shift);
				#pragma unroll
				for (int j = 0; j < kBwdPieces; ++j)
					if (from + j * step >= lo && from + j * step < hi)
						__stcs(out + from + j * step, gradient.template whole<true>(v[j]));
				if (mine && token_piece >= lo && token_piece < hi)
					piece<T>::store(dx + token, at_token);
				for (int i = from, j = 0; j < kBwdPieces && i < x.pieces; ++j, i += step)
					if (i < lo || i >= hi)
						for (int e = 0; e < N; ++e)
							if (x.has(i, e))
								piece<T>::store(dx + i * N - x.shift + e, at(i * N - x.shift + e));
			}
			else
			{
				// element by element, a CTA's elements side by side
				const int first = (from - (int)threadIdx.x) * N - x.shift, last = min(first + kBwdPieces * step * N, p.cols);
				for (int col = max(first, 0) + (int)threadIdx.x; col < last; col += step)
					piece<T>::store(dx + col, at(col));
			}
		}

		// ---- pairs of sequences: sums of their log probabilities, the loss, and its gradient for every token ----
		struct pair_params
		{
			const float * logp, * saved, * ref_logp;
			const void * offsets;
			int offsets_wide;
			int64_t rows;
			float * loss, * rewards, * dlogp;
			float beta, smoothing, scale;
			int kind, average;
		};

		constexpr int kPairThreads = 256;

		__device__ __forceinline__ float softplus(float x)
		{
			return fmaxf(x, 0.0F) + log1pf(expf(-fabsf(x)));
		}

		// A CTA per pair; sums in double, in an order that depends on nothing but the lengths. 16 pairs of 8192 rows: 7 us, a chain of latencies
		// (offsets, log probabilities, sums, loss, gradients) between two launches of 69 and 132 us. One launch for all three, in which resident CTAs
		// drew the rows' items and a pair's gradients followed its sums while the scores were in L2, was measured at 217 us against 212 and dropped.
		__global__ void __launch_bounds__(kPairThreads) vocab_pair_kernel(const pair_params p)
		{
			__shared__ double s_sum[2][kPairThreads / 32];
			__shared__ long long s_count[2][kPairThreads / 32];
			pdl_begin();
			const int64_t pair = blockIdx.x;
			int64_t begin[2], end[2];
			double sum[2];
			long long count[2];
			// in front of the barrier: the rewards may take its place
			const float ref[2] = {p.ref_logp[2 * pair], p.ref_logp[2 * pair + 1]};
			#pragma unroll
			for (int side = 0; side < 2; ++side)
			{
				begin[side] = within(index_at(p.offsets, p.offsets_wide, 2 * pair + side), p.rows);
				end[side] = within(index_at(p.offsets, p.offsets_wide, 2 * pair + side + 1), p.rows);
				double t = 0.0;
				long long n = 0;
				#pragma unroll 4
				for (int64_t r = begin[side] + threadIdx.x; r < end[side]; r += kPairThreads)
				{
					const float s = p.saved[p.rows + r], l = p.logp[r];
					t += s != 0.0F ? (double)l : 0.0;
					n += s != 0.0F;
				}
				#pragma unroll
				for (int o = 16; o > 0; o >>= 1)
				{
					t += __shfl_xor_sync(0xffffffffu, t, o);
					n += __shfl_xor_sync(0xffffffffu, n, o);
				}
				if ((threadIdx.x & 31) == 0)
				{
					s_sum[side][threadIdx.x >> 5] = t;
					s_count[side][threadIdx.x >> 5] = n;
				}
			}
			__syncthreads();
			float share[2], ratio[2];
			double gap[2];
			#pragma unroll
			for (int side = 0; side < 2; ++side)
			{
				sum[side] = 0.0;
				count[side] = 0;
				for (int i = 0; i < kPairThreads / 32; ++i)
				{
					sum[side] += s_sum[side][i];
					count[side] += s_count[side][i];
				}
				const double by = p.average && count[side] > 0 ? 1.0 / (double)count[side] : 1.0;
				share[side] = (float)by;
				gap[side] = sum[side] * by - (double)ref[side];
				ratio[side] = (float)gap[side];
			}
			const double h = gap[0] - gap[1];
			float loss, dh;
			if (p.kind == NNF_PREFERENCE_SQUARED)
			{
				const float off = (float)(h - 0.5 / (double)p.beta);
				loss = off * off;
				dh = 2.0F * off;
			}
			else
			{
				const float m = (float)(h * (double)p.beta);
				loss = (p.smoothing < 1.0F ? (1.0F - p.smoothing) * softplus(-m) : 0.0F) + (p.smoothing > 0.0F ? p.smoothing * softplus(m) : 0.0F);
				dh = p.beta * (p.smoothing / (1.0F + expf(-m)) - (1.0F - p.smoothing) / (1.0F + expf(m)));
			}
			if (threadIdx.x == 0)
			{
				p.loss[pair] = loss * p.scale;
				p.rewards[2 * pair] = p.beta * ratio[0];
				p.rewards[2 * pair + 1] = p.beta * ratio[1];
			}
			#pragma unroll
			for (int side = 0; side < 2; ++side)
			{
				const float g = (side == 0 ? -dh : dh) * p.scale * share[side];
				#pragma unroll 4
				for (int64_t r = begin[side] + threadIdx.x; r < end[side]; r += kPairThreads)
					p.dlogp[r] = p.saved[p.rows + r] != 0.0F ? g : 0.0F;
			}
		}

		// ---- launches -------------------------------------------------------------------------------------
		int element_size(int type)
		{
			switch (type)
			{
			case NNF_F32: case NNF_I32: return 4;
			case NNF_BF16: case NNF_F16: return 2;
			case NNF_I64: return 8;
			default: return 0;
			}
		}

		bool is_index(int type) { return type == NNF_I32 || type == NNF_I64; }
		bool is_float(int type) { return type == NNF_F32 || type == NNF_BF16 || type == NNF_F16; }
		bool misaligned(const void * p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

		// 0: fine
		int check_rows(const char * who, const char * what, const nnf_matrix * m, bool (*of)(int))
		{
			if (!m)
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: null pointer", who, what);
			if (!of(m->type))
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: type %d", who, what, (int)m->type);
			if (m->rows < 0 || m->cols <= 0 || (m->rows > 1 && m->stride < m->cols))
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: bad extents rows=%lld cols=%lld stride=%lld", who, what, (long long)m->rows, (long long)m->cols, (long long)m->stride);
			if (m->rows > 0 && !m->data)
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: null pointer", who, what);
			if (misaligned(m->data, element_size(m->type)))
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: misaligned buffer", who, what);
			return NNF_OK;
		}

		int check_indices(const char * who, const char * what, const nnf_indices * t)
		{
			if (!t || !t->data)
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: null pointer", who, what);
			if (!is_index(t->type))
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: type %d", who, what, (int)t->type);
			if (misaligned(t->data, element_size(t->type)))
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: %s: misaligned buffer", who, what);
			return NNF_OK;
		}

		// whether an element of one matrix lies in the other (of the same type and shape); what lies between rows belongs to neither
		bool overlap(const nnf_matrix& a, const nnf_matrix& b)
		{
			const int64_t size = element_size(a.type), width = a.cols * size;
			const int64_t step_a = (a.rows > 1 ? a.stride : a.cols) * size, step_b = (b.rows > 1 ? b.stride : b.cols) * size;
			const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(b.data) - reinterpret_cast<uintptr_t>(a.data));
			if (apart >= (a.rows - 1) * step_a + width || -apart >= (b.rows - 1) * step_b + width)
				return false;
			if (step_a == step_b)
			{
				const int64_t within = (apart % step_a + step_a) % step_a;   // of b's rows, in the steps of a
				return within < width || within > step_a - width;
			}
			for (int64_t r = 0; r < a.rows; ++r)   // rows side by side in one buffer, with strides of their own
			{
				const int64_t reach = r * step_a - apart;   // from b's first row to this one
				int64_t next = reach < width ? 0 : (reach - width) / step_b + 1;   // the first row of b that ends behind this one's start
				if (next < b.rows && next * step_b < reach + width)
					return true;
			}
			return false;
		}

		// logits, and their gradient if there is one
		int check_logits(const char * who, const nnf_matrix * x, const nnf_matrix * dx, int add, float temperature)
		{
			int st = check_rows(who, "logits", x, is_float);
			if (st == NNF_OK && dx)
				st = check_rows(who, "dlogits", dx, is_float);
			if (st != NNF_OK)
				return st;
			if (!(temperature >= 1.1754944e-38F) || !(temperature < INFINITY))   // 1/temperature is finite
				return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: temperature %g", who, (double)temperature);
			// a row's frame may hold a piece more than its elements fill
			const int64_t n = 16 / element_size(x->type);
			if ((x->cols + 2 * n - 2) / n > kMaxPieces)
				return set_error(NNF_ERR_UNSUPPORTED, "%s: rows of %lld scores: at most 1 MiB a row", who, (long long)x->cols);
			if (dx)
			{
				if (dx->type != x->type || dx->rows != x->rows || dx->cols != x->cols)
					return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: dlogits have another type or shape than the logits", who);
				if (dx->data == x->data && x->rows > 0 && (add || dx->stride != x->stride))
					return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: dlogits in the logits' place: with their stride, and not added to", who);
				if (dx->data != x->data && x->rows > 0 && overlap(*x, *dx))
					return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: dlogits overlap the logits", who);
			}
			return NNF_OK;
		}

		template <class... P>
		int launch_rows(void (*kernel)(P...), int64_t grid, int threads, size_t smem, int cluster, cudaStream_t s, const P&... args)
		{
			cudaLaunchAttribute attr[2];
			attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
			attr[0].val.programmaticStreamSerializationAllowed = 1;
			attr[1].id = cudaLaunchAttributeClusterDimension;
			attr[1].val.clusterDim.x = (unsigned)cluster;
			attr[1].val.clusterDim.y = 1;
			attr[1].val.clusterDim.z = 1;
			cudaLaunchConfig_t cfg = {};
			cfg.gridDim = dim3((unsigned)grid);
			cfg.blockDim = dim3((unsigned)threads);
			cfg.dynamicSmemBytes = smem;
			cfg.stream = s;
			cfg.attrs = attr;
			cfg.numAttrs = cluster > 1 ? 2 : 1;
			cudaLaunchKernelEx(&cfg, kernel, args...);   // the error, if any, is picked up by check_launch
			return check_launch("vocab_rows_kernel");
		}

		template <class K>
		int allow_shared(K kernel, size_t bytes, const char * who)
		{
			constexpr size_t granted = 44 * 1024;   // of 48 KB without being asked for, static data among them
			if (bytes <= granted)
				return NNF_OK;
			const int limit = running_config().max_shared_memory_per_block_optin - 4096;
			if (bytes > (size_t)limit)
				return set_error(NNF_ERR_UNSUPPORTED, "%s: %lld bytes of shared memory", who, (long long)bytes);
			// the attribute is the kernel's: the same value whatever the shape, so that host threads do not lower it under each other's launches
			const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, limit);
			return e == cudaSuccess ? NNF_OK : set_error(NNF_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", who, cudaGetErrorString(e));
		}

		template <class T, int OP>
		int run_held(cudaStream_t s, const vocab_params& v, int64_t pieces)
		{
			int64_t cluster = 1;
			while (cluster < kVocabCluster && pieces > cluster * 4200)
				cluster *= 2;
			// few rows: over more CTAs, as long as those are less than four an SM (32x32000 bf16 over 8 CTAs 4.8 us, over one 7.1; 148 rows over 2
			// 7.1 us, over 4 8.5, over one 7.5)
			while (cluster < kVocabCluster && v.rows * cluster * 2 < 4 * sm_count() && pieces > cluster * 512)
				cluster *= 2;
			if (tune().vocab_split > 0)
				cluster = tune().vocab_split < kVocabCluster ? tune().vocab_split : kVocabCluster;
			held_params p = {};
			p.v = v;
			p.v.cluster = (int)cluster;
			p.error = device_error_word();
			const int64_t per = div_up(pieces, cluster);
			// 16 pieces a thread, so that little is spent on joining threads; where the SMs are not full, four (16x32000 5.0 us, with eight
			// or 16 5.5; 256x32000 9.5, with 16 9.8)
			int threads = (int)(div_up(div_up(per, v.rows * cluster < 4 * sm_count() ? 4 : 16), 32) * 32);
			threads = threads < 64 ? 64 : threads > kHeldThreads ? kHeldThreads : threads;
			const int64_t chunk = int64_t(threads) * kHeldChunk;
			const bool aligned = v.dx && !v.add && ((reinterpret_cast<uintptr_t>(v.dx) ^ reinterpret_cast<uintptr_t>(v.x)) & 15) == 0 &&
				(v.rows < 2 || (v.lddx - v.ldx) * (int64_t)sizeof(T) % 16 == 0);
			const bool registers = aligned && threads == kHeldThreads && per >= 3 * chunk;
			p.slots = (int)((per - (registers ? chunk : 0) + 7) & ~int64_t(7));
			const size_t smem = size_t(p.slots) * 16 + (OP == kDistill ? size_t(v.kept) * (aligned ? 12 : 16) + size_t(div_up(per * piece<T>::N, 32)) * 4 : 0);
			auto kernel = registers ? vocab_held_kernel<T, OP, kRegisterRow> : aligned ? vocab_held_kernel<T, OP, kAlignedRow> : vocab_held_kernel<T, OP, kAnyRow>;
			const int st = allow_shared(kernel, smem, "vocab_held_kernel");
			if (st != NNF_OK)
				return st;
			return launch_rows(kernel, v.rows * cluster, threads, smem, (int)cluster, s, p);
		}

		template <class T>
		int run_score(cudaStream_t s, vocab_params& p, int64_t pieces)
		{
			const int64_t slots = (int64_t)sm_count() * 4 * kRowWarps;
			// In ns. Warps: what the last turn of all of them leaves unused; CTAs: 3/4 ns a row that starting and ending each costs. Warps / CTAs,
			// us: 16384x12000 70 / 75, 8192x8192 29 / 32, 32768x4096 52 / 85; the other way round 8192x32000 102 / 87, 4096x16384 28.1 / 27.6,
			// 1024x32000 22.7 / 15.3, 2048x131072 102 / 86
			const int64_t idle = (div_up(p.rows, slots) * slots - p.rows) * pieces * 16 / 6500, turnover = p.rows * 3 / 4;
			if (tune().vocab_form == 3 || (tune().vocab_form == 0 && idle < turnover))
			{
				const int64_t needed = div_up(p.rows, kRowWarps);
				launch(vocab_score_warp_kernel<T>, needed < slots / kRowWarps ? needed : slots / kRowWarps, kRowWarps * 32, 0, s, p);
				return check_launch("vocab_score_warp_kernel");
			}
			int64_t cluster = 1;
			while (cluster < kVocabCluster && p.rows * cluster < 2 * sm_count() && pieces > cluster * 512)
				cluster *= 2;
			if (tune().vocab_split > 0)
				cluster = tune().vocab_split < kVocabCluster ? tune().vocab_split : kVocabCluster;
			p.cluster = (int)cluster;
			int threads = (int)(div_up(div_up(div_up(pieces, cluster), 8), 32) * 32);
			// 128 threads a row: twice the rows of 256 are in flight, so that fewer of them are at their start or end (8192x32000 bf16 87
			// against 94 us, 3000x50000 54 / 58); 256 where that leaves the last turn emptier (2048x131072 86 against 89 us, 300x65536 12.7 / 14.5)
			const int most = p.rows < 4 * sm_count() || (pieces > 8192 && p.rows < 16 * sm_count()) ? kScoreThreads : kScoreThreads / 2;
			threads = threads > most ? most : threads;
			return launch_rows(vocab_score_kernel<T>, p.rows * cluster, threads, 0, (int)cluster, s, p);
		}

		template <class T, int OP, int NP>
		int run_short(cudaStream_t s, vocab_params& p)
		{
			const bool any = !p.dx || p.add || ((reinterpret_cast<uintptr_t>(p.dx) ^ reinterpret_cast<uintptr_t>(p.x)) & 15) != 0 ||
				(p.rows > 1 && (p.lddx - p.ldx) * (int64_t)sizeof(T) % 16 != 0);
			auto kernel = any ? vocab_short_kernel<T, OP, NP, true> : vocab_short_kernel<T, OP, NP, false>;
			const size_t smem = OP == kDistill ? size_t(kRowWarps) * 4 * (4 * size_t(p.kept) + NP * piece<T>::N + 1) : 0;
			const int st = allow_shared(kernel, smem, "vocab_short_kernel");
			if (st != NNF_OK)
				return st;
			const int64_t needed = div_up(p.rows, kRowWarps), resident = (int64_t)sm_count() * (NP > 4 ? 2 : 3);
			launch(kernel, needed < resident ? needed : resident, kRowWarps * 32, smem, s, p);
			return check_launch("vocab_short_kernel");
		}

		template <class T, int OP>
		int run_rows_of(cudaStream_t s, vocab_params& p)
		{
			constexpr int64_t n = piece<T>::N;
			const int64_t pieces = (p.cols + 2 * n - 2) / n;
			if constexpr (OP == kScore)
				return run_score<T>(s, p, pieces);
			else
			{
				// a warp's registers hold 256 pieces (32768x2000 bf16 61 us, in shared memory 80); longer rows would spill them
				if (pieces > 256 || tune().vocab_form == 2)
					return run_held<T, OP>(s, p, pieces);
				return pieces <= 32 ? run_short<T, OP, 1>(s, p) : pieces <= 64 ? run_short<T, OP, 2>(s, p) : pieces <= 128 ? run_short<T, OP, 4>(s, p) : run_short<T, OP, 8>(s, p);
			}
		}

		template <int OP>
		int run_rows(cudaStream_t s, vocab_params& p, const nnf_matrix& x, const nnf_matrix * dx, float temperature)
		{
			p.x = x.data; p.ldx = x.stride;
			p.dx = dx ? dx->data : nullptr; p.lddx = dx ? dx->stride : 0;
			p.add = dx && p.add;   // the loss alone is added to nothing: the kernels take `add` as leave to read what dx holds
			p.rows = x.rows; p.cols = (int)x.cols;
			p.tau = temperature;
			p.inv_tau = 1.0F / temperature;
			p.inv_rest = (float)(1.0 / (double)temperature - (double)p.inv_tau);
			p.k = 1.44269502162933349609375F / temperature;
			const double exact = 1.4426950408889634 / (double)temperature;
			p.k_down = (float)exact > exact ? nextafterf((float)exact, 0.0F) : (float)exact;
			// above 0, as it meets -infinity; no more above it than its type needs: beside a temperature of 1e37 k itself is 1e-37
			p.k_rest = fmaxf((float)(exact - (double)p.k_down), 1.4e-45F);
			switch (x.type)
			{
			case NNF_F32: return run_rows_of<float, OP>(s, p);
			case NNF_BF16: return run_rows_of<__nv_bfloat16, OP>(s, p);
			default: return run_rows_of<__half, OP>(s, p);
			}
		}

		int run_bwd(cudaStream_t s, vocab_bwd_params& p, const nnf_matrix& dx, const nnf_matrix& x, float temperature)
		{
			p.x = x.data; p.ldx = x.stride;
			p.dx = dx.data; p.lddx = dx.stride;
			p.rows = x.rows; p.cols = (int)x.cols;
			p.inv_tau = 1.0F / temperature;
			p.k = 1.44269502162933349609375F / temperature;
			const int64_t n = 16 / element_size(x.type), pieces = (x.cols + 2 * n - 2) / n;
			const int threads = pieces < kBwdThreads * kBwdPieces ? (int)div_up(div_up(pieces, kBwdPieces), 32) * 32 : kBwdThreads;
			p.slices = (int)div_up(pieces, threads * kBwdPieces);
			const bool aligned = !p.add && ((reinterpret_cast<uintptr_t>(dx.data) ^ reinterpret_cast<uintptr_t>(x.data)) & 15) == 0 &&
				(x.rows < 2 || (dx.stride - x.stride) * element_size(x.type) % 16 == 0);
			const int64_t most = 0x7fffffff / p.slices;   // rows of a launch
			for (p.last = x.rows - 1; p.last >= 0; p.last -= most)
			{
				const int64_t grid = (p.last + 1 < most ? p.last + 1 : most) * p.slices;
				switch (x.type)
				{
				case NNF_F32: launch(aligned ? vocab_bwd_kernel<float, true> : vocab_bwd_kernel<float, false>, grid, threads, 0, s, p); break;
				case NNF_BF16: launch(aligned ? vocab_bwd_kernel<__nv_bfloat16, true> : vocab_bwd_kernel<__nv_bfloat16, false>, grid, threads, 0, s, p); break;
				default: launch(aligned ? vocab_bwd_kernel<__half, true> : vocab_bwd_kernel<__half, false>, grid, threads, 0, s, p); break;
				}
				const int st = check_launch("vocab_bwd_kernel");
				if (st != NNF_OK)
					return st;
			}
			return NNF_OK;
		}
	}
}

using namespace nnf;

extern "C" int nnf_token_logp_fwd(nnf_stream_t stream, float * logp, float * saved, const nnf_matrix * logits, const nnf_indices * tokens, float temperature)
{
	const char * const who = "nnf_token_logp_fwd";
	int st = check_logits(who, logits, nullptr, 0, temperature);
	if (st != NNF_OK || logits->rows == 0)
		return st;
	if ((st = check_indices(who, "tokens", tokens)) != NNF_OK)
		return st;
	if (!logp)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
	vocab_params p = {};
	p.logp = logp; p.saved = saved;
	p.tokens = tokens->data; p.tokens_wide = tokens->type == NNF_I64;
	return run_rows<kScore>((cudaStream_t)stream, p, *logits, nullptr, temperature);
}

extern "C" int nnf_token_logp_bwd(nnf_stream_t stream, const nnf_matrix * dlogits, const float * dlogp, const nnf_matrix * logits, const nnf_indices * tokens,
	const float * saved, float temperature, int add_to_destination)
{
	const char * const who = "nnf_token_logp_bwd";
	if (!dlogits)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: dlogits: null pointer", who);
	int st = check_logits(who, logits, dlogits, add_to_destination, temperature);
	if (st != NNF_OK || logits->rows == 0)
		return st;
	if ((st = check_indices(who, "tokens", tokens)) != NNF_OK)
		return st;
	if (!dlogp || !saved)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
	vocab_bwd_params p = {};
	p.tokens = tokens->data; p.tokens_wide = tokens->type == NNF_I64;
	p.dlogp = dlogp; p.saved = saved;
	p.add = add_to_destination ? 1 : 0;
	return run_bwd((cudaStream_t)stream, p, *dlogits, *logits, temperature);
}

extern "C" int nnf_policy_loss(nnf_stream_t stream, float * loss, float * logp, float * kl, const nnf_matrix * dlogits, const nnf_matrix * logits,
	const nnf_indices * tokens, const float * old_logp, const float * advantages, const float * ref_logp, const float * mask,
	float clip_low, float clip_high, float kl_coef, float temperature, float scale, int add_to_destination)
{
	const char * const who = "nnf_policy_loss";
	int st = check_logits(who, logits, dlogits, add_to_destination, temperature);
	if (st != NNF_OK)
		return st;
	if (!(clip_low >= 0.0F) || !(clip_low <= 1.0F) || !(clip_high >= 0.0F))
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: ratios are held in [1 - %g, 1 + %g]", who, (double)clip_low, (double)clip_high);
	if (logits->rows == 0)
		return NNF_OK;
	if ((st = check_indices(who, "tokens", tokens)) != NNF_OK)
		return st;
	if (!loss || !logp || !old_logp || !advantages)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
	vocab_params p = {};
	p.loss = loss; p.logp = logp; p.kl = kl;
	p.tokens = tokens->data; p.tokens_wide = tokens->type == NNF_I64;
	p.old_logp = old_logp; p.advantages = advantages; p.ref_logp = ref_logp; p.mask = mask;
	p.low = 1.0F - clip_low; p.high = 1.0F + clip_high; p.kl_coef = kl_coef;
	p.scale = scale;
	p.add = add_to_destination ? 1 : 0;
	return run_rows<kPolicy>((cudaStream_t)stream, p, *logits, dlogits, temperature);
}

extern "C" int nnf_preference_loss(nnf_stream_t stream, float * loss, float * rewards, float * logp, float * saved, float * dlogp, const nnf_matrix * dlogits,
	const nnf_matrix * logits, const nnf_indices * tokens, const nnf_indices * offsets, int64_t pairs, const float * ref_logp, int kind, float beta,
	float label_smoothing, int average, float temperature, float scale, int add_to_destination)
{
	const char * const who = "nnf_preference_loss";
	int st = check_logits(who, logits, dlogits, add_to_destination, temperature);
	if (st != NNF_OK)
		return st;
	if (kind != NNF_PREFERENCE_LOGISTIC && kind != NNF_PREFERENCE_SQUARED)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: kind %d", who, kind);
	if (!(beta > 0.0F) || !(beta < INFINITY) || !(label_smoothing >= 0.0F) || !(label_smoothing <= 1.0F) || pairs < 0)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: beta %g, label smoothing %g, %lld pairs", who, (double)beta, (double)label_smoothing, (long long)pairs);
	if (pairs == 0)
		return NNF_OK;
	if (pairs > 0x3fffffff)
		return set_error(NNF_ERR_UNSUPPORTED, "%s: %lld pairs", who, (long long)pairs);
	if ((st = check_indices(who, "offsets", offsets)) != NNF_OK)
		return st;
	if (logits->rows > 0 && (st = check_indices(who, "tokens", tokens)) != NNF_OK)
		return st;
	if (!loss || !rewards || !ref_logp || (logits->rows > 0 && (!logp || !saved || !dlogp)))
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
	const cudaStream_t s = (cudaStream_t)stream;
	if (logits->rows > 0)
	{
		vocab_params p = {};
		p.logp = logp; p.saved = saved;
		p.tokens = tokens->data; p.tokens_wide = tokens->type == NNF_I64;
		p.offsets = offsets->data; p.offsets_wide = offsets->type == NNF_I64; p.sequences = 2 * pairs;
		if ((st = run_rows<kScore>(s, p, *logits, nullptr, temperature)) != NNF_OK)
			return st;
	}
	pair_params q = {};
	q.logp = logp; q.saved = saved; q.ref_logp = ref_logp;
	q.offsets = offsets->data; q.offsets_wide = offsets->type == NNF_I64;
	q.rows = logits->rows;
	q.loss = loss; q.rewards = rewards; q.dlogp = dlogp;
	q.beta = beta; q.smoothing = label_smoothing; q.scale = scale;
	q.kind = kind; q.average = average ? 1 : 0;
	launch(vocab_pair_kernel, pairs, kPairThreads, 0, s, q);
	if ((st = check_launch("vocab_pair_kernel")) != NNF_OK || !dlogits || logits->rows == 0)
		return st;
	vocab_bwd_params b = {};
	b.tokens = tokens->data; b.tokens_wide = tokens->type == NNF_I64;
	b.dlogp = dlogp; b.saved = saved;
	b.add = add_to_destination ? 1 : 0;
	b.offsets = offsets->data; b.offsets_wide = offsets->type == NNF_I64; b.sequences = 2 * pairs;
	return run_bwd(s, b, *dlogits, *logits, temperature);
}

extern "C" int nnf_distill_topk_loss(nnf_stream_t stream, float * loss, const nnf_matrix * dlogits, const nnf_matrix * logits, const nnf_matrix * teacher_ids,
	const nnf_matrix * teacher_logits, const float * mask, float temperature, float scale, int add_to_destination)
{
	const char * const who = "nnf_distill_topk_loss";
	int st = check_logits(who, logits, dlogits, add_to_destination, temperature);
	if (st == NNF_OK)
		st = check_rows(who, "teacher ids", teacher_ids, is_index);
	if (st == NNF_OK)
		st = check_rows(who, "teacher logits", teacher_logits, is_float);
	if (st != NNF_OK)
		return st;
	if (teacher_ids->rows != logits->rows || teacher_logits->rows != logits->rows || teacher_ids->cols != teacher_logits->cols)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: the teacher's ids and logits are [rows][kept]", who);
	if (teacher_ids->cols > kMaxKept)
		return set_error(NNF_ERR_UNSUPPORTED, "%s: %lld logits kept: at most %d", who, (long long)teacher_ids->cols, kMaxKept);
	if (logits->rows == 0)
		return NNF_OK;
	if (!loss)
		return set_error(NNF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
	vocab_params p = {};
	p.loss = loss; p.mask = mask;
	p.scale = scale;
	p.add = add_to_destination ? 1 : 0;
	p.ids = teacher_ids->data; p.ids_wide = teacher_ids->type == NNF_I64; p.ld_ids = teacher_ids->stride;
	p.teacher = teacher_logits->data; p.teacher_type = teacher_logits->type; p.ld_teacher = teacher_logits->stride;
	p.kept = (int)teacher_ids->cols;
	return run_rows<kDistill>((cudaStream_t)stream, p, *logits, dlogits, temperature);
}
