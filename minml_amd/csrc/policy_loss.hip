/*
 * policy_loss.hip — the clipped policy loss over the likelihoods of sampled tokens with a penalty for leaving a reference model, and its gradient.
 *
 * Of a token with negative log likelihood n now, o when it was sampled and f by the reference, and with advantage A:
 *   r = exp(o - n),   gain = min(r A, clip(r, 1 - low, 1 + high) A),   q = n - f,   kl = exp(q) - q - 1,   loss = -gain + kl_weight kl (with a weight of 0 without kl, whatever it is)
 * The result is the mean over the tokens, or over the sequences' means; the gradient of n is the token's weight times ([not clipped] r A + kl_weight (exp(q) - 1)).
 * Whether a token is clipped is decided in 64 bits by o - n against the logarithm of the border (r > 1 + high where A > 0, r < 1 - low where A < 0), so no rounding of an exponential moves a token across it.
 * r is a number of 64 bits that holds 32: beyond exp(88) it is none of fp32, but its product with an advantage or a weight may be one, and with an advantage of 0 is 0. A token without an advantage has no gain whatever its
 * likelihoods are, as long as they are numbers or infinite.
 * kl of close models is a small number from which 1 and q have been taken: below |q| = 1/2 it is q^2 (1/2 + q/6 + ..), where nothing cancels. Sums are in 64 bits: gains have both signs and cancel.
 * Memory bounds both passes, 12 to 20 bytes of a token: 1024 sequences of 8191 tokens, all five inputs, 28 us and 5 to join the sums (6.0 TB/s), the gradient 30 (6.8, partly from the last-level cache); 512 x 1024 6.2 and 2.9.
 */
#include "training_utils.hpp"

#include <algorithm>
#include <cmath>

namespace
{
	using namespace mlhip;

	struct PolicyArgs
	{
			const float *nll, *old, *reference, *advantages; /* reference: or null */
			const int *targets;
			int sequences, length, classes;
			bool per_token; /* advantages: of every token, else of every sequence */
			double log_low, log_high;
			double low, high;
			float kl_weight;
	};
	struct TokenLoss
	{
			double gain, slope, kl, kl_slope;
			bool clipped;
	};
	/* exp(x) = 2^f 2^n with the 32 bits of the hardware's 2^f, f in [-1/2, 1/2], at any power of two that 64 bits reach. Infinities and NaN, and what is beyond, go by f: so does what is left of x by then */
	__device__ __forceinline__ double exp_of(double x)
	{
		const double t = x * 1.4426950408889634 /* 1 / log 2 */, n = rint(fmin(fmax(t, -1100.0), 1100.0));
		return ldexp(static_cast<double>(__builtin_amdgcn_exp2f(static_cast<float>(t - n))), static_cast<int>(n));
	}
	__device__ __forceinline__ TokenLoss token_loss(const PolicyArgs &p, float nll, float old, float reference, float advantage)
	{
		TokenLoss t;
		const double d = static_cast<double>(old) - static_cast<double>(nll);
		const bool up = advantage > 0.0f && d > p.log_high, down = advantage < 0.0f && d < p.log_low;
		t.clipped = up || down;
		const double a = static_cast<double>(advantage), free = (a == 0.0 && d == d) ? 0.0 : exp_of(d) * a;
		t.gain = up ? p.high * a : down ? p.low * a : free;
		t.slope = t.clipped ? 0.0 : free;
		t.kl = t.kl_slope = 0.0;
		if (p.reference != nullptr)
		{
			const double wide = static_cast<double>(nll) - static_cast<double>(reference);
			const float q = static_cast<float>(wide);
			/* the terms left out are below 2^-28 of the sum */
			float series = 1.0f / 362880.0f;
			series = fmaf(series, q, 1.0f / 40320.0f);
			series = fmaf(series, q, 1.0f / 5040.0f);
			series = fmaf(series, q, 1.0f / 720.0f);
			series = fmaf(series, q, 1.0f / 120.0f);
			series = fmaf(series, q, 1.0f / 24.0f);
			series = fmaf(series, q, 1.0f / 6.0f);
			series = fmaf(series, q, 0.5f);
			const float close = series * q * q;
			const double beyond = exp_of(wide) - 1.0;
			const bool is_close = fabsf(q) < 0.5f;
			t.kl = is_close ? static_cast<double>(close) : beyond < HUGE_VAL ? beyond - wide : beyond;
			t.kl_slope = is_close ? static_cast<double>(close + q) : beyond;
		}
		return t;
	}
	/* the tokens of VEC neighbouring places of a sequence */
	template<int VEC>
	struct Tokens
	{
			Elements<float, VEC> nll, old, reference, advantages;
			Elements<int, VEC> targets;
			float advantage;
			int skip;

			__device__ __forceinline__ void load(const PolicyArgs &p, int sequence, int first)
			{
				const RowPlace place = place_in_row<VEC>(first, p.length);
				const size_t row = static_cast<size_t>(sequence) * p.length;
				skip = place.skip;
				targets.load(place.in(p.targets + row));
				nll.load(place.in(p.nll + row));
				old.load(place.in(p.old + row));
				if (p.reference != nullptr)
					reference.load(place.in(p.reference + row));
				if (p.per_token)
					advantages.load(place.in(p.advantages + row));
				else
					advantage = p.advantages[sequence];
			}
			__device__ __forceinline__ bool there(const PolicyArgs &p, int e) const
			{
				const int target = target_of(e);
				return e >= skip && target >= 0 && target < p.classes;
			}
			__device__ __forceinline__ int target_of(int e) const
			{
				if constexpr (VEC == 1)
					return targets.raw;
				else
					return targets.raw[e];
			}
			__device__ __forceinline__ TokenLoss loss(const PolicyArgs &p, int e) const
			{
				return token_loss(p, nll[e], old[e], p.reference != nullptr ? reference[e] : 0.0f, p.per_token ? advantages[e] : advantage);
			}
	};

	/* of some tokens: sums of gains and divergences, clipped ones, all of them. Where sequences are averaged: means of whole sequences added up, and sequences with tokens */
	struct Sums
	{
			double gain, kl, clipped, count;
	};
	__device__ __forceinline__ Sums operator+(const Sums &a, const Sums &b)
	{
		return Sums { a.gain + b.gain, a.kl + b.kl, a.clipped + b.clipped, a.count + b.count };
	}
	template<int LANES>
	__device__ __forceinline__ Sums lanes_sum(Sums s)
	{
#pragma unroll
		for (int offset = LANES / 2; offset >= 1; offset >>= 1)
			s = s + Sums { __shfl_xor(s.gain, offset), __shfl_xor(s.kl, offset), __shfl_xor(s.clipped, offset), __shfl_xor(s.count, offset) };
		return s;
	}
	/* of a workgroup of 256 threads, for all of them */
	__device__ __forceinline__ Sums group_sum(Sums s, Sums (&waves)[4])
	{
		s = lanes_sum<64>(s);
		if ((threadIdx.x & 63) == 0)
			waves[threadIdx.x >> 6] = s;
		__syncthreads();
		s = (waves[0] + waves[1]) + (waves[2] + waves[3]);
		__syncthreads();
		return s;
	}
	__device__ __forceinline__ Sums mean_of_sequence(const Sums &s)
	{
		return s.count > 0.0 ? Sums { s.gain / s.count, s.kl / s.count, s.clipped / s.count, 1.0 } : Sums { 0.0, 0.0, 0.0, 0.0 };
	}
	/* the loss of all means, by one thread */
	__device__ __forceinline__ void write_loss(const Sums &total, double each, float kl_weight, float *loss)
	{
		const double gain = total.gain * each, kl = total.kl * each;
		loss[0] = static_cast<float>((kl_weight != 0.0f ? kl_weight * kl : 0.0) - gain);
		loss[1] = static_cast<float>(-gain);
		loss[2] = static_cast<float>(kl);
		loss[3] = static_cast<float>(total.clipped * each);
	}
	/* what a token of a sequence counts */
	__device__ __forceinline__ float weight_of_sequence(double count, double each, bool average_sequences)
	{
		return static_cast<float>(count > 0.0 ? (average_sequences ? each / count : each) : 0.0);
	}
	/* of the tokens [begin, end) of a sequence those of one of LANES threads */
	template<int LANES, int VEC>
	__device__ __forceinline__ Sums sums_of_thread(const PolicyArgs &p, int sequence, int begin, int end)
	{
		Sums sums { 0.0, 0.0, 0.0, 0.0 };
		int clipped = 0, count = 0;
		for (int i = begin + (static_cast<int>(threadIdx.x) % LANES) * VEC; i < end; i += LANES * VEC)
		{
			Tokens<VEC> tokens;
			tokens.load(p, sequence, i);
#pragma unroll
			for (int e = 0; e < VEC; e++)
				if (tokens.there(p, e))
				{
					const TokenLoss t = tokens.loss(p, e);
					sums.gain += t.gain;
					sums.kl += t.kl;
					clipped += t.clipped ? 1 : 0;
					count++;
				}
		}
		sums.clipped = clipped;
		sums.count = count;
		return sums;
	}
	/*
	 * Sums of the workgroups. Whole sequences by LANES threads each, `sequences_of_group` by a workgroup (chunk_length 0), or a workgroup for every chunk_length tokens of a sequence (gridDim.y of them).
	 * counts: tokens of every sequence, where they are whole
	 */
	template<int LANES, int VEC>
	__global__ __launch_bounds__(256) void kernel_policy_sums(PolicyArgs p, int sequences_of_group, int chunk_length, bool average_sequences, Sums *partial, int *counts)
	{
		__shared__ Sums waves[4];
		const int begin = blockIdx.y * chunk_length, end = chunk_length > 0 ? begin + min(chunk_length, p.length - begin) : p.length;
		const int first = blockIdx.x * sequences_of_group, last = first + min(sequences_of_group, p.sequences - first);
		Sums total { 0.0, 0.0, 0.0, 0.0 };
		for (int s0 = first; s0 < last; s0 += 256 / LANES)
		{
			const int sequence = s0 + static_cast<int>(threadIdx.x) / LANES;
			Sums sums { 0.0, 0.0, 0.0, 0.0 };
			if (sequence < last)
				sums = sums_of_thread<LANES, VEC>(p, sequence, begin, end);
			if constexpr (LANES == 256)
				sums = group_sum(sums, waves);
			else
				sums = lanes_sum<LANES>(sums);
			if (sequence < last && threadIdx.x % LANES == 0)
			{
				if (chunk_length == 0)
				{
					counts[sequence] = static_cast<int>(sums.count);
					if (average_sequences)
						sums = mean_of_sequence(sums);
				}
				total = total + sums;
			}
		}
		total = group_sum(total, waves);
		if (threadIdx.x == 0)
			partial[static_cast<size_t>(blockIdx.x) * gridDim.y + blockIdx.y] = total;
	}
	/*
	 * The workgroups' sums joined (every group does it for itself, the first one gives the loss), then the weights of a token of every sequence. `chunks`: of a sequence, whose sums `partial` holds; else (0) of `items` workgroups.
	 * One thread walks a sequence's chunks, twice, which bounds few sequences that are very long: us of this launch and of the sums', 1 sequence of 2^20 tokens (256 chunks) 50 and 8, 4 of 2^20 56 and 17; a call of one of 2^22 213,
	 * of 2^18 23
	 */
	__global__ __launch_bounds__(256) void kernel_policy_join(const Sums *partial, int items, int chunks, bool average_sequences, int sequences, float kl_weight, const int *counts, float *loss, float *weights)
	{
		__shared__ Sums waves[4];
		Sums total { 0.0, 0.0, 0.0, 0.0 };
		const auto of_sequence = [&](int s)
		{
			Sums sums { 0.0, 0.0, 0.0, 0.0 };
			for (int c = 0; c < chunks; c++)
				sums = sums + partial[static_cast<size_t>(s) * chunks + c];
			return sums;
		};
		for (int i = threadIdx.x; i < items; i += 256)
		{
			Sums sums = chunks > 0 ? of_sequence(i) : partial[i];
			if (chunks > 0 && average_sequences)
				sums = mean_of_sequence(sums);
			total = total + sums;
		}
		total = group_sum(total, waves);
		const double each = total.count > 0.0 ? 1.0 / total.count : 0.0;
		if (blockIdx.x == 0 && threadIdx.x == 0)
			write_loss(total, each, kl_weight, loss);
		for (int s = blockIdx.x * 256 + threadIdx.x; s < sequences; s += gridDim.x * 256)
		{
			const double count = chunks > 0 ? of_sequence(s).count : static_cast<double>(counts[s]);
			weights[s] = weight_of_sequence(count, each, average_sequences);
		}
	}

	/* few tokens: everything by one workgroup, LANES threads to a sequence */
	constexpr int FEW_THREADS = 1024, FEW_SEQUENCES = 512;
	template<int LANES, int VEC>
	__global__ __launch_bounds__(FEW_THREADS) void kernel_policy_few(PolicyArgs p, bool average_sequences, float *loss, float *weights)
	{
		constexpr int WAVES = FEW_THREADS / 64;
		__shared__ Sums waves[WAVES];
		__shared__ int counts[FEW_SEQUENCES];
		Sums total { 0.0, 0.0, 0.0, 0.0 };
		for (int s0 = 0; s0 < p.sequences; s0 += FEW_THREADS / LANES)
		{
			const int s = s0 + static_cast<int>(threadIdx.x) / LANES;
			Sums sums { 0.0, 0.0, 0.0, 0.0 };
			if (s < p.sequences)
				sums = sums_of_thread<LANES, VEC>(p, s, 0, p.length);
			sums = lanes_sum<LANES>(sums);
			if (s < p.sequences && threadIdx.x % LANES == 0)
			{
				counts[s] = static_cast<int>(sums.count);
				total = total + (average_sequences ? mean_of_sequence(sums) : sums);
			}
		}
		total = lanes_sum<64>(total);
		if ((threadIdx.x & 63) == 0)
			waves[threadIdx.x >> 6] = total;
		__syncthreads();
		total = waves[0];
#pragma unroll
		for (int w = 1; w < WAVES; w++)
			total = total + waves[w];
		const double each = total.count > 0.0 ? 1.0 / total.count : 0.0;
		if (threadIdx.x == 0)
			write_loss(total, each, p.kl_weight, loss);
		for (int s = threadIdx.x; s < p.sequences; s += FEW_THREADS)
			weights[s] = weight_of_sequence(counts[s], each, average_sequences);
	}

	/* dnll = dloss * weight of the sequence * slope + beta dnll */
	template<int VEC>
	__global__ __launch_bounds__(256) void kernel_policy_gradient(PolicyArgs p, int vectors, const float *weights, const float *dloss, float beta, float *dnll)
	{
		const size_t count = static_cast<size_t>(p.sequences) * vectors;
		const float scale = dloss != nullptr ? *dloss : 1.0f;
		for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < count; i += static_cast<size_t>(gridDim.x) * 256)
		{
			int vector;
			const int sequence = static_cast<int>(split_index(i, vectors, vector));
			const RowPlace place = place_in_row<VEC>(vector * VEC, p.length);
			float *dst = place.in(dnll + static_cast<size_t>(sequence) * p.length);
			Tokens<VEC> tokens;
			tokens.load(p, sequence, vector * VEC);
			const double weight = static_cast<double>(weights[sequence]) * static_cast<double>(scale);
			Elements<float, VEC> before;
			if (beta != 0.0f)
				before.load(dst);
			float v[VEC];
#pragma unroll
			for (int e = 0; e < VEC; e++)
			{
				v[e] = 0.0f;
				if (tokens.there(p, e))
				{
					const TokenLoss t = tokens.loss(p, e);
					v[e] = static_cast<float>(weight * (p.kl_weight != 0.0f ? fma(static_cast<double>(p.kl_weight), t.kl_slope, t.slope) : t.slope));
				}
				if (beta != 0.0f)
					v[e] = fmaf(beta, before[e], v[e]);
			}
			store_nearest<VEC>(dst, v, place.skip);
		}
	}

	struct PolicyPlan
	{
			int lanes, sequences_of_group, groups, chunks, chunk_length;
	};
	constexpr int MOST_GROUPS = 1024;
	/*
	 * Every group's sums are read by the join, so there are 1024 of them at most; sequences are cut where there are too few of them to give every compute unit work. us of a forward call, sequences of up to 1024 tokens by a
	 * wavefront / by a workgroup: 4096 x 1024 19.0 / 22.9, 4096 x 300 12.6 / 19.4, 2048 x 1024 12.4 / 15.0, 2048 x 512 12.2 / 13.8; 512 x 1024 12.8 / 12.4, of which the sums are 7.9 / 6.2
	 */
	PolicyPlan policy_plan(int sequences, int length)
	{
		PolicyPlan plan { };
		plan.lanes = length <= 64 ? 8 : length <= 256 || (length <= 1024 && sequences >= 2048) ? 64 : 256;
		const int at_a_time = 256 / plan.lanes;
		plan.sequences_of_group = static_cast<int>(round_up(std::max(1, ceil_div(sequences, MOST_GROUPS)), at_a_time));
		plan.groups = ceil_div(sequences, plan.sequences_of_group);
		if (plan.lanes == 256 && sequences > 0 && sequences <= MOST_GROUPS / 2 && length >= 8192)
		{
			plan.chunk_length = static_cast<int>(round_up(std::max(4096, ceil_div(length, MOST_GROUPS / sequences)), 4));
			plan.chunks = ceil_div(length, plan.chunk_length);
		}
		return plan;
	}
	struct PolicyShape
	{
			int sequences, length;
	};
	PolicyShape policy_shape(const mlShape_t &s, const char *name)
	{
		const std::string who(name);
		MLHIP_REQUIRE(s.rank == 1 || s.rank == 2, who + ": the likelihoods must be [sequences, tokens] or [tokens]");
		const int sequences = s.rank == 2 ? s.dim[0] : 1, length = s.dim[s.rank - 1];
		MLHIP_REQUIRE(sequences >= 0 && length >= 0, who + ": negative dimension");
		MLHIP_REQUIRE(sequences <= (1 << 28) && length <= (1 << 28), who + ": too many sequences or tokens");
		return PolicyShape { sequences, length };
	}
	/*
	 * Threads of a sequence where one workgroup does everything, or 0 where two launches do. It takes about 2 us for every time that a thread goes to memory, and saves what a launch costs: us of a forward call and (on the device,
	 * profiled), so / in two launches: 4 x 113 tokens, once, 10.6 (6.1) / 14.1 (5.6); 32 x 128, twice, 10.9 (10.1) / 13.9 (6.6); 200 x 40, four times, 10.9 (10.1) / 14.0 (8.4); 32 x 512, four times, 13.0 (12.2) / 14.1 (6.7);
	 * 64 x 500, eight times, 21 (21) / 14.2 (6.6)
	 */
	int lanes_of_few(const PolicyShape &s)
	{
		if (s.sequences > FEW_SEQUENCES)
			return 0;
		const auto times = [&](int lanes)
		{
			return static_cast<long long>(ceil_div(s.sequences, FEW_THREADS / lanes)) * ceil_div(s.length, 4 * lanes);
		};
		const int lanes = times(8) < times(64) ? 8 : 64;
		return times(lanes) <= 4 ? lanes : 0;
	}
	size_t policy_space(const PolicyShape &s)
	{
		if (lanes_of_few(s) > 0)
			return 0;
		const PolicyPlan plan = policy_plan(s.sequences, s.length);
		return round_up(sizeof(Sums) * (plan.chunks > 0 ? static_cast<size_t>(s.sequences) * plan.chunks : plan.groups), 256) + sizeof(int) * s.sequences;
	}
	bool of_tokens(const mlTensor_t &t, const PolicyShape &s, mlDataType_t dtype)
	{
		const size_t tokens = static_cast<size_t>(s.sequences) * s.length;
		return t.dtype == dtype && volume(t) == tokens && (tokens == 0 || t.data != nullptr) && on_elements(t);
	}
	PolicyArgs check_policy(const mlTensor_t &nll, const mlTensor_t &old, const mlTensor_t &reference, const mlTensor_t &advantages, const mlTensor_t &targets, int classes, double clip_low, double clip_high,
			float kl_weight, const char *name)
	{
		const std::string who(name);
		const PolicyShape s = policy_shape(shape_of(nll), name);
		MLHIP_REQUIRE(of_tokens(nll, s, DTYPE_FLOAT32) && of_tokens(old, s, DTYPE_FLOAT32), who + ": likelihoods must be fp32, as many old as new ones");
		MLHIP_REQUIRE(reference.data == nullptr || of_tokens(reference, s, DTYPE_FLOAT32), who + ": the reference's likelihoods must be fp32, one for every token");
		MLHIP_REQUIRE(of_tokens(targets, s, DTYPE_INT32), who + ": there must be one int32 target for every token");
		const size_t given = volume(advantages), tokens = static_cast<size_t>(s.sequences) * s.length;
		MLHIP_REQUIRE(advantages.dtype == DTYPE_FLOAT32 && (given == tokens || given == static_cast<size_t>(s.sequences)) && (tokens == 0 || advantages.data != nullptr) && on_elements(advantages),
				who + ": there must be one fp32 advantage for every token or every sequence");
		MLHIP_REQUIRE(clip_low >= 0.0 && clip_high >= 0.0, who + ": the clip's range must not be negative");
		MLHIP_REQUIRE(std::isfinite(kl_weight), who + ": the divergence's weight must be finite");
		const double low = 1.0 - clip_low, high = 1.0 + clip_high;
		return PolicyArgs { ptr<float>(nll), ptr<float>(old), ptr<float>(reference), ptr<float>(advantages), ptr<int>(targets), s.sequences, s.length, classes, given == tokens,
				low > 0.0 ? std::log(low) : -HUGE_VAL, std::log(high), std::max(low, 0.0), high, reference.data != nullptr ? kl_weight : 0.0f };
	}
}

extern "C"
{
	using namespace mlhip;

	size_t hip_policy_loss_get_workspace_size(mlShape_t shape)
	try
	{
		return policy_space(policy_shape(shape, "policy_loss_get_workspace_size"));
	}
	catch (...)
	{
		return mlhip::entry_failed<size_t>();
	}

	void hip_policy_loss_forward(mlContext_t context, const mlTensor_t nll, const mlTensor_t old_nll, const mlTensor_t reference_nll, const mlTensor_t advantages, const mlTensor_t targets, int classes,
			double clip_low, double clip_high, float kl_weight, mlAverage_t average, mlTensor_t loss, mlTensor_t weights, void *workspace, size_t workspace_size)
	try
	{
		const char *name = "policy_loss_forward";
		const PolicyArgs p = check_policy(nll, old_nll, reference_nll, advantages, targets, classes, clip_low, clip_high, kl_weight, name);
		MLHIP_REQUIRE(average == AVERAGE_TOKENS || average == AVERAGE_SEQUENCES, "policy_loss_forward: unknown average");
		MLHIP_REQUIRE(loss.dtype == DTYPE_FLOAT32 && volume(loss) == 4 && loss.data != nullptr && on_elements(loss), "policy_loss_forward: the loss must be fp32 [4], aligned to an element");
		MLHIP_REQUIRE(weights.dtype == DTYPE_FLOAT32 && volume(weights) == static_cast<size_t>(p.sequences) && (p.sequences == 0 || weights.data != nullptr) && on_elements(weights),
				"policy_loss_forward: the weights must be fp32, one for every sequence, aligned to an element");
		const PolicyShape s { p.sequences, p.length };
		const size_t needed = policy_space(s);
		MLHIP_REQUIRE(needed == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 && workspace_size >= needed),
				"policy_loss_forward: the workspace is too small or not aligned to 256 bytes");
		require_apart( { loss, weights, Extent(workspace, workspace_size) }, { nll, old_nll, reference_nll, advantages, targets }, name);
		const OnDeviceOf on(context);
		const PolicyPlan plan = policy_plan(p.sequences, p.length);
		const bool average_sequences = average == AVERAGE_SEQUENCES;
		if (const int lanes = lanes_of_few(s))
		{
			const auto launch = [&](auto kernel)
			{
				hipLaunchKernelGGL(kernel, dim3(1), dim3(FEW_THREADS), 0, on.stream, p, average_sequences, ptr<float>(loss), ptr<float>(weights));
			};
			if (p.length < 4)
				launch(kernel_policy_few<8, 1>);
			else if (lanes == 8)
				launch(kernel_policy_few<8, 4>);
			else
				launch(kernel_policy_few<64, 4>);
			MLHIP_CHECK(hipGetLastError());
			return;
		}
		Sums *partial = reinterpret_cast<Sums*>(workspace);
		const size_t units = plan.chunks > 0 ? static_cast<size_t>(p.sequences) * plan.chunks : plan.groups;
		int *counts = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(workspace) + round_up(sizeof(Sums) * units, 256));
		if (p.sequences > 0)
		{
			const dim3 grid(plan.groups, std::max(1, plan.chunks));
			const auto launch = [&](auto kernel)
			{
				hipLaunchKernelGGL(kernel, grid, dim3(256), 0, on.stream, p, plan.sequences_of_group, plan.chunk_length, average_sequences, partial, counts);
			};
			if (p.length < 4)
				launch(kernel_policy_sums<8, 1>);
			else if (plan.lanes == 8)
				launch(kernel_policy_sums<8, 4>);
			else if (plan.lanes == 64)
				launch(kernel_policy_sums<64, 4>);
			else
				launch(kernel_policy_sums<256, 4>);
			MLHIP_CHECK(hipGetLastError());
		}
		hipLaunchKernelGGL(kernel_policy_join, dim3(std::max(1, std::min(ceil_div(p.sequences, 256), 256))), dim3(256), 0, on.stream, partial, plan.chunks > 0 ? p.sequences : plan.groups, plan.chunks,
				average_sequences, p.sequences, p.kl_weight, counts, ptr<float>(loss), ptr<float>(weights));
		MLHIP_CHECK(hipGetLastError());
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}

	void hip_policy_loss_backward(mlContext_t context, const mlTensor_t nll, const mlTensor_t old_nll, const mlTensor_t reference_nll, const mlTensor_t advantages, const mlTensor_t targets, int classes,
			double clip_low, double clip_high, float kl_weight, const mlTensor_t weights, const mlTensor_t dloss, float beta, mlTensor_t dnll)
	try
	{
		const char *name = "policy_loss_backward";
		const PolicyArgs p = check_policy(nll, old_nll, reference_nll, advantages, targets, classes, clip_low, clip_high, kl_weight, name);
		MLHIP_REQUIRE(weights.dtype == DTYPE_FLOAT32 && volume(weights) == static_cast<size_t>(p.sequences) && (p.sequences == 0 || weights.data != nullptr) && on_elements(weights),
				"policy_loss_backward: the weights must be fp32, one for every sequence, aligned to an element");
		MLHIP_REQUIRE(dloss.data == nullptr || (dloss.dtype == DTYPE_FLOAT32 && volume(dloss) == 1 && on_elements(dloss)), "policy_loss_backward: the loss's gradient must be a single fp32 number, aligned to an element");
		const PolicyShape s { p.sequences, p.length };
		MLHIP_REQUIRE(of_tokens(dnll, s, DTYPE_FLOAT32), "policy_loss_backward: the gradient must be fp32, one for every token");
		if (volume(dnll) == 0)
			return;
		require_apart( { dnll }, { nll, old_nll, reference_nll, advantages, targets, weights, dloss }, name);
		const OnDeviceOf on(context);
		const int vectors = p.length < 4 ? p.length : ceil_div(p.length, 4);
		const dim3 grid(static_cast<unsigned int>(std::min<size_t>((static_cast<size_t>(p.sequences) * vectors + 255) / 256, 1 << 16)));
		if (p.length < 4)
			hipLaunchKernelGGL((kernel_policy_gradient<1>), grid, dim3(256), 0, on.stream, p, vectors, ptr<float>(weights), ptr<float>(dloss), beta, ptr<float>(dnll));
		else
			hipLaunchKernelGGL((kernel_policy_gradient<4>), grid, dim3(256), 0, on.stream, p, vectors, ptr<float>(weights), ptr<float>(dloss), beta, ptr<float>(dnll));
		MLHIP_CHECK(hipGetLastError());
	}
	catch (...)
	{
		return mlhip::entry_failed<void>();
	}
}
