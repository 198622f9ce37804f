from .logprobs import TokenLogprob
from .params import SamplingParams, GREEDY, MAX_LOGPROBS, MAX_TOP_K
from .rng import uniform, resolve_seed, splitmix64

__all__ = ["SamplingParams", "GREEDY", "MAX_LOGPROBS", "MAX_TOP_K", "TokenLogprob", "uniform", "resolve_seed", "splitmix64"]
