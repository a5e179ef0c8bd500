from .params import SamplingParams, TokenChoice
from .rng import SplitMix64
from .rules import TokenRules, pack_mask
from .sampler import InvalidLogits, Sampler, sample_top_p_host
