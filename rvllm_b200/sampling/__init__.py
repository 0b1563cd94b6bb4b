from .params import GREEDY, SamplingParams
from .logprobs import LogprobReader, TokenLogprob
from .sampler import BatchSampler
