from .cross_entropy import CrossEntropyLoss, tied_cross_entropy
from .sampled_cross_entropy import SampledCrossEntropyLoss, sample_negative_indices
from .logprobs import TokenLogProbs, tied_token_logprobs, token_logprobs

__all__ = ["CrossEntropyLoss", "SampledCrossEntropyLoss", "sample_negative_indices", "tied_cross_entropy",
           "TokenLogProbs", "token_logprobs", "tied_token_logprobs"]
