from ._embedding import embedding_lookup
from ._generate import Answer, generate, score
from ._int4 import Int4Linear
from ._linear_xent import linear_cross_entropy
from ._logprobs import TokenLogprobs, token_logprobs
from ._module import ChannelMixFFN, Linear, LowRankFFN, lecun_normal, linear_fp8
from ._orthogonalize import orthogonalize
from ._optimizer import lion_update, momentum_update, momentum_update_stacked, muon_update
from ._wkv7 import wkv_state_scan
