"""What a decoder needs around its quantized linears: rotary positions, the quantized key/value cache and attention over it, and
the log probabilities of tokens.  No counterpart in the reference, whose quantized path ends at the linears."""
from .rotary import rotary_table, rotary_embedding
from .cache import quantized_cache, quantized_cache_append, quantized_cache_read
from .attention import quantized_cache_attention
from .log_probs import token_log_probs
