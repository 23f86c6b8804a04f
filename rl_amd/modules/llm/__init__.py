from .decode import GraphedGPT2Decoder, PagedGPT2Decoder
from .paged_cache import PagedKVCache
from .transformers_wrapper import LLMWrapperBase, TransformersWrapper
from .vllm_wrapper import SGLangWrapper, vLLMWrapper
