"""torchpp.llmops on B200: KV cache, LLM inference driver, decode engine."""
from .kvcache import KVCache  # noqa: F401
from .llm import LLMInference  # noqa: F401
from .scoring import PromptScores, pack, score  # noqa: F401
from .speculative import SpeculativeDecoder, lookup_draft, tree_mask  # noqa: F401
