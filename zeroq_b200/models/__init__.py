from .decoder import DecoderConfig, DecoderLM, DecoderLayer, LayerNorm, RMSNorm, PRESETS, get_config

__all__ = ["DecoderConfig", "DecoderLM", "DecoderLayer", "LayerNorm", "RMSNorm", "PRESETS", "get_config"]
