"""Model assembly.  Importing this package registers the built-in architectures."""
from dataclasses import replace

from ..config.model_config import ConfigError
from . import bosenex, bubotar, bumotar, megusun, qwen3, rikolix, topunex  # noqa: F401
from .decoder import DecoderModel


def build_model(config, dtype, cache_bits: int = 0):
    """A ``DecoderModel`` (without weights) for a typed configuration: anything with ``model_spec()``.  ``cache_bits`` 4: its layers cache keys
    and values in 4 bits; refused where a layer's mixer has no such form."""
    spec = config.model_spec()
    if cache_bits:
        try:
            if any(b.mixer.kind != "attention" for b in spec.blocks):
                raise ValueError(f"mixers {sorted({b.mixer.kind for b in spec.blocks} - {'attention'})} have no cache of {cache_bits} bits")
            return DecoderModel(replace(spec, blocks=tuple(replace(b, mixer=replace(b.mixer, cache_bits=cache_bits)) for b in spec.blocks)), dtype)
        except ValueError as e:
            raise ConfigError(f"cache_bits={cache_bits}: {e}") from None
    return DecoderModel(spec, dtype)
