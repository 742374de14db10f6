"""Model hyper-parameters, with the reference's constructor, defaults and validation (forgeserve/config.py:7-39), and
the rotary forms that the reference lacks (rope_layout, rotary_dim, rope_scaling)."""

import math
from dataclasses import asdict, dataclass
from numbers import Integral, Real
from typing import Optional

_SCALING_KEYS = {"linear": {"factor"}, "ntk": {"factor"},
                 "by_parts": {"factor", "original_max_len", "beta_slow", "beta_fast", "attn_factor"}}


def check_rope_scaling(scaling: Optional[dict]) -> None:
    if scaling is None:
        return
    if not isinstance(scaling, dict):
        raise ValueError("rope_scaling must be a dict with a kind and a factor")
    kind = scaling.get("kind")
    if not isinstance(kind, str) or kind not in _SCALING_KEYS:
        raise ValueError(f"rope_scaling kind must be one of {sorted(_SCALING_KEYS)}, not {kind!r}")
    extra = set(scaling) - _SCALING_KEYS[kind] - {"kind"}
    if extra:
        raise ValueError(f"rope_scaling kind {kind!r} does not take {sorted(extra)}")
    for name in set(scaling) - {"kind"}:
        value = scaling[name]
        if isinstance(value, bool) or not isinstance(value, Real) or not math.isfinite(value):
            raise ValueError(f"rope_scaling {name} must be a finite number, not {value!r}")
    if not scaling.get("factor", 0) >= 1:
        raise ValueError("rope_scaling needs a factor of at least 1")
    if kind == "by_parts":
        if not scaling.get("original_max_len", 0) > 0:
            raise ValueError("rope_scaling by parts needs original_max_len")
        if not 0 < scaling.get("beta_slow", 1.0) < scaling.get("beta_fast", 32.0):
            raise ValueError("rope_scaling needs 0 < beta_slow < beta_fast")
        if not scaling.get("attn_factor", 1.0) > 0:
            raise ValueError("rope_scaling attn_factor must be positive")


@dataclass
class ModelConfig:
    vocab_size: int = 256
    d_model: int = 128
    n_layers: int = 4
    n_heads: int = 8
    n_kv_heads: int = 4            # grouped-query attention: query head h reads KV head h // (n_heads // n_kv_heads)
    ffn_dim: Optional[int] = None  # default: 8/3 * d_model rounded up to a multiple of 64 (config.py:21)
    max_seq_len: int = 256
    rope_theta: float = 10000.0
    norm_eps: float = 1e-5
    # Extras (none in the reference; to_dict leaves them out while they hold these defaults):
    rope_layout: str = "half"            # pairs (x[i], x[i + r/2]); "interleaved": (x[2i], x[2i+1])
    rotary_dim: Optional[int] = None     # r: the first values of a head that turn (default: all of them)
    rope_scaling: Optional[dict] = None  # long contexts: {"kind": "linear" | "ntk" | "by_parts", "factor": f, ...}

    def __post_init__(self):
        if self.ffn_dim is None:
            self.ffn_dim = -(-int(8 / 3 * self.d_model) // 64) * 64
        if self.d_model % self.n_heads:
            raise ValueError(f"d_model ({self.d_model}) must be divisible by n_heads ({self.n_heads})")
        if self.n_heads % self.n_kv_heads:
            raise ValueError(f"n_heads ({self.n_heads}) must be divisible by n_kv_heads ({self.n_kv_heads})")
        if self.head_dim % 2:
            raise ValueError("head_dim must be even for rotary embeddings")
        if self.rope_layout not in ("half", "interleaved"):
            raise ValueError(f"rope_layout must be 'half' or 'interleaved', not {self.rope_layout!r}")
        r = self.rotary_dim
        if r is not None and not (isinstance(r, Integral) and not isinstance(r, bool) and 0 < r <= self.head_dim and r % 2 == 0):
            raise ValueError(f"rotary_dim must be an even whole number in 2..{self.head_dim}")
        check_rope_scaling(self.rope_scaling)

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_heads

    @property
    def rotary_width(self) -> int:
        return self.head_dim if self.rotary_dim is None else self.rotary_dim

    def check_tensor_parallel(self, size: int) -> None:
        for name in ("n_heads", "n_kv_heads", "ffn_dim"):
            n = getattr(self, name)
            if n % size:
                raise ValueError(f"{name} ({n}) must be divisible by the tensor-parallel size ({size})")

    def to_dict(self) -> dict:
        d = asdict(self)
        for name, default in (("rope_layout", "half"), ("rotary_dim", None), ("rope_scaling", None)):
            if d[name] == default:
                del d[name]
        return d
