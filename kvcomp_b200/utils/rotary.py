"""Frequencies of rotary embeddings, for ops.rotary and ops.rotary_paged_store: fp64 angles per position of each pair of channels, with the usual
ways of stretching them for contexts beyond the trained one, and the factor that goes with cos and sin."""
import math

import torch


# What a configuration's dict may hold; the last three say nothing that is needed here: how many channels are rotated is an argument, "finetuned" is a remark.
FIELDS = frozenset("factor original_max_position_embeddings max_position_embeddings attention_factor beta_fast beta_slow mscale mscale_all_dim truncate low_freq_factor "
                   "high_freq_factor short_factor long_factor rope_theta rope_type type partial_rotary_factor finetuned".split())


def frequencies(rotated, base=None, scaling=None, length=None, device=None, original_max_position_embeddings=None, max_position_embeddings=None):
    """(float64[rotated / 2], factor) of `rotated` channels: pair i turns by base^(-2i / rotated) per position.  base: 10000, or what scaling says.

    scaling: None, or a model configuration's dict with "rope_type" (or "type") and, with s = "factor" and L = "original_max_position_embeddings":
      linear    every angle divided by s
      ntk       the base raised to base * s^(r / (r - 2)): the slowest pair is stretched by s, the fastest not at all
      dynamic   the same with s (length / L) - (s - 1) in place of s for contexts `length` beyond L
      yarn      pairs that turn more than "beta_fast" (32) times in L positions stay, those that turn less than "beta_slow" (1) times are divided by s, a
                linear ramp over the pairs between, whose ends are rounded to whole pairs unless "truncate" is false; factor "attention_factor", or with both "mscale" and
                "mscale_all_dim" (0.1 mscale ln s + 1) / (0.1 mscale_all_dim ln s + 1), or 0.1 ln s + 1.  (A model that also multiplies its scores with the square of such a
                term does so in the attention's scaling.)
      llama3    the same idea by wavelengths: up to L / "high_freq_factor" stays, from L / "low_freq_factor" on divided by s, between them smoothed
      longrope  every angle divided by its own "short_factor", or "long_factor" once `length` is beyond L; factor "attention_factor", or with
                m = "max_position_embeddings" over L (or s) above 1 sqrt(1 + ln m / ln L)
    "rope_theta" is the base.  A dict with a field that is not known is refused: it would turn keys otherwise than the model does.
    length: the context's length, for the two that depend on it.
    original_max_position_embeddings, max_position_embeddings: for configurations that hold them beside the dict; without the first the second is L."""
    r = int(rotated)
    if r < 0 or r % 2:
        raise ValueError("the number of rotated channels must be even, got %d" % rotated)
    scaling = dict(scaling or {})
    unknown = sorted(str(key) for key, value in scaling.items() if key not in FIELDS and value is not None)
    if unknown:
        raise ValueError("scaling: %s not understood" % ", ".join(unknown))
    theta = scaling.get("rope_theta")
    if base is None:
        base = 10000.0 if theta is None else theta
    elif theta is not None and float(theta) != float(base):
        raise ValueError("base %r, but scaling says rope_theta %r" % (base, theta))
    base = float(base)
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    longest = scaling.get("max_position_embeddings") or max_position_embeddings
    s, trained = float(scaling.get("factor") or 1.0), scaling.get("original_max_position_embeddings") or original_max_position_embeddings or longest
    if kind in ("dynamic", "yarn", "llama3", "longrope") and not trained:
        raise ValueError("%s needs original_max_position_embeddings" % kind)
    i = torch.arange(0, r, 2, dtype=torch.float64)
    if kind == "ntk" or (kind == "dynamic" and length is not None and length > trained):
        grow = s if kind == "ntk" else s * length / trained - (s - 1.0)
        if r > 2:
            base = base * grow ** (r / (r - 2.0))
    f, factor = base ** (-i / max(r, 1)), 1.0
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        def pair(turns):                                             # the pair (a real number) that turns so often in the trained context
            return r * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = pair(scaling.get("beta_fast") or 32.0), pair(scaling.get("beta_slow") or 1.0)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, r - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f / s * ramp + f * (1.0 - ramp)

        def grown(mscale):
            return 0.1 * mscale * math.log(s) + 1.0 if s > 1.0 else 1.0
        factor, mscale, all_dim = (scaling.get(key) for key in ("attention_factor", "mscale", "mscale_all_dim"))
        if factor is not None:
            factor = float(factor)
        elif mscale and all_dim:
            factor = grown(float(mscale)) / grown(float(all_dim))
        elif all_dim or (mscale and float(mscale) != 1.0):           # (models differ in what one without the other means)
            raise ValueError("yarn: mscale and mscale_all_dim go together")
        else:
            factor = grown(1.0)
    elif kind == "llama3":
        slow, fast = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        turns = trained * f / (2.0 * math.pi)                        # in the trained context
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f / s * (1.0 - keep) + f * keep
    elif kind == "longrope":
        parts = scaling["long_factor" if length is not None and length > trained else "short_factor"]
        if len(parts) != r // 2:
            raise ValueError("longrope: %d factors for %d pairs" % (len(parts), r // 2))
        f = f / torch.tensor(parts, dtype=torch.float64)
        factor = scaling.get("attention_factor")
        if factor is None and not (longest or scaling.get("factor")):
            raise ValueError("longrope needs attention_factor, factor or max_position_embeddings")
        m = longest / trained if scaling.get("max_position_embeddings") or (longest and longest != trained) else s
        factor = (math.sqrt(1.0 + math.log(m) / math.log(trained)) if m > 1.0 else 1.0) if factor is None else float(factor)
    elif kind not in ("default", "ntk", "dynamic"):
        raise ValueError("unknown scaling %r" % (kind,))
    return f.to(device), factor
