"""``quantization_config`` of config.json: matrices in 8-bit floating point.

The form is the one that published checkpoints of the Qwen3 family have: ``quant_method`` "fp8", ``fmt`` "e4m3" (or absent),
``weight_block_size`` [128, 128], ``activation_scheme`` "dynamic" (activations are quantised as they come, a scale for every row and 128
columns).  Beside each such matrix the checkpoint has the scales of its blocks under the matrix's name and ``_scale_inv`` (the value of an
entry is the entry times its block's number).  It works for every architecture: the matrices of the part kinds ``KINDS`` are
expected in 8 bits, but for those of the modules in ``modules_to_not_convert``; embedding, head, norms, routers and all other kinds stay as
they are.  Anything else in the object is refused, never ignored.
"""
from __future__ import annotations

import dataclasses
import re
from typing import Any, Mapping

from .specs import ConfigError, ModelSpec, PartSpec

BLOCK = 128
# kind -> the names (of the part's ``names``) that are its matrices
KINDS = {"gqa_attention": ("q", "k", "v", "o", "gate"), "swiglu": ("gate", "up", "down"), "routed_experts": ("gate", "up", "down")}
_KNOWN = {"quant_method", "fmt", "weight_block_size", "activation_scheme", "modules_to_not_convert", "scale_fmt"}


def _check(q: Mapping[str, Any]) -> tuple:
    where = "config.json: quantization_config"
    if not isinstance(q, Mapping):
        raise ConfigError(f"{where} must be an object")
    unknown = sorted(set(q) - _KNOWN)
    if unknown:
        raise ConfigError(f"{where}: {', '.join(unknown)} not supported")
    if q.get("quant_method") != "fp8" or q.get("fmt", "e4m3") not in (None, "e4m3"):
        raise ConfigError(f"{where}: quant_method {q.get('quant_method')!r}, fmt {q.get('fmt')!r} is not supported (fp8, e4m3)")
    if list(q.get("weight_block_size") or ()) != [BLOCK, BLOCK]:
        raise ConfigError(f"{where}: weight_block_size {q.get('weight_block_size')!r} is not supported ([{BLOCK}, {BLOCK}])")
    if q.get("activation_scheme", "dynamic") != "dynamic":
        raise ConfigError(f"{where}: activation_scheme {q.get('activation_scheme')!r} is not supported ('dynamic')")
    if q.get("scale_fmt") not in (None, "float32"):
        raise ConfigError(f"{where}: scale_fmt {q.get('scale_fmt')!r} is not supported")
    left_out = q.get("modules_to_not_convert") or ()
    if not isinstance(left_out, (list, tuple)) or any(not isinstance(m, str) for m in left_out):
        raise ConfigError(f"{where}: modules_to_not_convert must be a list of names")
    return tuple(left_out)


def _module(name: str) -> str:
    return name[:-len(".weight")] if name.endswith(".weight") else name


def _one_expert(left_out: str, module: str) -> bool:
    """Whether ``left_out`` names ``module``, or what it is in, with a number in the place for an expert's."""
    if "{}" not in module:
        return False
    pattern = re.escape(module).replace(re.escape("{}"), "[0-9]+").split(re.escape("."))
    given = left_out.split(".")
    numbered = next(i for i, p in enumerate(pattern) if "[0-9]+" in p)
    return numbered < len(given) <= len(pattern) and all(re.fullmatch(p, g) for p, g in zip(pattern, given))


def _converted(part: PartSpec, prefix: str, left_out: tuple) -> PartSpec:
    if part is None:
        return part
    params = part.as_dict()
    if isinstance(params.get("shared"), PartSpec):
        params["shared"] = _converted(params["shared"], prefix, left_out)
    if part.kind in KINDS:
        names = dict(part["names"])
        # (a name with a place for an expert's number stands for all of them)
        modules = [_module(prefix + names[k]) for k in KINDS[part.kind] if k in names]
        one = [n for n in left_out if any(_one_expert(n, m) for m in modules)]
        if one:
            raise ConfigError(f"config.json: modules_to_not_convert leaves out {', '.join(one)} but not all matrices of that {part.kind}")
        out = [m for m in modules if any(m == n or m.startswith(n + ".") for n in left_out)]
        if out and len(out) < len(modules):
            raise ConfigError(f"config.json: modules_to_not_convert leaves out {', '.join(out)} but not all matrices of that {part.kind}")
        if not out:
            params["eight_bit"] = True
    return PartSpec.make(part.kind, **params)


def with_eight_bit(spec: ModelSpec, config: Mapping[str, Any]) -> ModelSpec:
    """``spec`` with its parts' matrices in 8 bits where ``config`` asks for it."""
    q = config.get("quantization_config")
    if q is None:
        return spec
    left_out = _check(q)
    layers = tuple(dataclasses.replace(layer, mixer=_converted(layer.mixer, layer.prefix, left_out),
                                       feed_forward=_converted(layer.feed_forward, layer.prefix, left_out)) for layer in spec.layers)
    if layers == spec.layers:
        raise ConfigError("config.json: quantization_config, but no matrix of this model is converted (kinds that are: "
                          + ", ".join(sorted(KINDS)) + ")")
    return dataclasses.replace(spec, layers=layers)
