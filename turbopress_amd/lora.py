"""Low-rank adapters of many requests beside a shared projection
(csrc/tp_lora.hip): the packed weights stay one for all, and each row of a batch
adds the product of its own request's adapter.  Inference only.
"""

from __future__ import annotations

import functools
import json
import math
from collections.abc import Mapping, Sequence
from pathlib import Path

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd.hip_kernel import raw_stream as _raw_stream
from turbopress_amd.norm import DTYPE_CODES
from turbopress_amd.paged import _elsewhere, _workspace

__all__ = ["lora_add", "LoraAdapters", "MAX_RANK"]

MAX_RANK = 256
_FAR = 1 << 24  # elements that rows may lie apart without a copy


@functools.lru_cache(maxsize=1024)
def _needs(rows: int, k: int, n: int, rank: int, count: int) -> int:
    """Workspace bytes of a call."""
    return _lib.lib().tp_lora_workspace_bytes(rows, k, n, rank, count)


def _refuse(y, x, a, b, adapters, scales) -> None:
    """Raise for arguments that lora_add does not take."""
    if not y.is_cuda:
        raise RuntimeError("y must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    dt, dev = y.dtype, y.device

    def expect(ok, name, t, what):
        if not ok:
            raise ValueError(f"{name} must be {what}, got {t.dtype} {list(t.shape)} on {t.device}")

    expect(dt in (torch.float16, torch.bfloat16) and y.dim() >= 1 and y.shape[-1] >= 1, "y", y, "fp16 or bf16 [..., out]")
    expect(x.dtype == dt and x.device == dev and x.dim() == y.dim() and x.shape[:-1] == y.shape[:-1] and x.shape[-1] >= 1, "x", x,
           f"{dt} {[*y.shape[:-1], 'in']} on {dev}")
    expect(a.dtype == dt and a.device == dev and a.dim() == 3 and a.shape[2] == x.shape[-1] and 1 <= a.shape[1] <= MAX_RANK, "a", a,
           f"{dt} [adapters, 1 to {MAX_RANK} ranks, {x.shape[-1]}] on {dev}")
    expect(b.dtype == dt and b.device == dev and b.shape == (a.shape[0], y.shape[-1], a.shape[1]), "b", b,
           f"{dt} {[a.shape[0], y.shape[-1], a.shape[1]]} on {dev}")
    expect(adapters.dtype == torch.int32 and adapters.device == dev and adapters.shape == y.shape[:-1], "adapters", adapters,
           f"int32 {list(y.shape[:-1])} on {dev}")
    expect(scales.dtype == torch.float32 and scales.device == dev and scales.shape == a.shape[:1], "scales", scales,
           f"fp32 {list(a.shape[:1])} on {dev}")


def _flat(t: Tensor, width: int) -> tuple:
    """(tensor, elements from a row to the next) of [..., width] as rows."""
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1) and t.stride(0) <= _FAR:
        return t, t.stride(0)
    return (t if t.is_contiguous() else t.contiguous()), width


def _weights(w: Tensor) -> Tensor:
    return w if (w.stride(2) == 1 or w.shape[2] == 1) and w.stride(1) <= _FAR else w.contiguous()


def lora_add(y: Tensor, x: Tensor, a: Tensor, b: Tensor, adapters: Tensor, scales: Tensor | None = None) -> Tensor:
    """``y + scales[i] * (x @ a[i]^T) @ b[i]^T`` with i = adapters of the row: y
    [..., out], the shared projection's output of x [..., in] (fp16 or bf16, all
    of one type); a [adapters, rank, in] and b [adapters, out, rank], the stacked
    adapters (ranks up to 256; smaller ones are padded with zeros); adapters int32
    [...], one per row, of which one that does not exist (-1) leaves its row as it
    is; scales fp32 [adapters] (None: 1).  Returns a new tensor; both products are
    summed in fp32, and the result rounds once."""
    code, index = DTYPE_CODES.get(y.dtype, _lib.TP_F32), y.get_device()
    lead = y.shape[:-1]
    if code == _lib.TP_F32 or index < 0 or y.dim() < 1 or x.dtype is not y.dtype or x.get_device() != index or x.dim() != y.dim() \
            or x.shape[:-1] != lead or a.dtype is not y.dtype or a.get_device() != index or a.dim() != 3 \
            or a.shape[2] != x.shape[-1] or not 1 <= a.shape[1] <= MAX_RANK or b.dtype is not y.dtype or b.get_device() != index \
            or b.shape != (a.shape[0], y.shape[-1], a.shape[1]) or adapters.dtype is not torch.int32 \
            or adapters.get_device() != index or adapters.shape != lead or x.shape[-1] < 1 or y.shape[-1] < 1 \
            or (scales is not None and (scales.dtype is not torch.float32 or scales.get_device() != index
                                        or scales.shape != a.shape[:1])):
        _refuse(y, x, a, b, adapters, scales)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return lora_add(y, x, a, b, adapters, scales)
    k, n = x.shape[-1], y.shape[-1]
    count, rank, _ = a.shape
    out = torch.empty_like(y, memory_format=torch.contiguous_format)
    rows = out.numel() // n
    (x, ldx), (y, ldy), a, b = _flat(x, k), _flat(y, n), _weights(a), _weights(b)
    if not adapters.is_contiguous():
        adapters = adapters.contiguous()
    if scales is not None and not scales.is_contiguous():
        scales = scales.contiguous()
    stream = _raw_stream(index)
    need = _needs(rows, k, n, rank, count)
    ws, _, _held = _workspace(index, stream, max(need, 16), 0)
    a_adapter, a_row, _ = a.stride()
    b_adapter, b_row, _ = b.stride()
    st = _lib.lib().tp_lora_add(code, rows, k, n, rank, count, x.data_ptr(), ldx, a.data_ptr(), a_adapter, a_row, b.data_ptr(), b_adapter,
                         b_row, adapters.data_ptr(), 0 if scales is None else scales.data_ptr(), y.data_ptr(), ldy,
                         out.data_ptr(), ws, need, stream)
    if st:
        _lib.check(st, "lora_add")
    return out


class LoraAdapters:
    """Adapters of one model, stacked by the projections that they change.

    adapters: of each, {module name: (a [rank, in], b [out, rank])}; scales: of
    each, what its products are multiplied by.  Adapters may have ranks and
    modules of their own: what one has not is zeros beside the others'."""

    def __init__(self, adapters: Sequence[Mapping], scales: Sequence[float], dtype: torch.dtype, device="cuda") -> None:
        if not adapters or len(adapters) != len(scales):
            raise ValueError(f"{len(adapters)} adapters and {len(scales)} scales: as many are needed, one at least")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be fp16 or bf16, got {dtype}")
        self.count = len(adapters)
        self.scales = torch.tensor([float(s) for s in scales], dtype=torch.float32, device=device)
        self.stacks: dict = {}
        for name in dict.fromkeys(n for one in adapters for n in one):
            pairs = [one.get(name) for one in adapters]
            for pair in pairs:
                if pair is not None and (pair[0].dim() != 2 or pair[1].dim() != 2 or pair[0].shape[0] != pair[1].shape[1]
                                         or not 1 <= pair[0].shape[0] <= MAX_RANK):
                    raise ValueError(f"{name}: a must be [rank, in] and b [out, rank] with 1 to {MAX_RANK} ranks, got "
                                     f"{list(pair[0].shape)} and {list(pair[1].shape)}")
            have = [pair for pair in pairs if pair is not None]
            sizes = {(pair[0].shape[1], pair[1].shape[0]) for pair in have}
            if len(sizes) != 1:
                raise ValueError(f"{name}: adapters of different (in, out): {sorted(sizes)}")
            (k, n), = sizes
            rank = max(pair[0].shape[0] for pair in have)
            a = torch.zeros(self.count, rank, k, dtype=dtype)
            b = torch.zeros(self.count, n, rank, dtype=dtype)
            for i, pair in enumerate(pairs):
                if pair is not None:
                    a[i, :pair[0].shape[0]] = pair[0]
                    b[i, :, :pair[0].shape[0]] = pair[1]
            self.stacks[name] = (a.to(device), b.to(device))

    @classmethod
    def load(cls, directories: Sequence, dtype: torch.dtype, device="cuda") -> "LoraAdapters":
        """From directories of ``adapter_config.json`` (r, lora_alpha, use_rslora)
        and ``adapter_model.safetensors`` (``base_model.model.<module>.lora_A.weight``
        [rank, in] and ``.lora_B.weight`` [out, rank]).  What such an adapter may have
        beside its two products is refused, and so are adapters of other weights than
        the model's own (``init_lora_weights`` of pissa, olora, corda, loftq)."""
        from safetensors.torch import load_file
        adapters, scales = [], []
        for directory in map(Path, directories):
            cfg = json.loads((directory / "adapter_config.json").read_text())
            for key in ("use_dora", "rank_pattern", "alpha_pattern", "modules_to_save", "fan_in_fan_out", "lora_bias", "use_qalora",
                        "layer_replication", "alora_invocation_tokens", "trainable_token_indices", "target_parameters"):
                if cfg.get(key):
                    raise ValueError(f"{directory}: {key} = {cfg[key]!r} is not supported")
            if cfg.get("init_lora_weights", True) not in (True, False, None, "gaussian", "eva", "orthogonal"):
                # (such a beginning took the two products out of the model's own weights)
                raise ValueError(f"{directory}: init_lora_weights = {cfg['init_lora_weights']!r}: not an adapter of the model's own weights")
            if cfg.get("bias", "none") != "none" or cfg.get("peft_type", "LORA") != "LORA":
                raise ValueError(f"{directory}: not a low-rank adapter without biases")
            parts: dict = {}
            for key, t in load_file(directory / "adapter_model.safetensors").items():
                name, _, kind = key.removeprefix("base_model.model.").rpartition(".lora_")
                if kind not in ("A.weight", "B.weight") or not name:
                    raise ValueError(f"{directory}: {key} is not supported")
                parts.setdefault(name, {})[kind[0]] = t
            if any(len(pair) != 2 for pair in parts.values()) or not parts:
                raise ValueError(f"{directory}: a module needs lora_A and lora_B")
            adapters.append({name: (pair["A"], pair["B"]) for name, pair in parts.items()})
            scales.append(cfg["lora_alpha"] / (math.sqrt(cfg["r"]) if cfg.get("use_rslora") else cfg["r"]))
        return cls(adapters, scales, dtype, device)

    def check(self, shapes: Mapping, dtype: torch.dtype, device) -> None:
        """Raise where these are not adapters of modules {name: (out, in)}."""
        for name, (a, b) in self.stacks.items():
            if name not in shapes:
                raise ValueError(f"an adapter changes {name}, which is no projection of the model")
            if (b.shape[1], a.shape[2]) != tuple(shapes[name]):
                raise ValueError(f"{name} is {list(shapes[name])}, its adapters {[b.shape[1], a.shape[2]]}")
            if a.dtype != dtype or a.device != device:
                raise ValueError(f"adapters are {a.dtype} on {a.device}, the model {dtype} on {device}")

    def add(self, name: str, y: Tensor, x: Tensor, rows: Tensor) -> Tensor:
        """``lora_add`` of module `name`, rows: each row's adapter; y where none
        changes the module."""
        stack = self.stacks.get(name)
        return y if stack is None else lora_add(y, x, *stack, rows, self.scales)
