"""Low-rank adapters of many requests beside projections that they share: the weights, and the cell around a linear one.

The reference's multi-adapter cells (mindformers/pet/tuners/slora_adapter.py) gather every request's pair of matrices into a batch of
their own; here the rows of a step are sorted by adapter once, and each adapter's matrices are read where they lie.
"""
import torch
from torch import nn

from .. import ops


class AdapterBank(nn.Module):
    """The adapters of one projection: ``n_adapters`` slots of rank up to ``rank`` (a multiple of 8, up to 128) beside a projection from
    ``in_features`` to ``widths`` columns, an int or the slices of a fused projection, each with matrices of its own.

        bank = AdapterBank(16, 4096, (4096, 1024, 1024), rank=32)
        bank.load(3, [a_q, None, a_v], [b_q, None, b_v], scale=alpha / r)       # a: [r, in], b: [out, r]; None: no adapter there
        rows = ops.adapter_rows(adapter_ids, 16)                                # once a step, for the banks of all projections
        y = bank(x, y, rows)                                                    # y + scale B (A x)

    Buffers: ``lora_a`` [n, slices, rank, in], ``lora_b`` [n, out, rank], ``ranks`` int32 [n] (0: an empty slot), ``scales`` fp32 [n]."""

    def __init__(self, n_adapters, in_features, widths, rank, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        widths = (int(widths),) if isinstance(widths, int) else tuple(int(w) for w in widths)
        if not (1 <= n_adapters <= 1024 and 1 <= len(widths) <= 8 and min(widths) > 0):
            raise ValueError(f"1 to 1024 adapters and 1 to 8 slices, got {n_adapters} and {widths}")
        if rank % 8 or not 0 < rank <= 128 or in_features % 8 or in_features <= 0:
            raise ValueError(f"rank ({rank}, up to 128) and in_features ({in_features}) must be multiples of 8")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("adapters are bfloat16 or float16")
        self.n_adapters, self.in_features, self.widths, self.rank = int(n_adapters), int(in_features), widths, int(rank)
        self.out_features, self.dtype = sum(widths), dtype
        self.register_buffer("lora_a", torch.zeros(n_adapters, len(widths), rank, in_features, dtype=dtype, device=device))
        self.register_buffer("lora_b", torch.zeros(n_adapters, self.out_features, rank, dtype=dtype, device=device))
        self.register_buffer("ranks", torch.zeros(n_adapters, dtype=torch.int32, device=device))
        self.register_buffer("scales", torch.zeros(n_adapters, dtype=torch.float32, device=device))

    def _slot(self, slot):
        if not 0 <= slot < self.n_adapters:
            raise ValueError(f"slot {slot} of {self.n_adapters}")

    @torch.no_grad()
    def load(self, slot, lora_a, lora_b, scale=1.0):
        """Puts an adapter into a slot: for every slice ``lora_a`` [r, in] and ``lora_b`` [width, r] (lists; one slice: the tensors), None
        and None where it has none.  On the current stream, behind the steps that it is ordered behind."""
        self._slot(slot)
        a, b = ([m] if isinstance(m, torch.Tensor) else list(m) for m in (lora_a, lora_b))
        if len(a) != len(self.widths) or len(b) != len(self.widths):
            raise ValueError(f"{len(self.widths)} slices, got {len(a)} and {len(b)} matrices")
        most = 0
        for ai, bi, n in zip(a, b, self.widths):
            if (ai is None) != (bi is None):
                raise ValueError("a slice has both matrices or neither")
            if ai is None:
                continue
            r = ai.shape[0]
            if not (ai.dim() == 2 and bi.dim() == 2 and 0 < r <= self.rank and ai.shape[1] == self.in_features and tuple(bi.shape) == (n, r)):
                raise ValueError(f"lora_a {tuple(ai.shape)} and lora_b {tuple(bi.shape)}: [r, {self.in_features}] and [{n}, r] with r up to {self.rank}")
            most = max(most, r)
        new_a, new_b, at = torch.zeros_like(self.lora_a[slot]), torch.zeros_like(self.lora_b[slot]), 0
        for i, (ai, bi, n) in enumerate(zip(a, b, self.widths)):
            if ai is not None:
                new_a[i, :ai.shape[0]].copy_(ai)
                new_b[at:at + n, :ai.shape[0]].copy_(bi)
            at += n
        self.lora_a[slot].copy_(new_a)                        # (only now: the matrices may be the slot's own)
        self.lora_b[slot].copy_(new_b)
        self.ranks[slot] = most
        self.scales[slot] = float(scale)
        return self

    @torch.no_grad()
    def unload(self, slot):
        """Empties a slot: rows that name it are their projection's."""
        self._slot(slot)
        self.ranks[slot] = 0
        return self

    def forward(self, x, base, rows, out=None):
        """base + scale B (A x) for the rows of each adapter (``ops.adapter_linear``); ``rows``: the step's ``ops.adapter_rows``."""
        return ops.adapter_linear(x, self.lora_a, self.lora_b, rows, base, widths=self.widths, ranks=self.ranks, scales=self.scales, out=out)

    construct = forward

    def _apply(self, fn, *args, **kw):
        dtype = fn(self.lora_a.new_empty(0)).dtype
        if dtype not in (torch.bfloat16, torch.float16):      # before anything is converted
            raise TypeError("adapters are bfloat16 or float16")
        scales = self.scales
        super()._apply(fn, *args, **kw)
        if self.scales.dtype != torch.float32:                # .half() and the like are for the matrices
            self.scales = scales.to(self.lora_a.device)
        self.dtype = dtype
        return self


class AdapterLinear(nn.Module):
    """A linear cell (float or quantised) with a bank of adapters beside it: ``forward(x, rows)`` is the cell's output plus each row's
    adapter, ``forward(x)`` the cell's alone.  Where x, and with it the float cells' output, is of another type than the bank (float32 rows
    beside 16-bit weights), the adapters' part is computed in the bank's and added in the output's."""

    def __init__(self, layer, bank):
        super().__init__()
        sizes = tuple(getattr(layer, n, getattr(layer, m, None)) for n, m in (("in_channels", "input_size"), ("out_channels", "output_size")))
        if sizes != (bank.in_features, bank.out_features):
            raise ValueError(f"the bank is for {bank.in_features} -> {bank.out_features}, the cell is {sizes[0]} -> {sizes[1]}")
        if getattr(layer, "activation_flag", False):
            raise NotImplementedError("adapters beside a cell with an activation of its own")
        self.layer, self.bank = layer, bank

    def forward(self, x, rows=None, **kw):
        y = self.layer(x, **kw)
        if rows is None:
            return y
        dtype = self.bank.dtype
        x = x if x.dtype == dtype else x.to(dtype)
        if y.dtype != dtype:
            return (y + self.bank(x, torch.zeros_like(y, dtype=dtype), rows)).to(y.dtype)  # (two 16-bit types: their sum is float32)
        return self.bank(x, y, rows, out=y)

    construct = forward
