"""Beam search over a paged cache, on the device: selection, forking of the block tables and the copies of the open blocks, one
step after the other without a host synchronisation.

The reference's generation loop keeps beams on the host (mindformers/generation/text_generator.py); here a step is four
enqueued operators, and the host reads tokens when it wants them.  Beams share the full blocks of what they have in common,
so that K beams of a prompt hold its blocks once.
"""
import numpy as np
import torch

from .. import ops


class BeamSearch:
    """B groups of K beams over ``caches`` (tensors [num_blocks, block_size, ...]: the key and value caches, and the scale caches, of
    all layers).  ``window`` / ``sinks``: those of the layers' attention, so that blocks behind the window are given back;
    ``held`` (bool or uint8 [num_blocks] on the device): blocks that belong to other sequences.

        search = BeamSearch(caches, beams=4, eos_token_id=2)
        tokens = search.start(block_tables, context_lens, logits)      # of the prompts, which the cache holds
        while ...:
            logits = model(tokens, search.context_lens, search.block_tables, search.slot_mapping)
            tokens = search.step(logits)
        best = search.hypotheses()

    ``context_lens`` counts the token that the model's step is about to write, as the decode operators want it."""

    def __init__(self, caches, beams, eos_token_id=-1, window=None, sinks=0, held=None):
        if not 1 <= beams <= 32:
            raise ValueError(f"1 to 32 beams, got {beams}")
        ops.check_window(window, sinks)
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("caches must not be empty")
        self.num_blocks, self.block_size = self.caches[0].shape[:2]
        self.beams, self.eos_token_id = beams, -1 if eos_token_id is None else int(eos_token_id)
        self.window, self.sinks, self.held = window, sinks, held
        self.block_tables = self.context_lens = self.slot_mapping = self.scores = None

    def start(self, block_tables, context_lens, logits):
        """First tokens of every prompt's beams: ``block_tables`` [B, M] and ``context_lens`` [B] of the prompts, host arrays or int32
        device tensors, whose tokens the cache holds; ``logits`` [B, vocab] of their last tokens.  M bounds a beam's length."""
        dev, k = self.caches[0].device, self.beams
        tables, lens = (torch.as_tensor(np.ascontiguousarray(a) if isinstance(a, np.ndarray) else a, dtype=torch.int32, device=dev)
                        for a in (block_tables, context_lens))
        b = lens.numel()
        if logits.dim() != 2 or logits.shape[0] != b or tables.dim() != 2 or tables.shape[0] != b:
            raise ValueError(f"block_tables, context_lens and logits must hold a row for each of {b} prompts")
        self.groups = b
        self.block_tables = tables.repeat_interleave(k, dim=0)
        # every beam starts as its prompt's row; only the first is in the search
        self.context_lens = lens.reshape(-1).repeat_interleave(k)
        self.scores = torch.full((b, k), -torch.inf, dtype=torch.float32, device=dev)
        self.scores[:, 0] = 0.0
        self._missing = torch.zeros(1, dtype=torch.int32, device=dev)
        self._out = None                                      # rows of groups that were released
        self._steps = []
        # All rows go on from it, those too whose candidate is of a beam that is out (a vocabulary of no more than K words has no K others): the
        # rows of a prompt share its open block, so that it has to have one lowest child.
        first = torch.arange(0, b * k, k, dtype=torch.int32, device=dev).repeat_interleave(k)
        return self._step(logits.repeat_interleave(k, dim=0), first)

    def step(self, logits):
        """From the logits [B * K, vocab] of the beams' last tokens to the next tokens, int32 [B * K]; block_tables, context_lens and
        slot_mapping then describe the model's step that reads them."""
        self._started()
        return self._step(logits)

    def _step(self, logits, parents=None):
        sel = ops.beam_search_select(logits, self.scores, eos_token_id=self.eos_token_id)
        parents = sel.next_rows.view(-1) if parents is None else parents
        if self._out is not None:
            parents = torch.where(self._out, -1, parents)
        fork = ops.fork_blocks(self.block_tables, self.context_lens, self.num_blocks, self.block_size, parents=parents, new_tokens=1,
                               window=self.window, sinks=self.sinks, held=self.held)
        ops.copy_blocks(self.caches, fork.copies)
        self._missing += fork.missing
        self.block_tables, self.context_lens, self.slot_mapping = fork.block_tables, fork.context_lens, fork.slot_mapping
        self.scores = sel.next_scores
        self._steps.append(sel)
        return sel.next_tokens.view(-1)

    def _started(self):
        if self.scores is None:
            raise RuntimeError("call start() first")

    def release(self, groups):
        """Takes groups out of the search: their rows are empty from the next step on, and their blocks free."""
        self._started()
        rows = torch.zeros(self.groups, dtype=torch.bool, device=self.scores.device)
        rows[torch.as_tensor(groups, device=rows.device)] = True
        self.scores = torch.where(rows[:, None], -torch.inf, self.scores)
        rows = rows.repeat_interleave(self.beams)
        self._out = rows if self._out is None else self._out | rows

    def compact(self):
        """Closes up the cache's blocks; returns the number in use, int32 [1] on the device: blocks from there on that are not held by
        others are free."""
        self._started()
        self.block_tables, copies, live = ops.compact_blocks(self.block_tables, self.num_blocks, self.block_size, held=self.held)
        ops.copy_blocks(self.caches, copies)
        if self.slot_mapping is not None:                     # the slots of the step to come, in the moved blocks
            pos = (self.context_lens - 1).clamp(min=0).long()
            page = torch.gather(self.block_tables, 1, (pos // self.block_size)[:, None])[:, 0]
            slot = page * self.block_size + (pos % self.block_size).int()
            self.slot_mapping = torch.where(self.slot_mapping < 0, self.slot_mapping, slot)
        return live

    def hypotheses(self, length_penalty=1.0):
        """The finished and the running continuations of every group, on the host: a list of (score / length ** length_penalty, tokens) per
        group, best first.  A continuation is finished where the end token is among a step's K best candidates; its end token
        counts.  Raises if a step found no block for a beam."""
        self._started()
        if int(self._missing):
            raise RuntimeError(f"the cache of {self.num_blocks} blocks was short of {int(self._missing)} blocks for the beams")
        host = [[t.cpu().numpy() for t in sel] for sel in self._steps]
        found = [[] for _ in range(self.groups)]

        def tokens(step, row, last):
            got = [int(last)]
            for s in range(step, -1, -1):                     # the row's tokens up to and including step `step`
                got.append(int(host[s][5].reshape(-1)[row]))
                row = int(host[s][4].reshape(-1)[row])
            return got[::-1]

        for t, (score, beam, token, *_) in enumerate(host):
            if self.eos_token_id < 0:
                break
            for g, r in zip(*np.nonzero((token == self.eos_token_id)[:, :self.beams])):
                if np.isfinite(score[g, r]):
                    row = g * self.beams + int(beam[g, r])
                    found[g].append((float(score[g, r]) / (t + 1) ** length_penalty, tokens(t - 1, row, self.eos_token_id)))
        n, scores = len(host), self.scores.cpu().numpy()
        for g in range(self.groups):
            for i in range(self.beams):
                if np.isfinite(scores[g, i]):
                    row = g * self.beams + i
                    found[g].append((float(scores[g, i]) / n ** length_penalty, tokens(n - 2, int(host[-1][4].reshape(-1)[row]),
                                                                                       host[-1][5].reshape(-1)[row])))
        return [sorted(f, key=lambda x: -x[0]) for f in found]
