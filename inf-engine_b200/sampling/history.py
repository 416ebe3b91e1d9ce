"""Penalties over what a request has said, biases and masks of allowed tokens, applied to the logits on the device before a token is
chosen (``kernels.adjust_logits``), and the history that the penalties read, kept on the device by request slot
(``kernels.history_reset``, ``kernels.history_append``).

The reference has one penalty, over the last 256 generated tokens and flat (engine/sampling.py:90-134); that one stays where it is
(``SamplingConfig.repetition_penalty`` with ``repetition_scope="window"``) and needs the tokens on the host.  The others need a
token on the host only when a request enters a slot, so a step can be enqueued before the tokens of the step before have been read.
"""

from __future__ import annotations

import numpy as np
import torch

from .. import kernels


def allowed_words(allowed, vocab: int) -> np.ndarray:
    """A mask as the kernel reads it, int32 [ceil(vocab / 32)], bit t % 32 of word t / 32, from token ids or from one truth value
    a token of the vocabulary."""
    a = np.asarray(allowed if isinstance(allowed, np.ndarray) else list(allowed))
    bits = np.zeros(-(-vocab // 32) * 32, dtype=bool)
    if a.dtype == np.bool_:
        if a.shape != (vocab,):
            raise ValueError(f"a mask of allowed tokens has one truth value for each of {vocab} tokens, not {a.shape}")
        bits[:vocab] = a
    elif a.size:
        if a.ndim != 1 or a.dtype.kind not in "iu":
            raise ValueError("allowed tokens are ids (whole numbers) or one truth value for each token")
        if int(a.min()) < 0 or int(a.max()) >= vocab:
            raise ValueError(f"an allowed token is outside the vocabulary of {vocab}")
        bits[a] = True
    return np.packbits(bits, bitorder="little").view(np.int32)


class TokenHistory:
    """Counts and bits of every slot (``kernels.history_append`` says what they hold), and whose they are: those of the request that was
    written into the slot last, as far as its tokens were recorded (``current``)."""

    def __init__(self, rt, n_slots: int, vocab: int):
        self.rt = rt
        self.counts = torch.zeros((n_slots, vocab), dtype=torch.int32, device=rt.device)
        self.seen = torch.zeros((n_slots, -(-vocab // 32)), dtype=torch.int32, device=rt.device)
        self._holds: dict[int, tuple[object, int]] = {}      # slot -> (request, tokens it had generated when last recorded)

    def current(self, slot: int, request) -> bool:
        """Whether the slot holds all that ``request`` has said."""
        held = self._holds.get(slot)
        return held is not None and held[0] is request and held[1] == len(request.generated)

    def forget(self, slot: int) -> None:
        """The slot has got a request, perhaps the one that it had before: nothing is known of what it holds."""
        self._holds.pop(slot, None)

    def enter(self, entries: list[tuple[int, object]]) -> None:
        """Writes the histories of requests anew, from their prompts and generated tokens: ``entries`` are (slot, request)."""
        tokens, starts = [], [0]
        for _, r in entries:
            tokens += r.prompt_ids
            tokens += r.generated
            starts.append(len(tokens))
        n = len(entries)
        head = [s for s, _ in entries] + starts + [len(r.prompt_ids) for _, r in entries]
        dev = self.rt.staging.upload(np.asarray(head + tokens, dtype=np.int32))
        slots, starts, n_prompt = dev[:n], dev[n:2 * n + 1], dev[2 * n + 1:3 * n + 1]
        kernels.history_reset(self.counts, self.seen, slots)
        kernels.history_append(self.counts, self.seen, dev[3 * n + 1:], slots, starts, n_prompt)
        for slot, r in entries:
            self._holds[slot] = (r, len(r.generated))

    def record(self, ids: torch.Tensor, slots: torch.Tensor, entries: list[tuple[int, object]]) -> None:
        """The tokens just sampled (int32 on the device, one a row; ``slots`` the rows' slots, -1 where nothing is kept) go into
        the histories; ``entries`` are the (slot, request) of the rows that keep one, whose ``generated`` has not got the token yet."""
        kernels.history_append(self.counts, self.seen, ids, slots)
        for slot, r in entries:
            self._holds[slot] = (r, len(r.generated) + 1)


class Adjuster:
    """What a step's rows ask for beyond drawing from their logits.  ``rows`` are (request, sampling configuration, slot, allowed)
    with ``allowed`` a row of words (``allowed_words``) or None."""

    def __init__(self, rt, n_slots: int, vocab: int):
        self.rt, self.n_slots, self.vocab = rt, n_slots, vocab
        self.history: TokenHistory | None = None             # made when the first request asks for it: 4 bytes a slot and token

    def apply(self, logits: torch.Tensor, rows) -> tuple[torch.Tensor, list[tuple[int, object]]] | None:
        """Adjusts float32 ``logits`` in place.  Returns what ``TokenHistory.record`` takes once the tokens are there, None when no
        row keeps a history."""
        n = len(rows)
        for c in {id(c): c for _, c, _, _ in rows}.values():
            c.validate()
        keep = [(slot, r) for r, c, slot, _ in rows if c.keeps_history]
        if keep:
            if self.history is None:
                self.history = TokenHistory(self.rt, self.n_slots, self.vocab)
            stale = [(slot, r) for slot, r in keep if not self.history.current(slot, r)]
            if stale:
                self.history.enter(stale)
        slots = np.asarray([slot if c.keeps_history else -1 for _, c, slot, _ in rows], dtype=np.int32)
        penalties = np.asarray([[c.repetition_penalty if c.repetition_scope == "history" else 1.0, c.presence_penalty,
                                 c.frequency_penalty] for _, c, _, _ in rows], dtype=np.float32)
        biases = [sorted(c.logit_bias.items()) if c.logit_bias else [] for _, c, _, _ in rows]
        start = np.concatenate([[0], np.cumsum([len(b) for b in biases])]).astype(np.int32)
        ids = np.asarray([t for b in biases for t, _ in b], dtype=np.int32)
        values = np.asarray([v for b in biases for _, v in b], dtype=np.float32)
        masks = [allowed for _, _, _, allowed in rows if allowed is not None]
        mask_rows = np.full(n, -1, dtype=np.int32)
        mask_rows[[i for i, row in enumerate(rows) if row[3] is not None]] = np.arange(len(masks))
        parts = [slots, penalties.reshape(-1).view(np.int32), start, ids, values.view(np.int32), mask_rows, *masks]
        dev = self.rt.staging.upload(np.concatenate(parts))
        cut, at = [], 0
        for p in parts[:6]:
            cut.append(dev[at:at + p.size])
            at += p.size
        kw = {}
        if keep:
            kw.update(slots=cut[0], penalties=cut[1].view(torch.float32).view(n, 3), counts=self.history.counts, seen=self.history.seen)
        if ids.size:
            kw.update(bias_start=cut[2], bias_ids=cut[3], bias_values=cut[4].view(torch.float32))
        if masks:
            kw.update(mask_rows=cut[5], masks=dev[at:].view(len(masks), -1))
        if kw:
            kernels.adjust_logits(logits, logits, **kw)
        return (cut[0], keep) if keep else None
