"""Synthetic data generators for the benchmark configs.

There is no network access for datasets (synthetic data /
random-init weights); these generate ImageNet-shape, CIFAR-shape and
BERT-token batches deterministically per (seed, rank, step) so loss
curves are exactly reproducible across world sizes — the correctness
check of SURVEY.md §5 item 4.
"""

from __future__ import annotations

from typing import Iterator, Tuple

import torch


class SyntheticImages:
    """Yields (images, labels); shapes per config.

    ImageNet-shape: 3x224x224, 1000 classes (config #2/#3/#5);
    CIFAR-shape:    3x32x32, 10 classes (config #1).
    """

    def __init__(self, batch_size: int, image_size: int = 224,
                 num_classes: int = 1000, seed: int = 0, rank: int = 0,
                 dtype: torch.dtype = torch.float32,
                 device: str = "cpu", channels_last: bool = False,
                 pinned: bool = False, pool: int = 0):
        self.batch_size = batch_size
        self.image_size = image_size
        self.num_classes = num_classes
        self.dtype = dtype
        self.device = device
        self.channels_last = channels_last
        self.pinned = pinned
        # pool > 0: cycle a FIXED set of batches.  Endless fresh random
        # labels have ln(num_classes) as their optimum, so a decreasing
        # loss (memorization) needs a finite pool — the synthetic-data
        # analogue of the reference's "CIFAR example converges" check.
        self.pool = pool
        self._pool_batches = []
        self.gen = torch.Generator().manual_seed(seed * 100003 + rank)

    def batch(self) -> Tuple[torch.Tensor, torch.Tensor]:
        x = torch.randn(self.batch_size, 3, self.image_size, self.image_size,
                        generator=self.gen, dtype=torch.float32)
        y = torch.randint(0, self.num_classes, (self.batch_size,),
                          generator=self.gen)
        x = x.to(self.dtype)
        if self.channels_last:
            x = x.contiguous(memory_format=torch.channels_last)
        if self.pinned:
            x, y = x.pin_memory(), y.pin_memory()
        if self.device != "cpu":
            x = x.to(self.device, non_blocking=True)
            y = y.to(self.device, non_blocking=True)
        return x, y

    def __iter__(self) -> Iterator[Tuple[torch.Tensor, torch.Tensor]]:
        if self.pool > 0:
            i = 0
            while True:
                if len(self._pool_batches) < self.pool:
                    self._pool_batches.append(self.batch())
                yield self._pool_batches[i % self.pool]
                i += 1
        else:
            while True:
                yield self.batch()


class SyntheticBertBatches:
    """Yields (input_ids, mlm_labels, nsp_labels) for BERT pretraining.

    ``doc_len`` > 0 packs documents of about that length into the rows and
    yields (input_ids, mlm_labels, nsp_labels, cu_seqlens): the documents'
    borders in the tokens of all rows, and a label for each.  Their number is
    fixed (a graph can be captured): unused ones are empty, at the end, with
    the label -100.
    """

    def __init__(self, batch_size: int, seq_len: int = 128,
                 vocab_size: int = 30522, mask_frac: float = 0.15,
                 seed: int = 0, rank: int = 0, device: str = "cpu",
                 pinned: bool = False, pool: int = 0, doc_len: int = 0):
        self.doc_len = doc_len
        self.batch_size, self.seq_len = batch_size, seq_len
        self.vocab_size, self.mask_frac = vocab_size, mask_frac
        self.device, self.pinned = device, pinned
        self.pool = pool            # >0: cycle a fixed batch set (see
        self._pool_batches = []     # SyntheticImages — memorization)
        self.gen = torch.Generator().manual_seed(seed * 100003 + rank)

    def batch(self):
        ids = torch.randint(0, self.vocab_size,
                            (self.batch_size, self.seq_len), generator=self.gen)
        labels = ids.clone()
        mask = torch.rand(ids.shape, generator=self.gen) < self.mask_frac
        labels[~mask] = -100
        if self.doc_len > 0:
            cu = self._pack()
            nsp = torch.randint(0, 2, (cu.numel() - 1,), generator=self.gen)
            nsp[cu[1:] == cu[:-1]] = -100
            batch = (ids, labels, nsp, cu)
        else:
            nsp = torch.randint(0, 2, (self.batch_size,), generator=self.gen)
            batch = (ids, labels, nsp)
        if self.pinned:
            batch = tuple(t.pin_memory() for t in batch)
        if self.device != "cpu":
            batch = tuple(t.to(self.device, non_blocking=True) for t in batch)
        return batch

    def _pack(self) -> torch.Tensor:
        """Borders of documents of half to one and a half of doc_len, none
        across two rows: int32, of a fixed number."""
        low = max(1, self.doc_len // 2)
        slots = self.batch_size * (-(-self.seq_len // low))
        ends = []
        for row in range(self.batch_size):
            at, end = row * self.seq_len, (row + 1) * self.seq_len
            while at < end:
                n = int(torch.randint(low, self.doc_len + low + 1, (1,),
                                      generator=self.gen))
                at = min(at + n, end)
                ends.append(at)
        ends += [self.batch_size * self.seq_len] * (slots - len(ends))
        return torch.tensor([0, *ends], dtype=torch.int32)

    def __iter__(self):
        if self.pool > 0:
            i = 0
            while True:
                if len(self._pool_batches) < self.pool:
                    self._pool_batches.append(self.batch())
                yield self._pool_batches[i % self.pool]
                i += 1
        else:
            while True:
                yield self.batch()
