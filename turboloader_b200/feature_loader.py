"""GPU-resident loader of cached features: the ``CudaResidentLoader`` of what an image encoder gives.

A frozen encoder runs once over the images; its token features are written into a microscaled cache in HBM
(``fill`` or ``write``), and every epoch is served from there in shuffled order.  Iteration, ``set_epoch``,
``state_dict``, ``return_indices`` and the permutation (``np.random.default_rng(seed + epoch).permutation(n)``)
follow ``CudaResidentLoader`` (turboloader/cuda_loader.py:385-535); the cache has no counterpart in the reference.
"""
from __future__ import annotations

import numpy as np

from . import ops
from .mx import MxCache, _dtype_id, _raw_stream

__all__ = ["CudaFeatureLoader"]


class CudaFeatureLoader:
    """``num_samples`` samples of ``tokens`` x ``dim`` features, served in batches.

    ``output``: ``"values"`` gives tensors of ``dtype`` (n, tokens, dim), ``"mx"`` the rows as they are held
    (``MxTensor``), for ``mx_linear``.  With ``ragged`` the samples have lengths of their own; a batch is then
    padded with zeros and followed by its lengths (n,).  ``labels`` and ``return_indices`` append theirs.  Every
    batch is made on the consumer's current stream and has memory of its own."""

    def __init__(self, num_samples, tokens, dim, batch_size=64, *, format="nvfp4", scale=1.0, ragged=False, dtype=None,
                 output="values", drop_last=True, shuffle=False, seed=42, return_indices=False, labels=None, device=None):
        import torch

        if not ops.cuda_available():
            raise RuntimeError("CudaFeatureLoader needs an sm_100 CUDA device and the built C-ABI library.")
        if int(num_samples) < 1 or int(batch_size) < 1:
            raise ValueError("num_samples and batch_size must be positive")
        if output not in ("values", "mx"):
            raise ValueError("output must be 'values' or 'mx'")
        self._torch = torch
        self.cache = MxCache.empty(num_samples, tokens, dim, format, ragged=ragged, scale=scale, device=device)
        self._device = self.cache.device
        self._n, self.batch_size = int(num_samples), int(batch_size)
        self.dtype = torch.bfloat16 if dtype is None else dtype
        _dtype_id(self.dtype, "dtype")
        self.output = output
        self.drop_last, self.shuffle, self.seed = bool(drop_last), bool(shuffle), int(seed)
        self.return_indices = bool(return_indices)
        self._labels = None if labels is None else torch.as_tensor(np.asarray(labels), dtype=torch.int64).to(self._device)
        if self._labels is not None and tuple(self._labels.shape) != (self._n,):
            raise ValueError("labels must hold one value per sample")
        self._epoch = 0
        self._resume_batches = 0
        self._batches_served = 0

    # ---- filling -----------------------------------------------------------------------------
    def write(self, indices, features, lengths=None):
        """Stores ``features[i]`` (tokens, dim) as sample ``indices[i]``; see ``MxCache.write``.  Host indices are
        checked and uploaded; a CUDA tensor is used in place."""
        torch = self._torch
        if not isinstance(indices, torch.Tensor) or not indices.is_cuda:
            host = np.asarray(indices, dtype=np.int64).reshape(-1)
            if host.size and (host.min() < 0 or host.max() >= self._n):
                raise IndexError(f"sample index outside [0, {self._n})")
            indices = torch.from_numpy(host).to(self._device)
        self.cache.write(indices, features, lengths=lengths)

    def fill(self, batches, encoder):
        """Runs ``encoder`` over an image loader that was made with ``return_indices=True`` (``CudaResidentLoader``)
        and stores what it returns: features (n, tokens, dim), or ``(features, lengths)``.  The images reach the
        encoder as CUDA tensors.  Returns the number of samples written.  A loader that leaves out its last, smaller
        batch is refused: those samples would read as zeros."""
        torch = self._torch
        if getattr(batches, "return_indices", True) is False:  # its second item would be labels
            raise ValueError("fill needs batches with indices (return_indices=True)")
        samples = getattr(batches, "_n", None)
        if getattr(batches, "drop_last", False) and samples is not None and samples % batches.batch_size:
            raise ValueError(f"the loader drops the last {samples % batches.batch_size} of its {samples} samples: make it with drop_last=False")
        written = 0
        with torch.no_grad():
            for items in batches:
                if not isinstance(items, tuple) or len(items) < 2:
                    raise ValueError("fill needs batches with indices (return_indices=True)")
                images = items[0] if isinstance(items[0], torch.Tensor) else torch.as_tensor(items[0], device=self._device)
                found = encoder(images)
                features, lengths = found if isinstance(found, tuple) else (found, None)
                self.write(items[-1], features, lengths)
                written += int(features.shape[0])
        return written

    # ---- the surface of the resident loaders ---------------------------------------------------
    def set_epoch(self, epoch):
        self._epoch = int(epoch)

    def __len__(self):
        return self._n // self.batch_size if self.drop_last else -(-self._n // self.batch_size)

    def state_dict(self):
        return {"version": 1, "epoch": int(self._epoch), "batches_served": int(self._batches_served)}

    def load_state_dict(self, state):
        if int(state.get("version", 0)) != 1:
            raise ValueError("unsupported state_dict version")
        self._epoch = int(state["epoch"])
        self._resume_batches = int(state["batches_served"])

    def device_status(self) -> int:
        """Status bits the kernels OR-ed so far (synchronises); 0 when every index and length was valid."""
        return self.cache.device_status()

    def epoch_order(self, epoch=None) -> np.ndarray:
        e = self._epoch if epoch is None else int(epoch)
        if self.shuffle:
            return np.random.default_rng(self.seed + e).permutation(self._n).astype(np.int64)
        return np.arange(self._n, dtype=np.int64)

    def __iter__(self):
        torch = self._torch
        order = torch.from_numpy(self.epoch_order()).to(self._device)
        made_on = _raw_stream(self._device.index)
        start = self._resume_batches
        self._resume_batches = 0
        self._batches_served = start
        for b in range(start, len(self)):
            index = order[b * self.batch_size:(b + 1) * self.batch_size]
            if _raw_stream(self._device.index) != made_on:  # the consumer changed streams: the order outlives its reads there too
                order.record_stream(torch.cuda.current_stream(self._device))
            batch = self.cache.read_mx(index) if self.output == "mx" else self.cache.read(index, self.dtype)
            items = list(batch) if isinstance(batch, tuple) else [batch]
            if self._labels is not None:
                items.append(self._labels[index])
            if self.return_indices:
                items.append(index)
            self._batches_served += 1
            yield items[0] if len(items) == 1 else tuple(items)
        self._batches_served = 0
