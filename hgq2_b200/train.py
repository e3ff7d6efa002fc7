"""The QAT training step: flat parameter bucket, fused Adam, data-parallel gradient exchange.

What Keras' torch trainer does around the layers of the hot path (forward with ``training=True``,
task loss + ``sum(model.losses)``, backward, optimizer update, constraints) is restated here on one
flat fp32 bucket:

* every trainable variable of the model becomes a view into ``params``; its ``.grad`` is a view into
  ``grads``.  One memset clears the gradients, one NCCL all-reduce averages them over the ranks, one
  fused kernel (``hgq_adam_step``) applies Adam, the MonoL1 regularisers and the MinMax constraints.
* data parallelism shards the batch; the only other exchange is a MAX all-reduce of the per-column
  abs-max statistics that drive the WRAP integer-bit tracking, so that every rank keeps identical
  quantizer state (and therefore identical EBOPs).
"""

from __future__ import annotations

import ctypes
import math
import os

import numpy as np
import torch
import torch.distributed as dist

from . import _lib, kernels
from .backend import Layer, Variable, join_bookkeeping
from .constraints import Constant as ConstantConstraint
from .constraints import Max, Min, MinMax
from .quantizer.internal import fixed_point_quantizer as _fpq
from .regularizers import MonoL1


def _bounds(v: Variable) -> tuple[float, float]:
    """The clamp a variable's constraint is, as (lowest, highest) value."""
    c = v.constraint
    if c is None:
        return -math.inf, math.inf
    if isinstance(c, MinMax):
        return c.min_value, c.max_value
    if isinstance(c, Min):
        return c.min_value, math.inf
    if isinstance(c, Max):
        return -math.inf, c.max_value
    if isinstance(c, ConstantConstraint):
        return c.value, c.value
    raise NotImplementedError(f'constraint {type(c).__name__} on {v.path} cannot be fused')


def _l1(v: Variable) -> float:
    """The constant gradient a variable's regularizer adds."""
    r = v.regularizer
    if r is None:
        return 0.0
    if isinstance(r, MonoL1):
        return r.l1
    raise NotImplementedError(f'regularizer {type(r).__name__} on {v.path} cannot be fused')


class FlatState:
    """Packs the trainable variables of ``model`` into one fp32 buffer (plus a matching gradient buffer and the
    per-element constraint / regulariser tables the fused optimizer reads)."""

    def __init__(self, model: Layer):
        self.variables: list[Variable] = [v for v in model.trainable_variables]
        if not self.variables:
            raise ValueError('model has no trainable variables (is it built?)')
        dev = self.variables[0].value.device
        sizes = [v.value.numel() for v in self.variables]
        # 4-element alignment keeps every view 16-byte aligned for the vectorised kernels
        self.offsets, off = [], 0
        for n in sizes:
            self.offsets.append(off)
            off += (n + 3) // 4 * 4
        self.n = off
        # one concatenation instead of a copy per variable (padding pieces are slices of one small zero tensor)
        pad = torch.zeros(3, dtype=torch.float32, device=dev)
        pieces = []
        for v, n in zip(self.variables, sizes):
            pieces.append(v.value.detach().reshape(-1).to(torch.float32))
            if (-n) % 4:
                pieces.append(pad[:(-n) % 4])
        self.params = torch.cat(pieces)
        assert self.params.numel() == self.n
        self.grads = torch.zeros(self.n, dtype=torch.float32, device=dev)
        lo = torch.full((self.n,), -math.inf, dtype=torch.float32)
        hi = torch.full((self.n,), math.inf, dtype=torch.float32)
        l1 = torch.zeros(self.n, dtype=torch.float32)
        for v, o, n in zip(self.variables, self.offsets, sizes):
            v.value.data = self.params[o:o + n].view(v.value.shape)
            v.value.grad = self.grads[o:o + n].view(v.value.shape)
            lo[o:o + n], hi[o:o + n] = _bounds(v)
            l1[o:o + n] = _l1(v)
        self.lo, self.hi, self.l1 = lo.to(dev), hi.to(dev), l1.to(dev)

    def zero_grad(self) -> None:
        self.grads.zero_()

    def check_views(self) -> None:
        """Autograd must have accumulated into the bucket views, not replaced them."""
        base = self.grads.data_ptr()
        for v, o in zip(self.variables, self.offsets):
            g = v.value.grad
            if g is None or g.data_ptr() != base + 4 * o:
                raise RuntimeError(f'gradient of {v.path} left the flat bucket')

    def regularization_loss(self) -> torch.Tensor:
        return torch.dot(self.l1, self.params)


class FusedAdam:
    """Keras-flavoured Adam on a ``FlatState`` through the C-ABI kernel (regulariser and constraints included)."""

    def __init__(self, state: FlatState, learning_rate=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7):
        self.state = state
        self.lr, self.b1, self.b2, self.eps = learning_rate, beta_1, beta_2, epsilon
        dev = state.params.device
        self.m = torch.zeros_like(state.params)
        self.v = torch.zeros_like(state.params)
        self.step_count = torch.zeros((), dtype=torch.int64, device=dev)

    def step(self, grad_scale: float = 1.0) -> None:
        s = self.state
        _lib.require_cuda(s.params)
        with torch.cuda.device(s.params.device):
            st = _lib.lib().hgq_adam_step(
                s.params.data_ptr(), s.grads.data_ptr(), self.m.data_ptr(), self.v.data_ptr(), s.lo.data_ptr(),
                s.hi.data_ptr(), s.l1.data_ptr(), s.n, self.lr, self.b1, self.b2, self.eps, grad_scale,
                self.step_count.data_ptr(), _lib.stream_handle(),
            )
        _lib.check(st, 'hgq_adam_step')

    def step_peers(self, peers: 'PeerExchange') -> None:
        """The update from the MEAN of the ranks' gradient buckets, read over peer memory inside the optimizer kernel
        (``hgq_adam_step_peers``).  ``state.grads`` keeps this rank's local gradients."""
        from . import kernels

        s = self.state
        _lib.require_cuda(s.params)
        with torch.cuda.device(s.params.device):
            st = _lib.lib().hgq_adam_step_peers(
                s.params.data_ptr(), s.grads.data_ptr(), self.m.data_ptr(), self.v.data_ptr(), s.lo.data_ptr(),
                s.hi.data_ptr(), s.l1.data_ptr(), s.n, self.lr, self.b1, self.b2, self.eps, self.step_count.data_ptr(),
                peers.ptrs, peers.world, peers.rank, peers.max_polls, kernels.status_word(s.params.device).data_ptr(),
                _lib.stream_handle(),
            )
        _lib.check(st, 'hgq_adam_step_peers')


class FusedAdamW:
    """AdamW over a list of tensors in one launch (two with clipping), with its moments in 32 or in 8 bits.

    ``tensors``: a ``FlatState``, or a sequence of ``Variable`` s and / or tensors (contiguous, on one GPU, no two of them over
    the same memory).  A ``Variable``'s constraint and ``MonoL1`` regularizer are applied in the same pass.  bf16 and fp16
    tensors are updated through an fp32 copy that the optimizer keeps (``masters``); the tensor gets its rounded value.

    The rule is Keras' AdamW: ``w`` is first scaled by ``1 - learning_rate * weight_decay``, then takes Adam's step;
    ``global_clipnorm`` scales all gradients so that their common 2-norm is at most that (a norm that is infinite or NaN makes
    every weight with a gradient NaN, as in Keras).  ``weight_decay`` is one number, or one per tensor (0 for biases and bitwidths, say).

    ``state_bits=8`` keeps the moments as e4m3 codes with an fp32 scale per 256 elements of a tensor: ``m`` (times ``m_scale``)
    and ``r`` (times ``r_scale``), the root of the second moment -- 2 bytes per weight instead of 8.  ``state_bits=32`` keeps
    fp32 ``m`` and ``v``.  The state arrays are flat; tensor ``i`` starts at ``offsets[i]``, a multiple of 256.

    The tensors' addresses are taken at construction: build the optimizer after whatever lays the parameters out
    (``FlatState``), and after assigning new values to bf16 / fp16 tensors call ``sync_masters``."""

    def __init__(self, tensors, learning_rate=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7, weight_decay=0.004,
                 global_clipnorm: float | None = None, state_bits: int = 32):
        items = list(tensors.variables if isinstance(tensors, FlatState) else tensors)
        if not items:
            raise ValueError('no tensors to optimize')
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits must be 8 or 32, got {state_bits}')
        if global_clipnorm is not None and not global_clipnorm > 0:
            raise ValueError(f'global_clipnorm must be positive, got {global_clipnorm}')
        if not (0 <= beta_1 < 1 and 0 <= beta_2 < 1):
            raise ValueError(f'beta_1 and beta_2 must lie in [0, 1), got {beta_1} and {beta_2}')
        decays = [float(d) for d in weight_decay] if hasattr(weight_decay, '__len__') else [float(weight_decay)] * len(items)
        if len(decays) != len(items):
            raise ValueError(f'{len(decays)} weight decays for {len(items)} tensors')
        self.lr, self.b1, self.b2, self.eps = learning_rate, beta_1, beta_2, epsilon
        self.global_clipnorm, self.state_bits = global_clipnorm, state_bits
        self.tensors = [v.value.data if isinstance(v, Variable) else v.detach() for v in items]
        self._leaves = [v.value if isinstance(v, Variable) else v for v in items]
        dev = self.tensors[0].device
        _lib.require_cuda(*self.tensors)
        spans = []
        for i, w in enumerate(self.tensors):
            if w.device != dev:
                raise ValueError(f'tensor {i} is on {w.device}, tensor 0 on {dev}')
            if w.dtype not in kernels.ELEMENT_TYPES:
                raise ValueError(f'tensor {i} is {w.dtype}; fp32, bf16 and fp16 are supported')
            if not w.is_contiguous():
                raise ValueError(f'tensor {i} is not contiguous')
            if w.numel():
                spans.append((w.data_ptr(), w.data_ptr() + w.numel() * w.element_size(), i))
        spans.sort()
        for (_, end, i), (start, _, j) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f'tensors {min(i, j)} and {max(i, j)} share memory')
        self.masters = [None if w.dtype == torch.float32 else w.float() for w in self.tensors]
        block = _lib.ADAMW_BLOCK
        self._numels, self._shapes = [w.numel() for w in self.tensors], [w.shape for w in self.tensors]
        ends = np.cumsum([-(-n // block) * block for n in self._numels])
        self.offsets = [0, *map(int, ends[:-1])]
        total = int(ends[-1])
        counts = [-(-n // _lib.ADAMW_CHUNK) for n in self._numels]
        first = np.zeros(len(items) + 1, dtype=np.int64)
        np.cumsum(counts, out=first[1:])
        self._first_chunk = (ctypes.c_int64 * len(first))(*first.tolist())
        table = (_lib.AdamWTensor * len(items))()
        for i, (t, v) in enumerate(zip(table, items)):
            w, master = self.tensors[i], self.masters[i]
            t.w, t.master, t.n, t.offset = w.data_ptr(), None if master is None else master.data_ptr(), w.numel(), self.offsets[i]
            t.decay, t.w_type = decays[i], kernels.ELEMENT_TYPES[w.dtype]
            t.lo, t.hi, t.l1 = (*_bounds(v), _l1(v)) if isinstance(v, Variable) else (-math.inf, math.inf, 0.0)
        raw = np.frombuffer(table, dtype=np.uint8).copy()
        pairs = np.empty((int(first[-1]), 2), dtype=np.int32)
        pairs[:, 0] = np.repeat(np.arange(len(items), dtype=np.int32), counts)
        pairs[:, 1] = np.arange(int(first[-1])) - np.repeat(first[:-1], counts)
        self._table, self._chunks = torch.from_numpy(raw).to(dev), torch.from_numpy(pairs).to(dev)
        kind = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.m = torch.zeros(total, dtype=torch.uint8 if state_bits == 8 else kind, device=dev).view(kind)
        second = torch.zeros_like(self.m.view(torch.uint8) if state_bits == 8 else self.m).view(kind)
        if state_bits == 8:
            self.r = second
            self.m_scale = torch.zeros(total // block, dtype=torch.float32, device=dev)
            self.r_scale = torch.zeros_like(self.m_scale)
        else:
            self.v = second
        self.step_count = torch.zeros((), dtype=torch.int64, device=dev)
        self._ticket = torch.zeros((), dtype=torch.int32, device=dev)

    def step(self, grads=None, grad_scale: float = 1.0) -> None:
        """One update.  ``grads``: one tensor (fp32, bf16 or fp16, of the parameter's shape) or None per parameter, None leaving
        that parameter and its moments as they are; by default the ``.grad`` of each."""
        if grads is None:
            grads = [w.grad for w in self._leaves]
        kernels.adamw_step(self, grads, grad_scale)

    def sync_masters(self) -> None:
        """Take the fp32 copies from the bf16 / fp16 tensors again (after new weights were loaded into those)."""
        for w, master in zip(self.tensors, self.masters):
            if master is not None:
                master.copy_(w)

    def moments(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The fp32 values of tensor ``i``'s first and second moment (for inspection; 8-bit states are decoded)."""
        a = self.offsets[i]
        b = a - (-self._numels[i] // _lib.ADAMW_BLOCK) * _lib.ADAMW_BLOCK
        shape = self.tensors[i].shape
        if self.state_bits == 32:
            m, v = self.m[a:b], self.v[a:b]
        else:
            s = slice(a // _lib.ADAMW_BLOCK, b // _lib.ADAMW_BLOCK)
            m, r = ((c[a:b].float().view(-1, _lib.ADAMW_BLOCK) * k[s, None]).view(-1)
                    for c, k in ((self.m, self.m_scale), (self.r, self.r_scale)))
            v = r * r
        n = self._numels[i]
        return m[:n].clone().view(shape), v[:n].clone().view(shape)

    def _state_arrays(self) -> dict:
        names = ('m', 'v') if self.state_bits == 32 else ('m', 'r', 'm_scale', 'r_scale')
        arrays = {name: getattr(self, name) for name in names}
        arrays['step_count'] = self.step_count
        arrays.update({f'master_{i}': w for i, w in enumerate(self.masters) if w is not None})
        return arrays

    def state_dict(self) -> dict:
        """Copies of the state arrays (codes as bytes) for a checkpoint."""
        return {k: (a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a).clone() for k, a in self._state_arrays().items()}

    def load_state_dict(self, state: dict) -> None:
        """Take over the arrays of ``state_dict`` of an optimizer over tensors of the same sizes and types."""
        own = self._state_arrays()
        if set(own) != set(state):
            raise ValueError(f'the state has {sorted(state)}, this optimizer keeps {sorted(own)}')
        for k, a in own.items():
            if tuple(state[k].shape) != tuple(a.shape):
                raise ValueError(f'{k} has shape {tuple(state[k].shape)}, expected {tuple(a.shape)}')
            if a.dtype == torch.float8_e4m3fn and state[k].dtype not in (torch.uint8, a.dtype):  # bytes, never numbers to round again
                raise ValueError(f'{k} holds e4m3 codes (bytes), got {state[k].dtype}')
        for k, a in own.items():
            if a.dtype == torch.float8_e4m3fn:
                a.view(torch.uint8).copy_(state[k].view(torch.uint8))
            else:
                a.copy_(state[k])


class PeerExchange:
    """This rank's gradient exchange buffer and its mappings of the other ranks' buffers (CUDA IPC over NVLink), for
    ``FusedAdam.step_peers``: the gradient sum over the ranks and the optimizer update as one kernel per rank, with plain
    peer loads instead of an NCCL all-reduce.  One node, one process per GPU.  ``PeerExchange.create`` returns None when
    some rank cannot map some other rank's buffer (the ranks then agree to keep the NCCL all-reduce)."""

    def __init__(self, own, ptrs, opened, world, rank, device):
        self.own, self.ptrs, self.opened = own, ptrs, opened
        self.world, self.rank, self.device = world, rank, device
        self.max_polls = int(os.environ.get('HGQ_PEER_MAX_POLLS', str(1 << 25)))  # a few seconds of polling at most

    @classmethod
    def create(cls, dp: 'DataParallel', n: int, device: torch.device):
        import ctypes

        L = _lib.lib()
        world, rank = dp.world, dp.rank
        own = ctypes.c_void_p()
        handle = (ctypes.c_ubyte * 64)()
        ok = 1
        with torch.cuda.device(device):
            st = L.hgq_peer_buffer_create(L.hgq_peer_exchange_bytes(n), ctypes.byref(own), handle)
            if st != 0:
                ok, own = 0, ctypes.c_void_p()
            mine = torch.tensor(list(bytes(handle)), dtype=torch.uint8, device=device)
            gathered = [torch.empty_like(mine) for _ in range(world)]
            dist.all_gather(gathered, mine, group=dp.group)
            ptrs = (ctypes.c_void_p * world)()
            opened = []
            for r, h in enumerate(gathered):
                if r == rank:
                    ptrs[r] = own.value
                    continue
                raw = (ctypes.c_ubyte * 64)(*h.cpu().tolist())
                p = ctypes.c_void_p()
                if ok and L.hgq_peer_buffer_open(raw, ctypes.byref(p)) == 0:
                    ptrs[r] = p.value
                    opened.append(p.value)
                else:
                    ok = 0
            agreed = torch.tensor([ok], dtype=torch.int32, device=device)
            dist.all_reduce(agreed, op=dist.ReduceOp.MIN, group=dp.group)
            self = cls(own.value, ptrs, opened, world, rank, device)
            if int(agreed.item()) == 0:
                self.close()
                return None
            return self

    def close(self) -> None:
        L = _lib.lib()
        with torch.cuda.device(self.device):
            for p in self.opened:
                L.hgq_peer_buffer_close(p)
            if self.own:
                L.hgq_peer_buffer_destroy(self.own)
        self.opened, self.own = [], None


def shard_batch(n: int, rank: int, world: int) -> slice:
    """Contiguous, equal shard of a batch of n samples (n must divide evenly so per-rank means average correctly)."""
    if n % world != 0:
        raise ValueError(f'batch {n} does not divide over {world} ranks')
    per = n // world
    return slice(rank * per, (rank + 1) * per)


class DataParallel:
    """Batch-sharded training over the ranks of a torch.distributed process group (NCCL on GPUs).

    ``sync_gradients`` averages the flat gradient bucket; ``absmax_sync`` is installed as the hook the WRAP
    quantizers call on their abs-max statistics (a MAX all-reduce), which keeps ``i`` -- and with it the EBOPs
    term -- identical on every rank and equal to what one rank would compute on the whole batch.
    """

    def __init__(self, group=None):
        if not dist.is_initialized():
            raise RuntimeError('torch.distributed is not initialised')
        self.group = group
        self.world = dist.get_world_size(group)
        self.rank = dist.get_rank(group)

    def sync_gradients(self, grads: torch.Tensor, average: bool = True) -> None:
        """Sum the gradient bucket over the ranks; ``average=False`` leaves the division by the number of ranks to the
        caller (the trainer folds it into the optimizer kernel's gradient scale instead of a pass of its own)."""
        if self.world > 1:
            dist.all_reduce(grads, op=dist.ReduceOp.SUM, group=self.group)
            if average:
                grads.div_(self.world)

    def absmax_sync(self, absmax: torch.Tensor) -> torch.Tensor:
        if self.world > 1:
            dist.all_reduce(absmax, op=dist.ReduceOp.MAX, group=self.group)
        return absmax

    def __enter__(self):
        from . import backend

        self._prev = (_fpq.absmax_sync_hook, backend.moments_group)
        _fpq.absmax_sync_hook = self.absmax_sync
        backend.moments_group = self.group  # synchronized batch statistics are averaged over this group's ranks
        return self

    def __exit__(self, *exc):
        from . import backend

        _fpq.absmax_sync_hook, backend.moments_group = self._prev


class _SoftmaxXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels):
        from . import kernels

        loss, dlogits = kernels.softmax_xent(logits, labels)
        ctx.save_for_backward(dlogits)
        return loss

    @staticmethod
    def backward(ctx, g):
        (dlogits,) = ctx.saved_tensors
        return dlogits * g, None


def sparse_categorical_crossentropy(logits, labels):
    """Mean softmax cross-entropy from logits with integer labels (what the reference's models are compiled with), on the
    fused kernel when the logits are a CUDA [B, C <= 64] fp32 matrix with int64 labels; torch's otherwise."""
    if logits.is_cuda and logits.dtype == torch.float32 and logits.dim() == 2 and logits.shape[1] <= 64 and labels.dtype == torch.int64:
        return _SoftmaxXentFn.apply(logits, labels)
    return torch.nn.functional.cross_entropy(logits, labels)


class Trainer:
    """One model, one flat bucket, one fused optimizer; ``step(x, y)`` runs a full QAT step and returns the loss.

    ``capture(x, y)`` records the whole step (forward, backward, gradient exchange, optimizer) into a CUDA graph over
    static input buffers; afterwards ``step`` copies the batch into those buffers and replays the graph, which removes
    the per-kernel launch and Python cost that dominates the small models.
    """

    def __init__(self, model: Layer, loss_fn, learning_rate=1e-3, dp: DataParallel | None = None, engine: bool | None = None,
                 optimizer=None):
        """``optimizer``: a callable that makes the optimizer from the trainer's ``FlatState`` (``lambda state: FusedAdamW(state,
        global_clipnorm=1.0)``); None: ``FusedAdam`` at ``learning_rate``.

        ``engine``: run forward and backward through the static step plan of ``hgq2_b200.engine`` (batched bitwidth
        arithmetic, no autograd graph).  None (default): use it when it covers the model, else the autograd path; True:
        require it (raises ``engine.Unsupported`` otherwise); False: always the autograd path.  The environment variable
        ``HGQ_ENGINE=0`` turns the default off."""
        self.model = model
        self.loss_fn = loss_fn
        self.dp = dp
        self.state = FlatState(model)
        self.opt = FusedAdam(self.state, learning_rate=learning_rate) if optimizer is None else optimizer(self.state)
        self.engine = None
        self.engine_refusal = None  # why the static step plan is not in use (None: it is, or it was not asked for)
        if engine is None:
            engine = None if os.environ.get('HGQ_ENGINE', '1') != '0' else False
        if engine is not False and self.state.params.is_cuda:
            from .engine import Engine, Unsupported

            try:
                self.engine = Engine(model, self.state)
                self.engine.dp = dp
            except Unsupported as why:
                if engine is True:
                    raise
                self.engine_refusal = str(why)
        # gradient exchange over peer memory inside the optimizer kernel (one node, NCCL process group on GPUs);
        # HGQ_PEER_EXCHANGE=0 keeps the NCCL all-reduce
        self.peers = None
        if (optimizer is None and dp is not None and dp.world > 1 and self.state.params.is_cuda and dist.get_backend(dp.group) == 'nccl'
                and os.environ.get('HGQ_PEER_EXCHANGE', '1') != '0'):
            self.peers = PeerExchange.create(dp, self.state.n, self.state.params.device)
        self._graphs = []      # captured steps, one per set of static input buffers
        self._sbuf = []        # the static (x, y) buffers the graphs read
        self._next_buf = 0
        # status word of the tensor-core kernels (set when a bounded device-side wait gives up), read back without a sync
        self._status_dev = None
        self._status_host = None
        self._status_event = None

    def forward_backward(self, x, y):
        if self.engine is not None:
            from .engine import Unsupported

            try:
                self.engine.check(int(x.shape[0]))
            except Unsupported as why:  # this batch size is outside some kernel: the autograd path takes over for good
                self.engine, self.engine_refusal = None, str(why)
            else:
                return self.engine.forward_backward(x, y, self.loss_fn)
        self.state.zero_grad()
        pred = self.model(x, training=True)
        task = self.loss_fn(pred, y)
        join_bookkeeping()  # the EBOPs terms were computed on the bookkeeping stream
        total = task
        for extra in self.model._losses:  # the beta * EBOPs terms; the weight regularisers are fused into the optimizer
            total = total + extra
        total.backward()
        return task.detach(), total.detach() + self.state.regularization_loss()

    def _eager_step(self, x, y):
        if self.dp is not None:
            with self.dp:
                task, total = self.forward_backward(x, y)
            if self.peers is not None:
                self.opt.step_peers(self.peers)  # gradient sum over peer memory and update in one kernel
            else:
                self.dp.sync_gradients(self.state.grads, average=False)
                self.opt.step(grad_scale=1.0 / self.dp.world)  # the mean over the ranks, folded into the optimizer kernel
        else:
            task, total = self.forward_backward(x, y)
            self.opt.step()
        self._queue_status_read()
        return total

    # -- device status ---------------------------------------------------------------------------------------------------
    def _queue_status_read(self) -> None:
        """Copy the device status word to pinned host memory behind the step (no synchronisation; part of a captured
        step like any other node)."""
        if not self.state.params.is_cuda:
            return
        from . import kernels

        if self._status_dev is None:
            self._status_dev = kernels.status_word(self.state.params.device)
            self._status_host = torch.zeros(1, dtype=torch.int32).pin_memory()
        self._status_host.copy_(self._status_dev, non_blocking=True)
        if not torch.cuda.is_current_stream_capturing():
            self._status_event = torch.cuda.Event()
            self._status_event.record()

    def check_status(self, wait: bool = False) -> None:
        """Raise ``HGQError`` (HGQ_ERR_TIMEOUT) if a kernel of an earlier step reported that one of its bounded waits gave
        up: that step's outputs, gradients and the update made from them are garbage.  Without ``wait`` only a read-back
        that has already landed is looked at, so calling this at the start of every step costs no synchronisation; the
        word is cleared once reported."""
        if self._status_host is None:
            return
        ev = self._status_event
        if ev is not None:
            if wait:
                ev.synchronize()
            elif not ev.query():
                return
        if int(self._status_host[0]) != 0:
            v = int(self._status_host[0])
            self._status_host.zero_()
            self._status_dev.zero_()
            raise _lib.HGQError(-7, f'training step (device status word = {v})')

    def capture(self, x, y, warmup: int = 3, double_buffer: bool = False) -> None:
        """Record the step as a CUDA graph for batches shaped like (x, y).  Runs ``warmup`` real steps first.

        ``double_buffer``: record the step twice, over two sets of static input buffers that share one memory pool;
        ``prefetch`` then copies a host batch straight into the set the step after next will read, with no staging copy
        on the device."""
        self._sbuf = [(x.clone(), y.clone()) for _ in range(2 if double_buffer else 1)]
        self._graphs, self._next_buf = [], 0
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warmup):
                self._eager_step(*self._sbuf[0])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        self.check_status(wait=True)
        pool = None
        for sx, sy in self._sbuf:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=pool):
                loss = self._eager_step(sx, sy)
            pool = graph.pool()
            self._graphs.append((graph, loss))

    def prefetch(self, hx, hy):
        """Start the host-to-device copy of a (pinned) host batch on a copy stream of its own and return a handle for
        ``step_prefetched``; the copy of batch n + 1 overlaps step n.  After ``capture(..., double_buffer=True)`` the
        batch lands directly in the static buffers of the graph that will consume it; otherwise two device staging
        slots alternate."""
        if not hasattr(self, '_copy_stream'):
            self._copy_stream = torch.cuda.Stream()
            self._slots = [None, None]
            self._slot = 0
        direct = len(self._graphs) == 2 and hx.shape == self._sbuf[0][0].shape and hy.shape == self._sbuf[0][1].shape
        if direct:
            j = self._next_buf
            self._next_buf ^= 1
            dx, dy = self._sbuf[j]
        else:
            j = self._slot
            self._slot ^= 1
            dev = self.state.params.device
            if self._slots[j] is None or self._slots[j][0].shape != hx.shape or self._slots[j][1].shape != hy.shape:
                self._slots[j] = (torch.empty(hx.shape, dtype=hx.dtype, device=dev), torch.empty(hy.shape, dtype=hy.dtype, device=dev))
            dx, dy = self._slots[j]
        # everything queued so far has consumed the buffer's previous batch (two steps back; the step that overlaps this
        # copy is launched after this call and reads the other buffer)
        self._copy_stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self._copy_stream):
            dx.copy_(hx, non_blocking=True)
            dy.copy_(hy, non_blocking=True)
            done = torch.cuda.Event()
            done.record()
        return dx, dy, done, (j if direct else None)

    def step_prefetched(self, handle):
        """``step`` on a batch started with ``prefetch``."""
        dx, dy, done, buf = handle
        torch.cuda.current_stream().wait_event(done)
        if buf is not None:
            self.check_status()
            return self._replay(buf)
        return self.step(dx, dy)

    def step(self, x, y):
        """One QAT step on a device batch; returns the loss (a device scalar, valid until the next step)."""
        self.check_status()
        if self._graphs and x.shape == self._sbuf[0][0].shape and y.shape == self._sbuf[0][1].shape:
            sx, sy = self._sbuf[0]
            if x.data_ptr() != sx.data_ptr():
                sx.copy_(x, non_blocking=True)
            if y.data_ptr() != sy.data_ptr():
                sy.copy_(y, non_blocking=True)
            return self._replay(0)
        return self._eager_step(x, y)

    def _replay(self, buf: int):
        graph, loss = self._graphs[buf]
        graph.replay()
        self._status_event = torch.cuda.Event()  # behind the replay, whose last node is the status read-back
        self._status_event.record()
        return loss

    @property
    def static_inputs(self):
        """The static (x, y) buffers of the captured step: a caller that writes its batch there itself (and passes these
        very tensors to ``step``) saves the device-to-device copy."""
        return self._sbuf[0] if self._sbuf else None
