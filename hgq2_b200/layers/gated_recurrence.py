"""QGatedRecurrence: a gated linear recurrence over the sequence axis, its input and gate made by one quantised projection.

The sequence layer beside QMultiHeadAttention for axes that attention's quadratic cost rules out: time and memory are linear in
the length, and a stream is served token by token from a state of ``units`` numbers.  No counterpart in the accelerated scope of
the reference (its recurrent cells, src/hgq/layers/rnn/, feed the state back through a matrix and run step by step)."""

from __future__ import annotations

import torch

from ..backend import Initializer, get_initializer
from ..quantizer.config import QuantizerConfig
from ._functions import GatedScanFn
from .core.base import QLayerBase
from .core.einsum_dense import QEinsumDense


class _PairBias(Initializer):
    """Bias [2, units]: the input's row and the gate's row from an initializer each."""

    def __init__(self, first: Initializer, second: Initializer):
        self.first, self.second = first, second

    def __call__(self, shape, dtype=torch.float32, device=None):
        return torch.stack([init(tuple(shape[1:]), dtype, device) for init in (self.first, self.second)])


class QGatedRecurrence(QLayerBase):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t on [batch, time, features] inputs, with (x, z) = one QEinsumDense of the inputs and
    a = sigmoid(z).  Returns h [batch, time, units] (``return_sequences=False``: its last step), with the fp32 state behind each
    row's last step when ``return_state``.

    ``gate_bias_initializer``: the bias of z; positive values start with a long memory.  At a call, ``initial_state`` [batch, units]
    carries a state over (token-by-token serving), ``lengths`` [batch] gives the steps of each row of a padded batch: h is zero
    behind them.  EBOPs are those of the projection; the recurrence itself runs in fp32, and ``enable_oq`` quantises h."""

    __output_quantizer_handled__ = True

    def __init__(self, units, use_bias=True, return_sequences=True, return_state=False, kernel_initializer='glorot_uniform',
                 bias_initializer='zeros', gate_bias_initializer=2.0, iq_conf: QuantizerConfig | None = None,
                 kq_conf: QuantizerConfig | None = None, bq_conf: QuantizerConfig | None = None, parallelization_factor=-1, **kwargs):
        super().__init__(**kwargs)
        if int(units) <= 0:
            raise ValueError(f'units must be positive, got {units}')
        self.units, self._use_bias = int(units), use_bias
        self.return_sequences, self.return_state = return_sequences, return_state
        self._kernel_initializer = get_initializer(kernel_initializer)
        self._bias_initializer = _PairBias(get_initializer(bias_initializer), get_initializer(gate_bias_initializer))
        self._iq_conf, self._kq_conf, self._bq_conf = iq_conf, kq_conf, bq_conf
        self.parallelization_factor = parallelization_factor

    def build(self, input_shape):
        if len(input_shape) != 3:
            raise NotImplementedError(f'only [batch, time, features] inputs are supported, got {len(input_shape)} axes')
        self._projection = QEinsumDense('abc,cde->abde', (input_shape[1], 2, self.units), bias_axes='de' if self._use_bias else None,
                                        kernel_initializer=self._kernel_initializer, bias_initializer=self._bias_initializer,
                                        iq_conf=self._iq_conf, kq_conf=self._kq_conf, bq_conf=self._bq_conf, enable_iq=self.enable_iq,
                                        enable_oq=False, enable_ebops=self.enable_ebops, beta0=self._beta0.clone(),
                                        ebops_factor=self.ebops_factor, parallelization_factor=self.parallelization_factor,
                                        name=f'{self.name}_projection')
        self._projection.build(input_shape)
        self._projection.built = True
        if self.enable_oq and not self.oq.built:
            self.oq.build(self.compute_output_shape(input_shape))
            self.oq.built = True
        self.built = True

    @property
    def projection(self) -> QEinsumDense:
        return self._projection

    @property
    def ebops(self):
        return self._projection.ebops if self.built else torch.zeros((), dtype=torch.uint32)

    def compute_output_shape(self, input_shape):
        shape = tuple(input_shape[:2]) if self.return_sequences else tuple(input_shape[:1])
        return shape + (self.units,)

    def _project(self, inputs, training):
        """(x, z) [batch, time, 2, units].  The projection is built on a number of steps; a call outside training may have another
        one if no bitwidth depends on the step."""
        proj, steps = self._projection, int(inputs.shape[1])
        built = proj.full_output_shape
        if steps == built[1]:
            return proj(inputs, training=training)
        if training:
            raise ValueError(f'{self.name} is built for {built[1]} steps, got {steps} in training')
        for q in ([proj.iq] if self.enable_iq else []) + ([self.oq] if self.enable_oq and self.return_sequences else []):
            k = getattr(q.quantizer, '_k', None)
            if k is not None and len(k.shape) == 3 and k.shape[1] != 1:
                raise ValueError(f'{q.name} has a bitwidth per step: {self.name} runs on the {built[1]} steps it is built for; make '
                                 'the time axis homogeneous (homogeneous_axis=(0, 1)) to run on others')
        return proj(inputs, training=training, output_shape=(steps, *built[2:]))

    def call(self, inputs, initial_state=None, lengths=None, training=None):
        h, state = GatedScanFn.apply(self._project(inputs, training), initial_state, lengths)
        if not self.return_sequences:
            h = state.to(h.dtype)
        if self.enable_oq:
            h = self.oq(h, training=training)
        return (h, state) if self.return_state else h

    def get_config(self):
        config = super().get_config()
        config.update({'units': self.units, 'use_bias': self._use_bias, 'return_sequences': self.return_sequences,
                       'return_state': self.return_state, 'parallelization_factor': self.parallelization_factor,
                       'iq_conf': self._projection._iq.config if self.built and self.enable_iq else self._iq_conf,
                       'kq_conf': self._projection.kq.config if self.built else self._kq_conf,
                       'bq_conf': self._projection.bq.config if self.built and self._use_bias else self._bq_conf})
        return config
