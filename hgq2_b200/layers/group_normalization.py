"""GroupNormalization: keras.layers.GroupNormalization for channels-last tensors with the activation that follows it in the same
pass.  Not a quantised layer: it stands between quantised layers, whose input quantizers take its output."""

from __future__ import annotations

from ..backend import Layer, get_initializer
from ..kernels import ACTIVATIONS
from ._functions import GroupNormFn


class GroupNormalization(Layer):
    """y = activation(gamma * (x - mean) / sqrt(variance + epsilon) + beta), the statistics taken per sample over all positions and
    the channels of each group; the same in training and evaluation.  ``groups=-1``: one group per channel.  ``activation``: None,
    'relu', 'silu' or 'gelu'.  Inputs are [batch, ..., channels] in fp32, bf16 or fp16."""

    def __init__(self, groups=32, axis=-1, epsilon=1e-3, center=True, scale=True, beta_initializer='zeros', gamma_initializer='ones',
                 beta_regularizer=None, gamma_regularizer=None, beta_constraint=None, gamma_constraint=None, activation=None, **kwargs):
        super().__init__(**kwargs)
        if activation not in ACTIVATIONS:
            raise ValueError(f'activation {activation!r} is not one of {list(ACTIVATIONS)}')
        self.groups, self.axis, self.epsilon = int(groups), int(axis), float(epsilon)
        self.center, self.scale, self.activation = center, scale, activation
        self.beta_initializer, self.gamma_initializer = get_initializer(beta_initializer), get_initializer(gamma_initializer)
        self.beta_regularizer, self.gamma_regularizer = beta_regularizer, gamma_regularizer
        self.beta_constraint, self.gamma_constraint = beta_constraint, gamma_constraint
        self._gamma = self._beta = None

    def build(self, input_shape):
        if self.axis not in (-1, len(input_shape) - 1):
            raise NotImplementedError(f'axis {self.axis}: only the last axis (channels last) is supported')
        dim = int(input_shape[-1])
        if self.groups == -1:
            self.groups = dim
        if self.groups <= 0 or dim % self.groups:
            raise ValueError(f'{self.groups} groups do not divide {dim} channels')
        if self.scale:
            self._gamma = self.add_weight(shape=(dim,), name='gamma', initializer=self.gamma_initializer,
                                          regularizer=self.gamma_regularizer, constraint=self.gamma_constraint)
        if self.center:
            self._beta = self.add_weight(shape=(dim,), name='beta', initializer=self.beta_initializer,
                                         regularizer=self.beta_regularizer, constraint=self.beta_constraint)
        super().build(input_shape)

    @property
    def gamma(self):
        return self._gamma.value if self._gamma is not None else None

    @property
    def beta(self):
        return self._beta.value if self._beta is not None else None

    def compute_output_shape(self, input_shape):
        return tuple(input_shape)

    def call(self, inputs):
        return GroupNormFn.apply(inputs, self.gamma, self.beta, self.groups, self.epsilon, self.activation)

    def get_config(self):
        config = super().get_config()
        config.update({'groups': self.groups, 'axis': self.axis, 'epsilon': self.epsilon, 'center': self.center, 'scale': self.scale,
                       'activation': self.activation})
        return config
