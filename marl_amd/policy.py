"""Actor-critic MLP with the parameter names of the reference's ``model.Agent``
(model.py:11-68), so that checkpoints interchange: ``network.{0,2}`` (obs -> 512 -> 256,
ReLU), ``actor`` (256 -> n_actions), ``critic`` (256 -> 1) and ``centralised_critics.{0,2,4}``
(obs_dim * num_agents * num_envs -> 512 -> 256 -> 1).  All layers start orthogonal with gain
sqrt(2) and zero bias (model.py:6-9).  The matrix products run on PyTorch-ROCm (rocBLAS /
hipBLASLt); which library call computes a layer of a small batch is a fixed function of its
shape (`_table_form`).  On request the trunk is computed in 4-bit floating point (`use_mxfp4_trunk`, the
HIP passes of `mxfp4`) and keeps its activations for the backward pass in 8 bits
(`use_activation_checkpoints`, those of `act8`)."""
from __future__ import annotations

import math
import os
import threading
import warnings

import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.distributions import Categorical

from . import act8, mxfp4


def _ortho(linear: nn.Linear, gain: float = math.sqrt(2.0), bias: float = 0.0) -> nn.Linear:
    nn.init.orthogonal_(linear.weight, gain)
    nn.init.constant_(linear.bias, bias)
    return linear


def _weight_grad(gy, x):
    """gy^T @ x for a tall batch (K rows, K >> features).  hipBLASLt's kernel choice for this
    skinny shape leaves most of the chip idle (1.15 ms for 512 x 202 over K = 262,144); cutting K
    into S slabs, one batched GEMM and a sum over the slabs is 2-4x faster on MI355X
    (0.50 ms for the same shape).  Same float32 products, another summation order."""
    K = gy.shape[0]
    S = 1
    while S < 128 and K % (2 * S) == 0 and K // (2 * S) >= 2048:
        S *= 2
    if S == 1 or not gy.is_cuda:
        return gy.t() @ x
    return torch.bmm(gy.view(S, K // S, -1).transpose(1, 2), x.view(S, K // S, -1)).sum(0)


def _bias_grad(gy):
    """gy.sum(0), from launches that replay (`act8.column_sums`): updates of small minibatches are captured.  Where the
    backward pass itself is differentiated it is torch's sum, which has a derivative."""
    if not gy.is_cuda or gy.dtype not in act8._TYPES or torch.is_grad_enabled():
        return gy.sum(0)
    return act8.column_sums(gy).to(gy.dtype)


# Below 512 rows (the reference's batch sizes: 16 envs x 2 agents = 32 rows per rollout step)
# hipBLASLt's pick for the fused call is erratic on MI355X: rows x 512 -> 256 takes 17.8 us at 32
# rows, 60 us at 128, 118 us at 256 and 6 us at 512, while a plain rocBLAS product takes 3.7 us at
# all of them (plus two small in-place launches for bias and ReLU); for the other layers of the same
# MLP the fused call wins (rows x 202 -> 512: 5.4 against 7.5 us).  (profiles/diag/small_gemm2.py)
# The forms sum in different orders, so which one runs must not depend on anything that varies from
# run to run or from rank to rank: it is a fixed function of the layer's shape (`_TABLE_FORM`).
# MARL_AMD_SMALL_GEMM=fused|plain|gemv forces one form; MARL_AMD_SMALL_GEMM=tune times the forms once
# per shape instead (a tuning aid: its choices can differ between runs, and with them the bits of a
# seeded run).
_SMALL_ROWS = 512
_GEMM_CHOICE = {}
_BLAS_LOCK = threading.Lock()


def _table_form(rows, in_features, out_features):
    """the measured winners on MI355X: a single row (the centralised critic's joint observation) as a
    matrix-vector product; the 512-wide hidden layer through rocBLAS; everything else fused"""
    if rows == 1 and in_features >= 1024:
        return "gemv"
    if in_features == 512 and out_features <= 256:
        return "plain"
    return "fused"


def gemm_choices():
    """the forms in use so far, {(rows, in_features, out_features, relu): "fused" | "plain" | "gemv"}"""
    return dict(_GEMM_CHOICE)


def _fused_linear(x, weight, bias, relu):
    if relu:
        return torch._addmm_activation(bias, x, weight.t(), use_gelu=False)
    return torch.addmm(bias, x, weight.t())


_blas_switch_announced = False


class _FirstBlasSwitch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t):
        blas = torch.backends.cuda.preferred_blas_library
        blas(blas())
        return t


def _announce_blas_switch_quietly(t):
    """PyTorch issues a one-time "experimental feature" notice when the preferred BLAS library is
    set: as a Python warning when the call happens inside an operator (raised only when the
    outermost operator returns, here `_LinearReLU.apply`, where it can no longer be filtered at its
    source), straight to stderr otherwise.  The first switch is therefore made inside a small
    operator of its own with warnings ignored around it."""
    global _blas_switch_announced
    if not _blas_switch_announced:
        _blas_switch_announced = True
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            _FirstBlasSwitch.apply(t)


def _plain_linear(x, weight, bias, relu):
    """the product through rocBLAS, bias and ReLU as in-place launches of their own"""
    blas = torch.backends.cuda.preferred_blas_library
    with _BLAS_LOCK:  # the preference is process-wide: one thread at a time, always put back
        prev = blas()
        blas("hipblas")
        try:
            out = torch.mm(x, weight.t())
        finally:
            blas(prev)
    out.add_(bias)
    return out.relu_() if relu else out


def _gemv_linear(x, weight, bias, relu):
    """a single row (the centralised critic's joint observation, model.py:45): matrix-vector product"""
    out = torch.addmv(bias, weight, x[0]).unsqueeze(0)
    return out.relu_() if relu else out


_FORMS = {"fused": _fused_linear, "plain": _plain_linear, "gemv": _gemv_linear}


def _small_gemm_form(x, weight, bias, relu):
    rows = x.shape[0]
    if rows >= _SMALL_ROWS:
        return "fused"
    key = (rows, weight.shape[1], weight.shape[0], bool(relu))
    form = _GEMM_CHOICE.get(key)
    if form is not None:
        return form
    forced = os.environ.get("MARL_AMD_SMALL_GEMM", "table")
    if forced in ("fused", "plain", "gemv"):
        form = forced if (forced != "gemv" or rows == 1) else "fused"
    elif forced != "tune":
        form = _table_form(rows, weight.shape[1], weight.shape[0])
    elif torch.cuda.is_current_stream_capturing():
        return "fused"  # cannot time under capture; decided at the next eager call
    else:
        # Timed as the small-batch rollouts and updates run them: replayed from a hipGraph.  (Launched
        # eagerly from Python both forms are bound by the host's launch rate and the form with fewer
        # launches always looks better, whatever its kernels cost.)
        times = []
        names = ("fused", "plain", "gemv") if rows == 1 else ("fused", "plain")
        for name in names:
            fn = _FORMS[name]
            fn(x, weight, bias, relu)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, capture_error_mode="thread_local"):
                for _ in range(10):
                    fn(x, weight, bias, relu)
            g.replay()
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            for _ in range(3):
                g.replay()
            e1.record()
            e1.synchronize()
            times.append(e0.elapsed_time(e1))
            del g
        # another form has to win clearly: a close call must not flip from run to run
        best = min(range(len(times)), key=lambda k: times[k])
        form = names[best] if times[best] * 1.25 < times[0] else "fused"
    _GEMM_CHOICE[key] = form
    return form


def _forward(x, weight, bias, relu, coarse, out_dtype):
    if coarse is not None:
        return mxfp4.linear(x, coarse, bias.float(), relu=relu, out_dtype=out_dtype or weight.dtype)
    return _FORMS[_small_gemm_form(x, weight, bias, relu)](x, weight, bias, relu)


class _LinearReLU(torch.autograd.Function):
    """relu(x @ W^T + b) (or without the ReLU): one GEMM with a fused epilogue, or for the small
    batches where that call is slow a plain product plus in-place bias and ReLU; the backward
    pass forms the weight gradient with `_weight_grad`.  With `coarse`, the weight in 4 bits, the forward pass is
    `mxfp4.linear`'s, its result in `out_dtype`, and the backward pass is the unrounded layer's: its input and weight as they
    were before they went to 4 bits, the ReLU's mask that of the 4-bit result."""

    @staticmethod
    def forward(ctx, x, weight, bias, relu, coarse=None, out_dtype=None):
        out = _forward(x, weight, bias, relu, coarse, out_dtype)
        ctx.relu = relu
        ctx.save_for_backward(x.to(weight.dtype), weight, out if relu else None)
        return out

    @staticmethod
    def backward(ctx, gy):
        x, weight, out = ctx.saved_tensors
        if ctx.relu:
            gy = torch.ops.aten.threshold_backward(gy, out, 0)
        gy = gy.contiguous().to(weight.dtype)
        gw, gb = _weight_grad(gy, x), _bias_grad(gy)
        gx = gy @ weight if ctx.needs_input_grad[0] else None
        return gx, gw, gb, None, None, None


class _StraightLinear(torch.autograd.Function):
    """`_LinearReLU` with a weight in 4 bits whose backward pass is the 4-bit layer's, with the roundings' derivatives taken as
    one: it reads input and weight as the product did, and keeps the input in 4 bits."""

    @staticmethod
    def forward(ctx, x, weight, bias, relu, coarse, out_dtype=None):
        kept = mxfp4.quantize(x)
        out = _forward(kept, weight, bias, relu, coarse, out_dtype)
        ctx.relu, ctx.cols, ctx.dtype = relu, x.shape[1], weight.dtype
        back = coarse.dequantize(weight.dtype) if ctx.needs_input_grad[0] else None
        ctx.save_for_backward(kept.codes, kept.scales, back, out if relu else None)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        codes, scales, back, out = ctx.saved_tensors
        if ctx.relu:
            gy = torch.ops.aten.threshold_backward(gy, out, 0)
        gy = gy.contiguous().to(ctx.dtype)
        # the input's values are gone before there is a gradient of their size
        gw = _weight_grad(gy, mxfp4.MXFP4(codes, scales, ctx.cols).dequantize(ctx.dtype))
        gb, gx = _bias_grad(gy), gy @ back if ctx.needs_input_grad[0] else None
        return gx, gw, gb, None, None, None


class _KeptLinear(torch.autograd.Function):
    """`_LinearReLU` that keeps its input, and behind a ReLU its output, in 8 bits for the backward pass instead of in
    float32.  The input comes with its kept form (codes, scales, whether nonnegative); the output's goes on to the next layer, so that
    what lies between two layers is kept once.  The gradient of the weight is formed from the kept input, the ReLU's mask is the
    kept output's and exact; the forward pass and the gradient of the input are those of `_LinearReLU`.  With `straight` the kept
    input is x in 4 bits (codes and scales of an MXFP4, whose values 8 bits hold exactly)."""

    @staticmethod
    def forward(ctx, x, codes, scales, nonnegative, weight, bias, relu, coarse=None, out_dtype=None, straight=False):
        ctx.cols = x.shape[1] if straight else None
        out = _forward(mxfp4.MXFP4(codes, scales, ctx.cols) if straight else x, weight, bias, relu, coarse, out_dtype)
        kept = act8.compress(out, nonnegative=True) if relu else None
        ctx.nonnegative, ctx.dtype = nonnegative, weight.dtype
        back = weight if not straight else coarse.dequantize(weight.dtype) if ctx.needs_input_grad[0] else None
        ctx.save_for_backward(codes, scales, back, kept.codes if relu else None, kept.scales if relu else None)
        if not relu:
            return out
        ctx.set_materialize_grads(False)  # no zeros as large as the codes in the place of their gradients
        ctx.mark_non_differentiable(kept.codes, kept.scales)
        return out, kept.codes, kept.scales

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, *_kept):
        codes, scales, weight, out_codes, out_scales = ctx.saved_tensors
        if gy is None:  # what reads the output has no gradient for it
            return (None,) * 10
        mask = None if out_codes is None else act8.Act8(out_codes, out_scales, True)
        if ctx.cols is None:
            x = act8.Act8(codes, scales, ctx.nonnegative)
        else:
            x = act8.compress(mxfp4.MXFP4(codes, scales, ctx.cols).dequantize(), ctx.nonnegative)
        gw, gb, masked = act8.weight_grad(gy, x, mask, want_masked=ctx.needs_input_grad[0])
        del x
        gx = (gy if mask is None else masked).to(ctx.dtype) @ weight if ctx.needs_input_grad[0] else None
        return gx, None, None, None, gw, gb, None, None, None, None


def _linear(layer: nn.Linear, x, relu, coarse=None, out_dtype=None, straight=False):
    if x.is_cuda and x.dim() == 2:
        if x.shape[0] < _SMALL_ROWS and coarse is None:
            _announce_blas_switch_quietly(x)
        return (_StraightLinear if straight else _LinearReLU).apply(x.contiguous(), layer.weight, layer.bias, relu, coarse, out_dtype)
    out = layer(x)
    return torch.relu(out) if relu else out


def _mlp(sizes, final_activation):
    layers = []
    for k in range(len(sizes) - 1):
        layers.append(_ortho(nn.Linear(sizes[k], sizes[k + 1])))
        if k < len(sizes) - 2 or final_activation:
            layers.append(nn.ReLU())
    return nn.Sequential(*layers)


class Agent(nn.Module):
    def __init__(self, obs_space, action_space, num_agents=4, num_envs=1, build_centralised=True):
        super().__init__()
        self.obs_space, self.action_space = obs_space, action_space
        self.num_agents, self.num_envs = int(num_agents), int(num_envs)
        d = int(obs_space.shape[0])
        self.network = _mlp([d, 512, 256], final_activation=True)
        self.actor = _ortho(nn.Linear(256, int(action_space.n)))
        self.critic = _ortho(nn.Linear(256, 1))
        # model.py:28-34: one value for the concatenated observations of every row
        # Its first layer is obs_dim * num_agents * num_envs wide: 54 GB of weights at 65,536 envs, and
        # an orthogonal initialisation (a QR factorisation) of that matrix on the host.  A
        # decentralised learner never evaluates it and may leave it out.
        self.sampler = None  # set by use_fused_sampling(); plain torch.distributions otherwise
        self._head_w = self._head_b = None  # stacked heads of rollout_step
        self._coarse = None  # 4-bit weights of the trunk, set by use_mxfp4_trunk()
        self._straight = False  # the 4-bit trunk's backward pass, set by use_mxfp4_trunk()
        self._keep_in_8_bits = False  # set by use_activation_checkpoints()
        self.centralised_critics = (_mlp([d * self.num_agents * self.num_envs, 512, 256, 1], final_activation=False)
                                    if build_centralised else None)

    def _trunk(self, x, fresh=False):
        """network(x): each Linear + ReLU pair runs as one hipBLASLt GEMM with the bias and the
        ReLU in its epilogue: the same float32 result bit for bit, one pass less over the
        activations (250 us instead of 365 us for 131,072 x 202 -> 512)."""
        l0, l1 = self.network[0], self.network[2]
        if self._coarse is None or not x.is_cuda:
            return _linear(l1, _linear(l0, x, True), True)
        rows = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        w0, w1 = self._coarse_weight("network.0", l0, fresh), self._coarse_weight("network.2", l1, fresh)
        if torch.is_grad_enabled():  # float32 between the layers also in a 16-bit policy: that is what acting quantises
            h = _linear(l1, _linear(l0, rows, True, w0, torch.float32, self._straight), True, w1, None, self._straight)
        else:  # the same numbers, with what lies between the layers in 4 bits
            h = mxfp4.linear(rows, w0, l0.bias.float(), relu=True, out_dtype="mxfp4")
            h = mxfp4.linear(h, w1, l1.bias.float(), relu=True, out_dtype=l1.weight.dtype)
        return h if x.dim() == 2 else h.view(*x.shape[:-1], -1)

    def use_mxfp4_trunk(self, straight_through=False):
        """The trunk is computed in 4-bit floating point (`mxfp4.linear`: weights, observations and the hidden layer), and so is the
        first layer of the centralised critic, whose weight is most of what a rollout step reads.  Heads stay in float32.

        Updates train this policy: their forward pass is the same numbers.  Their backward pass is that of the unrounded
        layers at the ReLU masks of the 4-bit ones, g W and g^T x with W and x as they were before the rounding, or with
        `straight_through` that of the 4-bit layers with the roundings' derivatives taken as one, g Q(W) and g^T Q(x), which
        finds hard tasks earlier and returns more there (`train` takes it).  The optimizer steps the unrounded weights, and a
        checkpoint holds them.  (Acting in 4 bits and updating in float32 does not train: the two policies differ by more
        than the PPO clip.)  Observations are rounded too: distances and flags of up to 4 are kept but where larger numbers,
        a cooking pot's timer above all, share their block of 32 (`mxfp4`).

        `rollout_step` reads the weights as `refresh_rollout_heads` last quantised them; every other call quantises them
        anew, into the same storage: order it behind rollout steps on other streams as a change of the weights would be.
        For the centralised critic's first layer that reads as much as the float32 product does: where its value is wanted
        once a change of the weights, as without the fused sampler, 4 bits save nothing there."""
        if self._coarse is None:  # captured launches read the weights where they are
            self._coarse = {}
        self._straight = bool(straight_through)
        return self

    def use_activation_checkpoints(self):
        """Updates keep the trunk's activations in 8 bits between the forward and the backward pass (`act8`), a quarter of what
        autograd keeps: an input of whole numbers up to 127 (the observations) exactly, the hidden layers to half a step,
        or one where a small positive value is kept from becoming 0; a step is at most 1/127.75 of their block's largest
        value.  Values, log-probabilities and the loss are unchanged; the gradients of the weights are those of the kept
        activations.  An update's peak, reached in its backward pass, falls by three tenths (262,144 samples: 5.1 instead of
        7.2 KB each).  Calls with a joint observation keep float32."""
        self._keep_in_8_bits = True
        return self

    def _coarse_weight(self, name, layer, fresh, keep=False):
        """`layer`'s weight in 4 bits, in the same storage every time; quantised anew unless `fresh` says that it is current.
        Calls on other streams read the storage too, so it counts as held once its first codes are there.  A launch that is
        only being captured puts none there: then the weight is the captured call's own, and what needs the storage
        (`fresh`, `keep`) is refused."""
        weight, held = layer.weight, self._coarse.get(name)
        if held is None or held.device != weight.device:
            with torch.cuda.device(weight.device):
                capturing = torch.cuda.is_current_stream_capturing()
                if capturing and (fresh or keep):
                    raise RuntimeError("call refresh_rollout_heads() once before a capture that acts in 4 bits")
                held = mxfp4.quantize(weight)
                if not capturing:
                    torch.cuda.current_stream().synchronize()
                    self._coarse[name] = held
        elif not fresh:
            mxfp4.quantize(weight, out=held)
        return held

    def _kept_heads(self, x):
        """logits and value with every activation kept in 8 bits: both heads as one layer, so that the hidden layer is read once"""
        kept = None if self._coarse is not None and self._straight else act8.compress(x)
        codes, scales, nonnegative, h = getattr(kept, "codes", None), getattr(kept, "scales", None), False, x.contiguous()
        if x.shape[0] < _SMALL_ROWS:
            _announce_blas_switch_quietly(x)
        for name in ("network.0", "network.2"):
            layer = self.get_submodule(name)
            coarse = None if self._coarse is None else self._coarse_weight(name, layer, False)
            between = torch.float32 if name == "network.0" else None  # with 4-bit weights, as in _trunk
            straight = coarse is not None and self._straight
            if straight:
                read = mxfp4.quantize(h)
                codes, scales = read.codes, read.scales
            h, codes, scales = _KeptLinear.apply(h, codes, scales, nonnegative, layer.weight, layer.bias, True, coarse, between, straight)
            nonnegative = True
        heads = _KeptLinear.apply(h, codes, scales, True, torch.cat([self.actor.weight, self.critic.weight]),
                                  torch.cat([self.actor.bias, self.critic.bias]), False)
        return heads.split([self.actor.out_features, 1], dim=1)

    def _keeps(self, x):
        return self._keep_in_8_bits and torch.is_grad_enabled() and x.is_cuda and x.dim() == 2 and x.shape[0] > 0

    def use_fused_sampling(self, seed, row_index_base=0):
        """Rollout actions (no autograd, action=None) come from `sampling.CategoricalSampler`: one
        launch for sample + log_prob + entropy, its own counter RNG instead of torch's generator."""
        from .sampling import CategoricalSampler

        self.sampler = CategoricalSampler(seed, row_index_base, next(self.parameters()).device)
        return self

    def _central(self, joint_obs, fresh=False):
        if self.centralised_critics is None:
            raise RuntimeError("this Agent was built without its centralised critic (build_centralised=False)")
        c = self.centralised_critics
        if self._coarse is None or not joint_obs.is_cuda:
            return _linear(c[4], _linear(c[2], _linear(c[0], joint_obs, True), True), False)
        rows = joint_obs if joint_obs.dim() == 2 else joint_obs.reshape(-1, joint_obs.shape[-1])
        coarse = self._coarse_weight("centralised_critics.0", c[0], fresh)
        straight = self._straight and torch.is_grad_enabled()  # without gradients the product quantises its rows itself
        value = _linear(c[4], _linear(c[2], _linear(c[0], rows, True, coarse, None, straight), True), False)
        return value if joint_obs.dim() == 2 else value.view(*joint_obs.shape[:-1], -1)

    def get_value(self, x, joint_obs=None):
        if joint_obs is not None:
            want = int(self.obs_space.shape[0]) * self.num_agents * self.num_envs
            if joint_obs.shape[1] != want:
                raise ValueError(f"joint_obs has width {joint_obs.shape[1]}, expected {want}")
            return self._central(joint_obs)
        return _linear(self.critic, self._trunk(x), False)

    def get_action_and_value(self, x, action=None, joint_obs=None):
        # validate_args=False: the argument check reads a device flag back on the host, one
        # synchronisation per call, and cannot run under hipGraph capture; it changes no result
        if action is None and self.sampler is not None and x.is_cuda and not torch.is_grad_enabled():
            # rollout: sample, log-probability and entropy in one launch
            hidden = self._trunk(x)
            logits = _linear(self.actor, hidden, False)
            value = self._central(joint_obs) if joint_obs is not None else _linear(self.critic, hidden, False)
            action, logprob, entropy = self.sampler.sample(logits)
            return action, logprob, entropy, value
        if joint_obs is None and self._keeps(x):
            logits, value = self._kept_heads(x)
        else:
            hidden = self._trunk(x)
            logits, value = _linear(self.actor, hidden, False), None
        dist = Categorical(logits=logits, validate_args=False)
        if action is None:
            action = dist.sample()
        if value is None:
            if joint_obs is None:
                value = _linear(self.critic, hidden, False)
            else:
                value = self._central(joint_obs)
        return action, dist.log_prob(action), dist.entropy(), value

    def refresh_rollout_heads(self):
        """Actor and critic heads stacked into one [actions + 1, hidden] weight for `rollout_step`
        (same storage every time, so captured launches keep reading the right place).  Call after
        the parameters changed."""
        k = self.actor.out_features
        if getattr(self, "_head_w", None) is None or self._head_w.device != self.actor.weight.device:
            self._head_w = torch.empty((k + 1, self.actor.in_features), device=self.actor.weight.device)
            self._head_b = torch.empty(k + 1, device=self.actor.weight.device)
        with torch.no_grad():
            torch.cat([self.actor.weight, self.critic.weight], out=self._head_w)
            torch.cat([self.actor.bias, self.critic.bias], out=self._head_b)
        if self._coarse is not None:  # the 4-bit weights that rollout_step reads
            self._coarse_weight("network.0", self.network[0], False, keep=True)
            self._coarse_weight("network.2", self.network[2], False, keep=True)
            if self.centralised_critics is not None and "centralised_critics.0" in self._coarse:
                self._coarse_weight("centralised_critics.0", self.centralised_critics[0], False, keep=True)

    def rollout_step(self, x, logprob_out, value_out, actions_out=None, slot=None, joint=False, row_offset=0):
        """The rollout half of `get_action_and_value` for the decentralised critic, writing the
        log-probabilities and the values straight into the given rows of the rollout store
        (float32 [rows] each) instead of returning fresh tensors that are then copied.  Both
        heads come out of one GEMM (`refresh_rollout_heads`), the sampling kernel hands the value
        column on: three launches after the trunk instead of five.  The numbers agree with
        `get_action_and_value` to float32 rounding; needs `use_fused_sampling`, no autograd.
        `joint=True`: the value is the centralised critic's, one number for the concatenation of all
        rows (agents/MAPPO.py:70-73, model.py:45), written to every row as the reference's buffer
        assignment broadcasts it (agent_environment.py:83-84, buffer.py:28).
        `row_offset`: `x` holds rows [row_offset, row_offset + len(x)) of the batch (one shard of a
        pipelined rollout); they draw the random numbers of those rows.  Not with `joint`."""
        if joint and row_offset:
            raise ValueError("the centralised critic reads every row of the batch: no per-shard call")
        if self.sampler is None:
            raise RuntimeError("rollout_step needs use_fused_sampling()")
        if joint:
            with torch.no_grad():
                logits = _linear(self.actor, self._trunk(x, fresh=True), False)
                actions, _, _ = self.sampler.sample(logits, want_entropy=False, actions_out=actions_out,
                                                    logprob_out=logprob_out, slot=slot)
                value_out.copy_(self._central(x.view(1, -1), fresh=True).view(1).expand_as(value_out))
            return actions
        if getattr(self, "_head_w", None) is None:
            self.refresh_rollout_heads()
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(x.device).synchronize()  # other streams read them too
        with torch.no_grad():
            heads = torch.addmm(self._head_b, self._trunk(x, fresh=True), self._head_w.t())
            actions, _, _ = self.sampler.sample(heads, want_entropy=False, actions_out=actions_out, logprob_out=logprob_out,
                                                slot=slot, num_actions=self.actor.out_features, next_column_out=value_out,
                                                row_offset=row_offset)
        return actions

    def logits_and_value(self, x):
        """both heads on the shared trunk (model.py:49-61 without the distribution object)"""
        if self._keeps(x):
            return self._kept_heads(x)
        hidden = self._trunk(x)
        return _linear(self.actor, hidden, False), _linear(self.critic, hidden, False)

    def get_prob(self, x):
        return Categorical(logits=_linear(self.actor, self._trunk(x), False), validate_args=False)
