"""Mixed-precision Adam with the reference's `CPUAdam` interface (axonn/optim.py), and AdamW
with moments in 32 or in 8 bits over the same buffers.

The reference keeps fp32 master weights and Adam moments in pinned host memory
and streams them through four GPU staging buffers in 16 M-element buckets,
issuing per bucket two PCIe copies each way, about ten elementwise kernels and a
host synchronisation (optim.py:138-193).  An MI355X holds 288 GB of HBM, so here
the fp32 master weights, both moments, the low-precision weights and the
low-precision gradients all stay resident in flat HBM buffers
(axonn/utils.py:11-30 layout) and one step is two kernels:

  scan   reads the gradients once: overflow flag, sum of squares, clip coefficient
  adam   reads g, p, m, v and writes p, m, v and the low-precision p once,
         skipping every write on the device when the scan saw an overflow

`bucket_size` and `coalescing_factor` are accepted for compatibility and have no
effect.  Behaviour that follows the live training engine rather than this legacy
class (axonn/inter_layer.py:426-432): the step counter advances once per applied
step (the reference advances it twice on torch >= 1.12 and also for skipped
buckets) and an overflow skips the whole step, not single buckets.
"""

import torch
from torch.optim.optimizer import Optimizer

from . import _native as nv
from . import ops
from .inter_layer import LossScaler, sync_scale
from .utils import _coalesce_and_reassign


class CPUAdam(Optimizer):
    """Adam over flat HBM-resident buffers with fp32 master weights.

    `params` are the model's (low-precision or fp32) parameters.  On
    construction they are packed into one flat buffer per param group (their
    `.data` is re-pointed, as the reference's registration step does), an fp32
    master copy and zeroed moments are created, and a flat gradient buffer is
    installed as the parameters' `.grad`, so backward accumulates straight into
    it.

    Extra keyword arguments over the reference: `max_grad_norm` (clip the global
    2-norm inside the step; None = no clipping), `loss_scaler` (a LossScaler;
    default: dynamic scaling for fp16 parameters, scale 1 otherwise) and
    `dynamic_loss_scale` (force the state machine on or off).
    """

    def __init__(
        self,
        params,
        lr=1e-3,
        betas=(0.9, 0.999),
        eps=1e-8,
        weight_decay=0,
        bucket_size=16000000,
        coalescing_factor=4,
        max_grad_norm=None,
        loss_scaler=None,
        dynamic_loss_scale=None,
    ):
        if not 0.0 <= lr:
            raise ValueError("Invalid learning rate: {}".format(lr))
        if not 0.0 <= eps:
            raise ValueError("Invalid epsilon value: {}".format(eps))
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError("Invalid beta parameter at index 0: {}".format(betas[0]))
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError("Invalid beta parameter at index 1: {}".format(betas[1]))
        if not 0.0 <= weight_decay:
            raise ValueError("Invalid weight_decay value: {}".format(weight_decay))
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)

        self.bucket_size = bucket_size
        self.coalescing_factor = coalescing_factor
        self.max_grad_norm = max_grad_norm

        super(CPUAdam, self).__init__(params, defaults)

        self.calculate_group_offsets()
        self._build_flat_buffers()

        lowp = self._lowp_dtype
        if dynamic_loss_scale is None:
            dynamic_loss_scale = lowp == torch.float16
        self.dynamic_loss_scale = dynamic_loss_scale
        if loss_scaler is None:
            loss_scaler = LossScaler() if dynamic_loss_scale else LossScaler(loss_scale=1.0)
        self.scaler = loss_scaler
        self.step_count = 0
        self.last_step_skipped = False
        self._scan = None

    def __setstate__(self, state):
        super(CPUAdam, self).__setstate__(state)
        for group in self.param_groups:
            group.setdefault("amsgrad", False)

    # -- layout -------------------------------------------------------------
    _span = None   # elements that a parameter of so many takes in the flat buffers (None: as many)

    def _room(self, n):
        return n if self._span is None else self._span(n)

    def calculate_group_offsets(self):
        """Cumulative element counts of the param groups (optim.py:59-65)."""
        self.group_offsets = [0] * (len(self.param_groups) + 1)
        for i in range(1, len(self.group_offsets)):
            group_num_params = 0
            for param in self.param_groups[i - 1]["params"]:
                group_num_params += self._room(param.nelement())
            self.group_offsets[i] = self.group_offsets[i - 1] + group_num_params

    def _build_flat_buffers(self):
        all_params = [p for g in self.param_groups for p in g["params"]]
        if len(all_params) == 0:
            raise ValueError("optimizer got an empty parameter list")
        dtypes = {p.dtype for p in all_params}
        if len(dtypes) != 1:
            raise TypeError("all parameters must share one dtype, got %s" % sorted(map(str, dtypes)))
        self._lowp_dtype = all_params[0].dtype
        if self._lowp_dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise TypeError("parameters must be bf16, fp16 or fp32")
        device = all_params[0].device
        if device.type != "cuda":
            raise RuntimeError("CPUAdam's kernels run on the GPU; move the model to the GPU first")
        with torch.no_grad():
            # flat low-precision weights; every p.data becomes a view into it
            self.model_params_fp16 = _coalesce_and_reassign(all_params, self._span)
            total = self.model_params_fp16.numel()
            if self._lowp_dtype == torch.float32:
                # fp32 model: the model weights are the master weights
                self.model_params_fp32 = self.model_params_fp16
            else:
                self.model_params_fp32 = self.model_params_fp16.float()
            self.model_grads_fp16 = torch.zeros(total, dtype=self._lowp_dtype, device=device)
            self._make_moments(total, device)
            offset = 0
            self._views = []
            self._params = all_params
            self._grad_views = []   # flat 1-D views, one per parameter: what the scan walks
            self._linked = []       # the `.grad` tensors installed here, one per parameter
            for p in all_params:
                n = p.numel()
                flat_view = self.model_grads_fp16[offset:offset + n]
                p.grad = flat_view.view(p.shape)
                self._linked.append(p.grad)
                self._views.append((offset, n))
                if n:
                    self._grad_views.append(flat_view)
                offset += self._room(n)
        self._writes_lowp = self._lowp_dtype != torch.float32

    def _make_moments(self, total, device):
        self.exp_avg = torch.zeros(total, dtype=torch.float32, device=device)
        self.exp_avg_sq = torch.zeros(total, dtype=torch.float32, device=device)

    def empty_param_state(self, param):
        """Zeroed Adam state for a slice (optim.py:67-78); states live in HBM."""
        return {
            "step": torch.tensor(0),
            "exp_avg": torch.zeros_like(param, memory_format=torch.preserve_format),
            "exp_avg_sq": torch.zeros_like(param, memory_format=torch.preserve_format),
        }

    def zero_grad(self, set_to_none=False):
        """Zeroes the flat gradient buffer (optim.py:80-81).  Gradients are never
        set to None: they are views into the buffer the step reads."""
        self.model_grads_fp16.zero_()

    # -- step -----------------------------------------------------------------
    @property
    def loss_scale(self):
        return self.scaler.loss_scale

    def _group_slices(self, group_no):
        lo, hi = self.group_offsets[group_no], self.group_offsets[group_no + 1]
        return lo, hi

    def _parts(self, lo, hi, *flats):
        """One-element lists of the flat buffers' elements lo to hi."""
        whole = hi - lo == self.model_grads_fp16.numel()   # one group: the buffers themselves
        return [[t if whole else t[lo:hi]] for t in flats]

    def _update(self, group_no, t, lo, hi, inv_scale, scan):
        """Step number t of one param group, elements lo to hi of the flat buffers."""
        group = self.param_groups[group_no]
        hp = ops.adam_hparams(t, group["lr"], *group["betas"], group["eps"], group["weight_decay"])
        g, p, m, v, low = self._parts(lo, hi, self.model_grads_fp16, self.model_params_fp32, self.exp_avg,
                                      self.exp_avg_sq, self.model_params_fp16)
        ops.mt_adam(g, p, m, v, low if self._writes_lowp else None, hp, inv_scale=inv_scale, scan=scan)

    def _relink_gradients(self):
        """The step reads the flat gradient buffer; a parameter's `.grad` is a view into
        it.  Code that rebinds `.grad` (`model.zero_grad()` sets it to None by default, a
        cast makes a new tensor) breaks that link without an error: backward would then
        write elsewhere and the step would apply zeros.  A gradient that has moved is
        copied into its slice and the view is installed again; a missing one counts as
        zero: the step runs over the whole flat buffer, as the reference's does
        (axonn/optim.py:157-190), so momentum and weight decay still move that parameter."""
        flat = self.model_grads_fp16
        base, esz = flat.data_ptr(), flat.element_size()
        for i, (p, (offset, n)) in enumerate(zip(self._params, self._views)):
            g = p.grad
            if g is self._linked[i]:   # the view installed by this class: nothing was rebound
                continue
            if g is not None and g.data_ptr() == base + offset * esz and g.numel() == n \
                    and g.dtype == flat.dtype and g.is_contiguous():
                continue
            view = flat[offset:offset + n].view(p.shape)
            if g is None:
                view.zero_()
            else:
                if g.numel() != n:
                    raise RuntimeError("a parameter's gradient changed its size (%d -> %d elements)"
                                       % (n, g.numel()))
                view.copy_(g)
            p.grad = view
            self._linked[i] = p.grad

    @torch.no_grad()
    def step(self, closure=None):
        assert closure is None, "AxoNN CPUAdam does not support closure yet"
        self._relink_gradients()
        inv_scale = 1.0 / self.scaler.loss_scale
        max_norm = float(self.max_grad_norm) if self.max_grad_norm else 0.0
        need_scan = self.dynamic_loss_scale or max_norm > 0.0
        scan = None
        if need_scan:
            # The overflow test is the reference's, per parameter: a tensor's sum, in
            # the gradient dtype, is inf or nan (axonn/inter_layer.py:447-460 walks the
            # parameters; the legacy class walks 16 M-element buckets,
            # axonn/optim.py:158-161).  One sum over the whole flat buffer would trip on
            # fp16 as soon as all scaled gradients together sum past 65504.
            scan = ops.mt_scan(self._grad_views, inv_scale, max_norm, result=self._scan)
            self._scan = scan
        t = self.step_count + 1
        for group_no, group in enumerate(self.param_groups):
            lo, hi = self._group_slices(group_no)
            if hi == lo:
                continue
            self._update(group_no, t, lo, hi, inv_scale, scan)
        skipped = False
        if scan is not None:
            skipped = bool(scan.found_inf.item())  # one 4-byte read back per step
        if self.dynamic_loss_scale:
            sync_scale(self.scaler, skipped)
        if not skipped:
            self.step_count = t
        self.last_step_skipped = skipped
        return None

    def grad_norm(self):
        """Global 2-norm of the unscaled gradients seen by the last step (a
        0-dim device tensor), when the step scanned them."""
        return None if self._scan is None else self._scan.total_norm.clone()


class AdamW(CPUAdam):
    """Adam whose weight decay acts on the weights themselves, p <- (1 - lr weight_decay) p before
    the step, over the same flat buffers, with the same loss scaling, clipping and skipped steps.

    `state_bits`: 32 keeps the moments in fp32 (`exp_avg`, `exp_avg_sq`), 8 keeps them as codes of
    8 bits with an exponent byte for each 256 elements and moment (`codes`, `exponents`; 2 bytes an
    element instead of 8).  Codes are rounded stochastically, `seed` and the step's number make the
    random words: runs with equal seeds are equal bit by bit.  Every parameter then starts at a
    whole block, so `model_params_fp32` and its like have zeros between the parameters.

    `state_dict()` holds all that the next step depends on, so that a run goes on bit by bit where it
    was saved; its tensors are the optimizer's own, as torch's are."""

    def __init__(
        self,
        params,
        lr=1e-3,
        betas=(0.9, 0.999),
        eps=1e-8,
        weight_decay=1e-2,
        max_grad_norm=None,
        loss_scaler=None,
        dynamic_loss_scale=None,
        state_bits=32,
        seed=0,
    ):
        if state_bits not in (8, 32):
            raise ValueError("Invalid number of bits of the moments: {}".format(state_bits))
        self.state_bits, self.seed = state_bits, int(seed)
        if state_bits == 8:
            self._span = lambda n: -(-n // nv.ADAMW8_BLOCK) * nv.ADAMW8_BLOCK
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_grad_norm=max_grad_norm,
                         loss_scaler=loss_scaler, dynamic_loss_scale=dynamic_loss_scale)

    def _check_eps(self, eps):
        if self.state_bits == 8 and not eps > 0.0:
            raise ValueError("8-bit moments need a positive epsilon, got {}".format(eps))

    def add_param_group(self, param_group):   # (torch's constructor adds every group by it)
        if isinstance(param_group, dict):     # (anything else torch refuses)
            self._check_eps(param_group.get("eps", self.defaults["eps"]))
        super().add_param_group(param_group)

    def _make_moments(self, total, device):
        if self.state_bits == 8:
            self.codes, self.exponents = ops.adamw8_state(total, device)
        else:
            super()._make_moments(total, device)

    def _step_seed(self, t, group_no):
        odd = 0x9E3779B97F4A7C15
        return ((self.seed * odd + t) * odd + group_no) * odd % (1 << 64)

    def _update(self, group_no, t, lo, hi, inv_scale, scan):
        group = self.param_groups[group_no]
        hp = ops.adamw_hparams(t, group["lr"], *group["betas"], group["eps"], group["weight_decay"])
        g, p, low = self._parts(lo, hi, self.model_grads_fp16, self.model_params_fp32, self.model_params_fp16)
        low = low if self._writes_lowp else None
        if self.state_bits == 8:
            first, last = lo // nv.ADAMW8_BLOCK, hi // nv.ADAMW8_BLOCK
            ops.mt_adamw8(g, p, [self.codes[first:last]], [self.exponents[first:last]], low, hp,
                          self._step_seed(t, group_no), inv_scale=inv_scale, scan=scan)
        else:
            m, v = self._parts(lo, hi, self.exp_avg, self.exp_avg_sq)
            ops.mt_adamw(g, p, m, v, low, hp, inv_scale=inv_scale, scan=scan)

    # -- saved states -------------------------------------------------------
    def _saved_tensors(self):
        return ["model_params_fp32"] + (["exp_avg", "exp_avg_sq"] if self.state_bits == 32 else ["codes", "exponents"])

    def state_dict(self):
        """torch's, whose param groups have no state of their own, and "flat": the fp32 weights, the
        moments or their codes, the step's number, the seed and the loss scale."""
        state = super().state_dict()
        state["flat"] = {
            "state_bits": self.state_bits,
            "sizes": [[p.numel() for p in group["params"]] for group in self.param_groups],
            "step_count": self.step_count,
            "seed": self.seed,
            "scaler": {field: getattr(self.scaler, field) for field in LossScaler.__dataclass_fields__},
            **{name: getattr(self, name) for name in self._saved_tensors()},
        }
        return state

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes the state in place: the weights of the model are then those of the saved fp32 weights.
        One of other sizes or another `state_bits`, or without moments, is refused as a whole."""
        flat = state_dict.get("flat")
        if flat is None:
            raise ValueError("AdamW: the saved state holds neither moments nor weights")
        if flat["state_bits"] != self.state_bits:
            raise ValueError("AdamW: the saved moments have %s bits, this optimizer's %d" % (flat["state_bits"], self.state_bits))
        if flat["sizes"] != [[p.numel() for p in group["params"]] for group in self.param_groups]:
            raise ValueError("AdamW: the saved state is that of parameters of other sizes, or in other groups")
        for name in self._saved_tensors():
            saved, mine = flat[name], getattr(self, name)
            if saved.shape != mine.shape or saved.dtype != mine.dtype:
                raise ValueError("AdamW: saved %s is %s %s, expected %s %s" % (name, saved.dtype, tuple(saved.shape), mine.dtype,
                                                                              tuple(mine.shape)))
        for group in state_dict["param_groups"]:
            self._check_eps(group["eps"])
        super().load_state_dict({name: value for name, value in state_dict.items() if name != "flat"})
        for name in self._saved_tensors():
            getattr(self, name).copy_(flat[name])
        if self._writes_lowp:
            self.model_params_fp16.copy_(self.model_params_fp32)   # (rounded as the step does)
        self.step_count, self.seed = flat["step_count"], flat["seed"]
        for field, value in flat["scaler"].items():
            setattr(self.scaler, field, value)

    def moments(self):
        """(exp_avg, exp_avg_sq) of every parameter, in fp32 and its shape: with 32 bits views of the
        flat buffers, with 8 bits what the codes stand for now."""
        m, v = (self.exp_avg, self.exp_avg_sq) if self.state_bits == 32 else ops.adamw8_moments(self.codes, self.exponents)
        return [(m[offset:offset + n].view(p.shape), v[offset:offset + n].view(p.shape))
                for p, (offset, n) in zip(self._params, self._views)]
