"""Adam on flat buffers (cpfn_adam_flat): the optimizer of the training step as one streaming kernel.

`FlatAdam` is a torch.optim.Optimizer with torch.optim.Adam's arithmetic and hyper-parameters (the reference
builds `optim.Adam(spfn_module.parameters(), lr=...)`, training_SPFN.py; torch/optim/adam.py).  It re-points
every parameter at a view of ONE contiguous fp32 buffer and reads the gradients from the trainer's
FlatGradBucket, so a step is a single launch over 1.4 M elements instead of a multi-tensor launch over ~100
tensors.  Capturable: learning rate, step count and `found_inf` (set it before `step()` to skip on non-finite
gradients) are device scalars.  GPU only — on CPU the trainer keeps torch.optim.Adam.

`grad_norm`, `clip_grads_` and `clip_grad_norm_` take any list of gradients (csrc/gradnorm.hip): the norm over all of them and their
clipping: two launches for up to 130 tensors of together a few million values, three where they are more; `FlatAdam.step(max_grad_norm=...)` clips what it reads from the flat buffer."""
import torch

from . import lib as _l
from .ops import _native_call, _ptr, _stream

_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}


def _list_of(grads):
    return [grads] if isinstance(grads, torch.Tensor) else list(grads)


def _norm_code(norm_type):
    p = _NORMS.get(norm_type)
    if p is None:
        raise RuntimeError("norm_type must be 1, 2 or inf (got %r)" % (norm_type,))
    return p


def grad_norm(grads, norm_type=2.0):
    """The norm over all values of a list of tensors (fp32, bf16 and fp16 together; any lengths; dense, in any order of their dimensions,
    on one device) -> 0-dim fp32 tensor on that device, without a host synchronisation.  norm_type 1, 2 or inf; fp64 sums in a fixed order
    (bit-reproducible); NaN if any value is NaN.  An empty list: a zero on the CPU.
    A value, not a differentiable function (no gradient penalty): of tensors that autograd follows (gradients of create_graph=True,
    parameters) the result requires a gradient and raises where one is asked of it; under torch.no_grad() it is a plain tensor.
    Forward-mode tangents are refused."""
    return _native_call("grad_norm", _list_of(grads), _norm_code(norm_type), None, None)


def clip_grads_(grads, max_norm, norm_type=2.0, out=None):
    """grads *= min(1, max_norm / (norm + 1e-6)) with the norm of grad_norm -> that norm (before clipping, on the device).  Nothing is
    synchronised, and in place nothing is written where the factor is 1.  out: tensors of the same shapes, of the gradients' types or
    fp32 (master gradients), that take the result instead; a gradient listed twice, or memory shared with a tensor that is written, is
    refused.  It works on values, as under torch.no_grad(), whatever autograd follows; forward-mode tangents are refused.  An infinite norm
    gives the factor 0 and a NaN one NaN, as the formula has it."""
    return _native_call("grad_norm", _list_of(grads), _norm_code(norm_type), float(max_norm), None if out is None else _list_of(out))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ on clip_grads_: clips the .grad of the parameters that have one, in place -> their norm before.
    error_if_nonfinite reads the norm on the host first (a synchronisation and another pass over the gradients; not inside a capture) and
    raises before anything is scaled."""
    grads = [p.grad for p in _list_of(parameters) if p.grad is not None]
    if error_if_nonfinite and grads:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("error_if_nonfinite reads the norm on the host: not inside a stream capture")
        with torch.no_grad():
            norm = float(grad_norm(grads, norm_type))
        if not norm < float("inf"):
            raise RuntimeError("the norm of the gradients is %r: not clipped" % norm)
    return clip_grads_(grads, max_norm, norm_type)


class FlatAdam(torch.optim.Optimizer):
    def __init__(self, bucket, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        params = list(bucket.params)
        dev = bucket.flat.device
        if not bucket.flat.is_cuda:
            raise RuntimeError("FlatAdam runs on the GPU only (CPU not supported)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.bucket = bucket
        n = bucket.flat.numel()
        self.flat_p = torch.empty(n, dtype=torch.float32, device=dev)
        off = 0
        with torch.no_grad():
            for p in params:
                if p.dtype != torch.float32:
                    raise RuntimeError("FlatAdam expects fp32 master parameters")
                k = p.numel()
                view = self.flat_p[off:off + k].view_as(p)
                view.copy_(p.data)
                p.data = view                      # same nn.Parameter object, storage inside the flat buffer
                off += k
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)
        self.step_count = torch.zeros((), dtype=torch.float32, device=dev)
        self.lr_dev = torch.zeros((), dtype=torch.float32, device=dev)
        self._coef = torch.zeros(4, dtype=torch.float32, device=dev)
        self.beta_pows = torch.ones(2, dtype=torch.float64, device=dev)      # beta1^step, beta2^step
        self._lr_host = None
        self.found_inf = None
        self._nf_ws = None
        self.grad_norm = torch.zeros((), dtype=torch.float32, device=dev)     # before clipping, of the last step(max_grad_norm=...)
        self._parts = torch.empty(max(1, _l.lib().cpfn_grad_sumsq_blocks(n)), dtype=torch.float64, device=dev)
        g = self.param_groups[0]
        g["lr"] = self.lr_dev                      # the trainer's staircase does `group['lr'].fill_(lr)`
        self.lr_dev.fill_(float(lr))

    @torch.no_grad()
    def step(self, closure=None, check_gradients=False, skipped=None, nf_flags=None, combine=None, max_grad_norm=None):
        """check_gradients: scan the flat gradient for NaN / inf in the same launch sequence and skip the step if any
        is found (the reference's per-parameter isinf/isnan scan, Utils/training_utils.py:151-156) — the scan's final
        reduction and the optional `skipped` device counter (+1 per skipped step) live in the 1-wave prepare kernel.
        nf_flags = (int32 flags tensor, count[, n_sticky]): per-workgroup flags of a scan that already happened (the checked packing
        copy of FlatGradBucket.collect); the step is skipped if any of them is set.  The first n_sticky words are OR-ed into by
        the launches that wrote the gradients (fused_mlp.GradSink) and are cleared by this step's prepare kernel.
        combine = (S [7 C], coef [3, C], C, out [C, 3] — a slice of the flat gradient): the pass's last gradient, finished (and
        checked) by the prepare kernel (fused_mlp.GradSink.combine, cpfn_adam_flat_xw).
        max_grad_norm: step on the gradients times min(1, max_grad_norm / (norm + 1e-6)), norm = the 2-norm over the whole bucket (left in
        `self.grad_norm`, a 0-dim device tensor); the factor is applied as the step reads the gradients, which stay as they are in the
        bucket.  A norm that is not finite skips the step like check_gradients does.  Not together with `combine` (that gradient is not
        finished when the norm is taken)."""
        if max_grad_norm is not None:
            max_grad_norm = float(max_grad_norm)
            if not max_grad_norm >= 0.0:
                raise RuntimeError("max_grad_norm must not be negative (got %r)" % max_grad_norm)
            if combine is not None:
                raise RuntimeError("max_grad_norm needs finished gradients: not together with combine")
        g = self.param_groups[0]
        lr = g["lr"]
        if not isinstance(lr, torch.Tensor):       # someone assigned a float: mirror it into the device scalar
            if lr != self._lr_host:
                self.lr_dev.fill_(float(lr))
                self._lr_host = lr
            lr = self.lr_dev
        b1, b2 = g["betas"]
        h = _l.lib()
        grads = self.bucket.flat
        with torch.cuda.device(self.flat_p.device):
            nf_ws, nf_count, n_sticky = None, 0, 0
            if nf_flags is not None:
                nf_ws, nf_count = nf_flags[0], nf_flags[1]
                n_sticky = nf_flags[2] if len(nf_flags) > 2 else 0       # words OR-ed into by the gradients' writers: cleared here
            elif check_gradients and max_grad_norm is None:
                if self._nf_ws is None:
                    self._nf_ws = torch.empty(256, dtype=torch.int32, device=self.flat_p.device)
                nf_ws, nf_count = self._nf_ws, h.cpfn_nonfinite_blocks(grads.numel())
                _l.check(h.cpfn_nonfinite_partial(_ptr(grads), grads.numel(), _ptr(nf_ws), _stream()), "cpfn_nonfinite_partial")
            if max_grad_norm is not None:
                _l.check(h.cpfn_adam_flat_clip(_ptr(self.flat_p), _ptr(grads), _ptr(self.exp_avg), _ptr(self.exp_avg_sq),
                                               self.flat_p.numel(), _ptr(lr), float(b1), float(b2), float(g["eps"]),
                                               float(g["weight_decay"]), _ptr(self.step_count), _ptr(self.beta_pows),
                                               _ptr(self.found_inf), _ptr(self._coef), _ptr(nf_ws), nf_count, n_sticky, _ptr(skipped),
                                               max_grad_norm, _ptr(self._parts), _ptr(self.grad_norm), _stream()), "cpfn_adam_flat_clip")
                _l.add_bytes("cpfn_adam_flat_clip", 32 * self.flat_p.numel())
                return
            xS, xc, xC, xo = combine if combine is not None else (None, None, 0, None)
            _l.check(h.cpfn_adam_flat_xw(_ptr(self.flat_p), _ptr(grads), _ptr(self.exp_avg), _ptr(self.exp_avg_sq),
                                         self.flat_p.numel(), _ptr(lr), float(b1), float(b2), float(g["eps"]),
                                         float(g["weight_decay"]), _ptr(self.step_count), _ptr(self.beta_pows),
                                         _ptr(self.found_inf), _ptr(self._coef), _ptr(nf_ws), nf_count, n_sticky, _ptr(skipped),
                                         _ptr(xS), _ptr(xc), int(xC), _ptr(xo), _stream()), "cpfn_adam_flat")
        _l.add_bytes("cpfn_adam_flat", 28 * self.flat_p.numel() + (4 * grads.numel() if check_gradients and nf_flags is None else 0))

    def state_dict(self):
        return {"flat": {"exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "step": self.step_count,
                         "beta_pows": self.beta_pows},
                "hyper": {k: (float(v) if isinstance(v, torch.Tensor) else v) for k, v in self.param_groups[0].items()
                          if k != "params"}}

    def load_state_dict(self, sd):
        self.exp_avg.copy_(sd["flat"]["exp_avg"])
        self.exp_avg_sq.copy_(sd["flat"]["exp_avg_sq"])
        self.step_count.copy_(sd["flat"]["step"])
        self.beta_pows.copy_(sd["flat"]["beta_pows"])
        for k, v in sd.get("hyper", {}).items():
            if k == "lr":
                self.lr_dev.fill_(float(v))
            else:
                self.param_groups[0][k] = v
