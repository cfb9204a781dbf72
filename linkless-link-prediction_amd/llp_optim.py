"""AdamW over many tensors, its moments in f32 or in 8 bits (csrc/adamw.hip).

``AdamW`` is a torch.optim.Optimizer: torch.optim.AdamW's update (decoupled weight decay) in one launch
for each parameter group, ``state_bits=8`` with block-scaled moments of 8.25 bits a value, rounded
stochastically so that their means are kept (the second moment's down to its block's least code, which a
positive one never falls below).  The training engines take it in place of
torch.optim.Adam (src/main.py:400-402).  ``AdamWTable`` is the step itself over lists of tensors, in
place or into other buffers.
"""
from __future__ import annotations

import bisect

import numpy as np
import torch

import llp_hip as K


def _check(name, ts, ref, dtypes, dev):
    if len(ts) != len(ref):
        raise ValueError(f"AdamWTable: {len(ref)} params, {len(ts)} {name}")
    for t in ts:
        if t.device != dev:
            raise ValueError(f"AdamWTable: {name} on {t.device}, params on {dev}")
        if not t.is_contiguous():
            raise ValueError(f"AdamWTable: {name} must be contiguous")
        if t.dtype != ts[0].dtype or t.dtype not in dtypes:
            raise TypeError(f"AdamWTable: {name} must share one dtype of {[str(d) for d in dtypes]}")


_FLOATS = (torch.float32, torch.bfloat16)


def _pairs(counts):
    """(tensor, 0), (tensor, 1) .. up to each tensor's count as int32 pairs; counts: two runs over the tensors."""
    c = np.asarray(counts, dtype=np.int64)
    out = np.empty((int(c.sum()), 2), dtype=np.int32)
    out[:, 0] = np.repeat(np.arange(c.size) % (c.size // 2), c)
    out[:, 1] = np.arange(out.shape[0]) - np.repeat(np.cumsum(c) - c, c)
    return torch.from_numpy(out)


class AdamWTable:
    """The tensors of an AdamW step: ``params`` and ``grads`` (lists, f32 or bf16) and the moments
    ``exp_avg`` / ``exp_avg_sq``: f32 lists, or uint8 codes with ``exp_avg_scale`` /
    ``exp_avg_sq_scale`` (uint8, one per 32 elements of a tensor; ``AdamWTable.state8`` makes zero ones).

    groups     clip group (0..7) of each tensor, an index into the step's ``sumsq``
    copies     working copies of the new params (f32 or bf16; None entries: none): a tensor of the
               param's shape, or (tensor, row stride) for rows inside a wider operand
    copies_t   transposed working copies, likewise
    out        {"params", "exp_avg", "exp_avg_sq"[, "exp_avg_scale", "exp_avg_sq_scale"]}: lists to
               write instead of the inputs (default: in place); the state before the step then stays
    values     {"exp_avg", "exp_avg_sq"}: lists that ``values()`` fills with the 8-bit moments' values

    The table holds the addresses; it stays valid while the tensors keep their storage, and the
    launches of ``step`` can be captured into a graph."""

    def __init__(self, params, grads, exp_avg, exp_avg_sq, exp_avg_scale=None, exp_avg_sq_scale=None, groups=None,
                 copies=None, copies_t=None, out=None, values=None):
        if not params:
            raise ValueError("AdamWTable: no params")
        if len(params) > 65536:
            raise ValueError("AdamWTable: at most 65,536 params")
        dev = params[0].device
        _check("params", params, params, _FLOATS, dev)
        _check("grads", grads, params, _FLOATS, dev)
        self.bits = 8 if exp_avg_scale is not None else 32
        if (exp_avg_scale is None) != (exp_avg_sq_scale is None):
            raise ValueError("AdamWTable: exp_avg_scale and exp_avg_sq_scale go together")
        kinds = (torch.uint8,) if self.bits == 8 else (torch.float32,)
        ins = {"params": params, "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}
        if self.bits == 8:
            ins.update(exp_avg_scale=exp_avg_scale, exp_avg_sq_scale=exp_avg_sq_scale)
        outs = dict(ins)
        for k, v in (out or {}).items():
            if v is not None:
                if k not in ins:
                    raise ValueError(f"AdamWTable: out has no {k!r} here")
                outs[k] = v
        values = {k: v for k, v in (values or {}).items() if v is not None}
        if values and self.bits != 8:
            raise ValueError("AdamWTable: f32 moments are their values")
        for d in (ins, outs):
            for k, ts in d.items():
                _check(k, ts, params, (params[0].dtype,) if k == "params" else kinds, dev)
        self.values_dtype = None
        for k, ts in values.items():
            if k not in ("exp_avg", "exp_avg_sq"):
                raise ValueError(f"AdamWTable: values has no {k!r}")
            _check(f"values[{k!r}]", ts, params, _FLOATS, dev)
            if self.values_dtype not in (None, ts[0].dtype):
                raise TypeError("AdamWTable: values in one dtype")
            self.values_dtype = ts[0].dtype
        for i, p in enumerate(params):
            n, blocks = p.numel(), -(-p.numel() // 32)
            for d in (ins, outs, {"grads": grads}, values):
                for k, ts in d.items():
                    want = blocks if k.endswith("scale") else n
                    if ts[i].numel() != want:
                        raise ValueError(f"AdamWTable: {k}[{i}] has {ts[i].numel()} elements, {want} are needed")
        groups = [0] * len(params) if groups is None else [int(g) for g in groups]
        if len(groups) != len(params) or any(not 0 <= g < 8 for g in groups):
            raise ValueError("AdamWTable: a clip group in 0..7 for each param")
        self.n_groups = max(groups) + 1
        copies, copies_t = self._copies(copies, params, dev), self._copies(copies_t, params, dev)
        shapes = [(p.shape[0], p.shape[1]) if p.dim() == 2 else (1, p.numel()) for p in params]
        for i, (c, ct) in enumerate(zip(copies, copies_t)):
            if c[0] is not None and ct[0] is not None and c[0].dtype != ct[0].dtype:
                raise TypeError("AdamWTable: a param's copies in one dtype")
            self._fits(c, *shapes[i], i)
            self._fits(ct, *shapes[i][::-1], i)
        if not params[0].is_cuda:
            raise RuntimeError("AdamWTable runs only on the MI355X HIP device (got CPU tensors; no CPU fallback)")
        self._apart(ins, outs, grads, copies, copies_t, values)
        L = K.load()
        descs, items, tiles = [], [], []

        def at(ts, i):
            return None if ts is None else ts[i].data_ptr()

        for i, p in enumerate(params):
            rows, cols = shapes[i]
            c, ct = copies[i], copies_t[i]
            kinds = {t.dtype for t, _ in (c, ct) if t is not None}
            descs.append(K.AdamWDesc(
                p.data_ptr(), grads[i].data_ptr(), exp_avg[i].data_ptr(), exp_avg_sq[i].data_ptr(),
                at(ins.get("exp_avg_scale"), i), at(ins.get("exp_avg_sq_scale"), i), outs["params"][i].data_ptr(),
                outs["exp_avg"][i].data_ptr(), outs["exp_avg_sq"][i].data_ptr(), at(outs.get("exp_avg_scale"), i),
                at(outs.get("exp_avg_sq_scale"), i), K.ptr(c[0]), K.ptr(ct[0]),
                at(values.get("exp_avg"), i), at(values.get("exp_avg_sq"), i), p.numel(), rows, cols,
                c[1], ct[1], groups[i], K.dtype_code(kinds.pop()) if kinds else K.LLP_F32))
            items.append(L.llp_adamw_work_items(p.numel()))
            tiles.append(L.llp_adamw_copy_t_items(rows, cols) if ct[0] is not None else 0)
        self.device = dev
        self.n = len(params)
        self.param_code, self.grad_code = K.dtype_code(params[0].dtype), K.dtype_code(grads[0].dtype)
        self._descs, self._work = K.descs_to_device(descs, dev), _pairs(items + tiles).to(dev)
        self.n_work, self.n_tiles = sum(items), sum(tiles)
        self._args = (self._descs.data_ptr(), self.n, self._work.data_ptr(), self.n_work)
        self._args_t = (self._descs.data_ptr(), self._work.data_ptr() + 8 * self.n_work, self.n_tiles, self.param_code)
        self._keep, self._grads = (ins, outs, copies, copies_t, values), grads

    @staticmethod
    def state8(numel, device):
        """Zero 8-bit moments of ``numel`` elements: (codes, scales)."""
        return (torch.zeros(numel, dtype=torch.uint8, device=device),
                torch.zeros(-(-numel // 32), dtype=torch.uint8, device=device))

    @staticmethod
    def _copies(ts, params, dev):
        if ts is None:
            return [(None, 0)] * len(params)
        if len(ts) != len(params):
            raise ValueError("AdamWTable: an entry (or None) of copies for each param")
        got = []
        for t in ts:
            t, ld = t if isinstance(t, tuple) else (t, 0)
            if t is not None:
                if t.device != dev or t.dtype not in _FLOATS:
                    raise TypeError(f"AdamWTable: copies in f32 or bf16 on {dev}")
                if not ld and not t.is_contiguous():
                    raise ValueError("AdamWTable: copies contiguous, or given with their row stride")
            got.append((t, int(ld)))
        return got

    @staticmethod
    def _fits(copy, rows, cols, i):
        """A copy of [rows, cols] lies within its tensor's storage."""
        t, ld = copy
        if t is None:
            return
        if not ld and t.numel() != rows * cols:
            raise ValueError(f"AdamWTable: a copy of param {i} has {t.numel()} elements, {rows * cols} are needed")
        room = t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()
        if ld and (ld < cols or (rows - 1) * ld + cols > room):
            raise ValueError(f"AdamWTable: rows {ld} apart of a copy of param {i} ([{rows}, {cols}]) leave its storage")

    @staticmethod
    def _apart(ins, outs, grads, copies, copies_t, values):
        """What a step writes overlaps nothing else that it reads or writes but its own input in place."""
        spans, strided = [], []      # (first byte, byte past the last, written); rows of copies with a stride, likewise

        def add(t, write):
            if t.numel():
                lo = t.data_ptr()
                spans.append((lo, lo + t.numel() * t.element_size(), write))

        for k in ins:
            for a, b in zip(ins[k], outs[k]):
                if a.data_ptr() == b.data_ptr():
                    add(a, True)
                else:
                    add(a, False)
                    add(b, True)
        for t in grads:
            add(t, False)
        for ts, turned in ((copies, False), (copies_t, True)):
            for p, (t, ld) in zip(ins["params"], ts):
                if t is None:
                    continue
                rows, cols = (p.shape[0], p.shape[1]) if p.dim() == 2 else (1, p.numel())
                rows, cols = (cols, rows) if turned else (rows, cols)
                if not ld:
                    add(t, True)
                elif rows and cols:
                    strided.append((t.data_ptr(), rows, ld * t.element_size(), cols * t.element_size()))
        for ts in (values or {}).values():
            for t in ts:
                add(t, True)
        spans.sort()
        clash = ValueError("AdamWTable: a buffer that the step writes overlaps another one")
        end, wrote, ends = 0, 0, []       # the furthest ends of what was seen, read or written
        for lo, hi, write in spans:
            if lo < wrote or (write and lo < end):
                raise clash
            end = max(end, hi)
            wrote = max(wrote, hi) if write else wrote
            ends.append(end)
        # the rows of each strided copy against the pieces within its span, and against the copies before it
        strided.sort()
        before = []
        for rows in strided:
            lo, hi = rows[0], rows[0] + (rows[1] - 1) * rows[2] + rows[3]
            i = bisect.bisect_left(spans, (hi,)) - 1
            while i >= 0 and ends[i] > lo:
                if K.rows_meet(rows, (spans[i][0], 1, 1, spans[i][1] - spans[i][0])):
                    raise clash
                i -= 1
            before = [(h, r) for h, r in before if h > lo]
            if any(K.rows_meet(rows, r) for _, r in before):
                raise clash
            before.append((hi, rows))

    def step(self, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, sumsq=None, max_norm=1.0, seed=0):
        """One update, number *step + 1 (``step``: int64 device scalar, read and not advanced).  sumsq (f32,
        one per clip group; llp_grad_sumsq): gradients are taken times min(1, max_norm / (norm + 1e-6)) of
        their group.  ``seed`` keys the stochastic rounding of 8-bit moments."""
        if step.dtype != torch.int64 or step.device != self.device:
            raise TypeError(f"AdamWTable.step: step as an int64 tensor on {self.device}")
        if sumsq is not None and (sumsq.dtype != torch.float32 or sumsq.device != self.device
                                  or sumsq.numel() < self.n_groups or not sumsq.is_contiguous()):
            raise TypeError(f"AdamWTable.step: sumsq as f32[{self.n_groups}] on {self.device}")
        K.launch("llp_adamw_step", self.device, *self._args, self.bits, self.param_code, self.grad_code, K.ptr(sumsq),
                 max_norm, lr, betas[0], betas[1], eps, weight_decay, step.data_ptr(), int(seed) & 0xFFFFFFFFFFFFFFFF)
        if self.n_tiles:
            K.launch("llp_adamw_copy_t", self.device, *self._args_t)

    def values(self):
        """Fill the ``values`` lists with the values of the 8-bit moments that the last step wrote."""
        if self.values_dtype is None:
            raise RuntimeError("AdamWTable: built without values")
        K.launch("llp_adamw_values", self.device, self._args[0], self._args[2], self._args[3],
                 K.dtype_code(self.values_dtype))


def add_flags(parser):
    """--optimizer / --weight_decay / --optim_bits of the training commands."""
    parser.add_argument('--optimizer', type=str, default='adam', choices=['adam', 'adamw'])
    parser.add_argument('--weight_decay', type=float, default=0.01, help="decoupled decay of --optimizer=adamw")
    parser.add_argument('--optim_bits', type=int, default=32, choices=[32, 8],
                        help="bits of the moments of --optimizer=adamw")


def from_args(args, params):
    """The optimizer that those flags name."""
    if getattr(args, "optimizer", "adam") == "adam":
        if getattr(args, "optim_bits", 32) != 32:
            raise ValueError("--optim_bits=8 needs --optimizer=adamw")
        return torch.optim.Adam(params, lr=args.lr)
    return AdamW(params, lr=args.lr, weight_decay=args.weight_decay, state_bits=args.optim_bits)


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on the HIP step: ``lr``, ``betas``, ``eps``, ``weight_decay`` as there (no amsgrad,
    no maximize: groups and checkpoints that ask for them are refused); ``state_bits`` 32 or 8; ``seed`` of the
    8-bit moments' rounding (the engines mix it into their own; the same on every rank).

    Params in f32 or bf16 on the GPU, dense gradients of one dtype in a group.  ``state[p]`` holds
    ``step`` and exp_avg / exp_avg_sq (f32, or uint8 codes with exp_avg_scale / exp_avg_sq_scale; a NaN or
    an infinity takes the moments of its block of 32 with it).  A param without a gradient is left as it
    is; the update number is the group's, so params that step together must always have done so (refused
    else).  After a first eager step on the same gradients' storage ``step()`` can be captured into a
    graph (``zero_grad(set_to_none=False)``); a graph keeps the hyper-parameters and the state that were
    there, so ``load_state_dict`` asks for a new capture.

    The kernel works from a table of addresses, which lasts while params, gradients and state stay where
    they are.  Gradients elsewhere, as after ``zero_grad()``, take a new table and a device synchronisation, some
    0.3 ms a step: in a loop of short steps keep them (``zero_grad(set_to_none=False)``).  A student of 0.5 M
    params on 512 rows, forward, backward and step: 496 us with the gradients kept, 786 without
    (torch.optim.AdamW 694 and 645, fused 523 and 556)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("AdamW: lr, eps, weight_decay >= 0 and betas in [0, 1)")
        if state_bits not in (32, 8):
            raise ValueError("AdamW: state_bits 32 or 8")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._tables = {}      # per group: (addresses, table, device step counter, params)
        self._counters, self._captured = {}, []

    @staticmethod
    def _known(group):
        """A group asks for nothing that the step does not do."""
        for name in ("amsgrad", "maximize"):
            if group.get(name):
                raise ValueError(f"AdamW: no {name}")
        if group.get("weight_decay") and not group.get("decoupled_weight_decay", True):
            raise ValueError("AdamW: the decay is decoupled (the group's is Adam's)")

    def add_param_group(self, param_group):
        self._known(param_group)
        super().add_param_group(param_group)

    def __getstate__(self):
        self._sync_steps()
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._tables = {}
        self.__dict__.setdefault("_counters", {})
        self.__dict__.setdefault("_captured", [])

    def init_state(self, p):
        """state[p], made on first use."""
        st = self.state[p]
        if "exp_avg" not in st:
            st["step"] = torch.tensor(0.0)
            if self.state_bits == 8:
                st["exp_avg"], st["exp_avg_scale"] = AdamWTable.state8(p.numel(), p.device)
                st["exp_avg_sq"], st["exp_avg_sq_scale"] = AdamWTable.state8(p.numel(), p.device)
            else:
                st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return st

    def table(self, params, grads, **more):
        """The AdamWTable of these params with this optimizer's state."""
        sts = [self.init_state(p) for p in params]
        if self.state_bits == 8:
            more.update(exp_avg_scale=[s["exp_avg_scale"] for s in sts],
                        exp_avg_sq_scale=[s["exp_avg_sq_scale"] for s in sts])
        return AdamWTable([p.detach() for p in params], [g.detach() for g in grads], [s["exp_avg"] for s in sts],
                          [s["exp_avg_sq"] for s in sts], **more)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        moments = ("exp_avg", "exp_avg_sq") + (("exp_avg_scale", "exp_avg_sq_scale") if self.state_bits == 8 else ())
        for i, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            grads = [p.grad for p in params]
            if any(g.is_sparse for g in grads):
                raise RuntimeError("AdamW: dense gradients only")
            # all that the table took from these tensors: where they and the moments lie, types and layouts
            where = tuple((p.data_ptr(), g.data_ptr(), p.numel(), p.dtype, g.dtype, p.is_contiguous(), g.is_contiguous(),
                           *(self.init_state(p)[k].data_ptr() for k in moments))
                          for p, g in zip(params, grads))
            at = self._tables.get(i)
            capturing = params[0].is_cuda and torch.cuda.is_current_stream_capturing()
            if at is None or at[0] != where:
                if capturing:
                    raise RuntimeError("AdamW: run one eager step on these gradients before a capture")
                if at is not None:
                    self._sync_steps()
                steps = {float(self.state[p]["step"]) for p in params}
                if len(steps) != 1:
                    raise RuntimeError("AdamW: a group's params must have taken the same number of steps")
                table = self.table(params, grads)
                table._grads = None            # p.grad's: zero_grad() frees them
                ctr = self._counters.setdefault(i, torch.zeros(1, dtype=torch.int64, device=params[0].device))
                ctr.fill_(int(steps.pop()))
                at = self._tables[i] = (where, table, ctr, params)
            if capturing:
                self._captured.append((at, grads))      # a replay reads the table and these gradients
            _, table, ctr, _ = at
            table.step(ctr, lr=float(group["lr"]), betas=group["betas"], eps=float(group["eps"]),
                       weight_decay=float(group["weight_decay"]), seed=self.seed + (i << 48))
            K.launch("llp_increment", ctr.device, ctr.data_ptr())
            # written in place, as autograd has to know: a backward through what was saved of them raises
            torch.autograd.graph.increment_version(params)
        return loss

    def hand_over(self):
        """state[p]["step"] brought up to date, for whoever takes over the state's tensors (the training
        engines); a later ``step`` continues from what state[p]["step"] then holds."""
        self._sync_steps()
        self._tables = {}

    def _sync_steps(self):
        for _, _, ctr, params in self._tables.values():
            n = float(ctr.item())
            for p in params:
                self.state[p]["step"] = torch.tensor(n)

    def state_dict(self):
        self._sync_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        # (all looked at before anything is taken over)
        for group in state_dict["param_groups"]:
            self._known(group)
        for st in state_dict["state"].values():
            if "exp_avg" in st and ("exp_avg_scale" in st) != (self.state_bits == 8):
                raise ValueError(f"AdamW: the loaded moments are not in {self.state_bits} bits")
        super().load_state_dict(state_dict)
        self._tables = {}
        # the base class casts state to the param's dtype: the moments are taken over as they are
        order = [p for g in self.param_groups for p in g["params"]]
        ids = [k for g in state_dict["param_groups"] for k in g["params"]]
        for k, p in zip(ids, order):
            if k in state_dict["state"]:
                for name, v in state_dict["state"][k].items():
                    self.state[p][name] = v.detach().clone() if name == "step" else v.detach().clone().to(p.device)
                if self.state_bits == 8 and "exp_avg" in self.state[p]:
                    # a second moment of 0 beside a first one that is not, as a step does not leave them: its least code
                    m, r = self.state[p]["exp_avg"], self.state[p]["exp_avg_sq"]
                    r[(r == 0) & ((m & 127) != 0)] = 1
