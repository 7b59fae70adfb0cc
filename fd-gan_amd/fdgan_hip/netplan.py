"""NetPlan: builds the static launch sequence of one network forward for one input
shape.  Ops are collected as closures, the shared statistics workspace is sized from
`fdgan_conv2d_fwd_info`, then everything is recorded once into an FdPlan (native
launch list / hipGraph) and replayed per step.

Train-mode BatchNorm (reference: never `.eval()`, README.md:38) is split in two:
the PRODUCER conv's epilogue emits per-workgroup (sum, sum^2) partials which
`fdgan_bn_finalize` reduces to (mean, var) per channel ONCE; every CONSUMER conv
folds (gamma, beta, mean, var) into a per-channel scale/shift in its prologue and
updates that norm's running statistics.  Inside a dense block the statistics of a
channel never change once produced, so the concat buffer is normalised without ever
being re-read by a BatchNorm kernel (SURVEY section 7 "hard parts").
"""
import torch
import torch.nn as nn

from . import engine as E
from . import lib as L


class ChanStats:
    """Per-channel batch mean / biased variance of an NHWC buffer (fp32)."""

    def __init__(self, channels, device):
        self.mean = torch.zeros(channels, dtype=torch.float32, device=device)
        self.var = torch.ones(channels, dtype=torch.float32, device=device)


class NetPlan:
    def __init__(self, device):
        self.device = device
        self.weights = []          # PackedWeight, refreshed by ONE batched pack launch per parameter update
        self.norm_params = []      # layer norms' weights and biases: the recorded launches hold their addresses
        self.flipped = {}          # id(forward PackedWeight) -> its data-gradient twin (created by the first backward)
        self._table = None
        self._ops = []             # (closure, stats_floats)
        self.ws = None             # stats partial workspace
        self.main = None
        self.packp = None
        self.keep = []             # anything that must outlive the plan
        self.grad_alias = {}       # activation buffer data_ptr -> data_ptr of the buffer whose GRADIENT buffer it shares
        self._param_versions = None
        self.records = []          # per op, in forward order: what the backward pass needs (fdgan_hip/backward.py)
        self.drops = []            # (mask buffer, channels, p) of every element-wise dropout, in plan order
        self.forced_dropout = None
        import os
        # Opt-in: the producer's last workgroup finalizes the batch statistics (86 fdgan_bn_finalize launches less per netG
        # forward).  Measured twice, slower both times.  With device-scope release / acquire fences in every workgroup (an L2
        # write-back + invalidate per XCD on MI355X): 10.7 ms per forward against 5.25.  With relaxed agent-scope atomics
        # instead of fences (csrc/conv_igemm.h: fd_finalize_last_block, what is there now): 6.4 ms against 4.84, the step 32.7
        # against 31.2 -- +33 us per conv1x1_ds launch, +8 us per conv3x3_rs launch: ONE workgroup pulling 256 rows x 128
        # channels of partials through one CU's address unit costs more than the separate 32-workgroup launch does in the
        # stream (~3 us).  Off.
        self.fuse_finalize = os.environ.get("FDGAN_FUSED_FINALIZE") is not None
        self.counter = torch.zeros(1, dtype=torch.int32, device=device)   # last-workgroup counter of the fused finalize

    # ---- registration -----------------------------------------------------------
    def weight(self, param, cout, cin, k, transposed=False, stride=1):
        w = E.PackedWeight(param, cout, cin, k, transposed, stride=stride)
        self.weights.append(w)
        return w

    def bn_prologue(self, bn, src_stats, count, act=L.ACT_RELU, pool=False):
        """Prologue of a conv whose input passes through BatchNorm `bn` (+activation)."""
        if bn.training or not bn.track_running_stats:
            assert src_stats is not None
            p = E.make_prologue(act=act, pool=pool, mean=src_stats.mean, var=src_stats.var, gamma=bn.weight,
                                beta=bn.bias, eps=bn.eps, momentum=bn.momentum if bn.momentum is not None else 0.1,
                                running_mean=bn.running_mean if bn.track_running_stats else None,
                                running_var=bn.running_var if bn.track_running_stats else None,
                                nbt=bn.num_batches_tracked if bn.track_running_stats else None, count=count)
            p._meta.update(bn=bn, stats=src_stats, batch_stats=True)
            return p
        p = E.make_prologue(act=act, pool=pool, mean=bn.running_mean, var=bn.running_var, gamma=bn.weight,
                            beta=bn.bias, eps=bn.eps)
        p._meta.update(bn=bn, stats=None, batch_stats=False)
        return p

    def conv(self, x, w, y, k, pad=0, stride=1, bias=None, pro=None, e_act=L.ACT_NONE, upsample=False,
             stats=None, stats_c0=0, y_fd=None, label=None, stats_also=()):
        """x, y: engine.View (y_fd overrides for NCHW fp32 output).  stats: ChanStats to
        receive the batch statistics of the `w.cout` stored channels at [stats_c0, ...); stats_also: further
        (ChanStats, c0) targets for the same statistics (a tensor that is concatenated into two buffers).
        With upsample the kernel sums each value once, before the replication: the count follows."""
        yfd = y_fd if y_fd is not None else y.fd
        desc = E.conv_desc(k, stride, pad, e_act, upsample, cout=w.cout, w_layout=w.layout)
        need = 0
        info = None
        if stats is not None:
            info = E.conv_info(x.fd, yfd, w.cout, desc, pro)
            need = info.stats_rows * info.stats_cpad * 2
            n, h, ww, _ = (yfd.n, yfd.h, yfd.w, yfd.c)
            count = n * h * ww // (4 if upsample else 1)

        fused = None
        if stats is not None and info.fused_finalize and self.fuse_finalize and not stats_also:
            fused = (stats.mean.data_ptr() + 4 * stats_c0, stats.var.data_ptr() + 4 * stats_c0, self.counter.data_ptr(), count)

        def run():
            E.conv2d(x.fd, w, bias, pro, yfd, desc, self.ws if stats is not None else None, fused)
            if stats is not None and fused is None:
                E.bn_finalize(self.ws, info, w.cout, count, stats.mean, stats.var, stats_c0)
                for st2, c2 in stats_also:
                    E.bn_finalize(self.ws, info, w.cout, count, st2.mean, st2.var, c2)

        pro_nofx = E.prologue_without_side_effects(pro)

        def rerun():   # the same launch without BatchNorm's running-statistics side effects (recomputation)
            E.conv2d(x.fd, w, bias, pro_nofx, yfd, desc, self.ws if stats is not None else None, fused)
            if stats is not None and fused is None:
                E.bn_finalize(self.ws, info, w.cout, count, stats.mean, stats.var, stats_c0)
        self.records.append(dict(kind="conv", x=x, w=w, y=y if y_fd is None else None, k=k, pad=pad, stride=stride, bias=bias,
                                 pro=pro_nofx, e_act=e_act, upsample=bool(upsample), rerun=rerun))
        # algorithmic work of this launch: every conv reads its input once and
        # writes its output once; MACs counted on the reference's formulation (conv before pool)
        up = 2 if upsample else 1
        ho, wo = yfd.h // up, yfd.w // up
        pool = bool(pro is not None and pro.pool2)
        macs_px = ho * wo * (4 if pool else 1)
        out_bytes = yfd.n * yfd.h * yfd.w * w.cout * (4 if yfd.dtype == L.FD_F32 else 2)
        self._ops.append((run, need, dict(
            label=label or "conv%dx%d_%d_%d" % (k, k, w.cin, w.cout), k=k, cin=w.cin, cout=w.cout,
            n=yfd.n, h_out=yfd.h, w_out=yfd.w, flops=2.0 * yfd.n * macs_px * w.cout * w.cin * k * k,
            flops_done=2.0 * yfd.n * ho * wo * w.cout * w.cin * k * k,
            bytes=x.fd.n * x.fd.h * x.fd.w * w.cin * 2 + out_bytes)))
        self.keep += [x, y, w, bias, pro, yfd, desc, stats, stats_also]

    def copy(self, src, dst):
        self._ops.append((lambda: E.copy_nhwc(src, dst), 0, dict(label="copy", flops=0.0, flops_done=0.0,
                                                                   bytes=4 * src.fd.n * src.fd.h * src.fd.w * src.c)))
        self.keep += [src, dst]
        self.records.append(dict(kind="copy", src=src, dst=dst))

    def maxpool(self, src, dst):
        self._ops.append((lambda: E.maxpool2(src, dst), 0, dict(label="maxpool", flops=0.0, flops_done=0.0,
                                                                 bytes=2 * src.fd.n * src.fd.h * src.fd.w * src.c * 5 // 4)))
        self.keep += [src, dst]
        self.records.append(dict(kind="maxpool", src=src, dst=dst))

    def layer_norm(self, src, dst, ln):
        """dst = layer norm over each pixel's channels of `src`, with module `ln` (fdgan_hip.norm.LayerNorm over the channels): a tensor of its
        own, because a pixel's mean and variance are no per-channel scale and shift that the next conv's prologue could apply.  `src` is read
        again by the reverse walk: no later op may overwrite it; other ops may read it.  A caller that puts a gradient of its own into src's
        gradient buffer (a network output) needs a second reader on record, a `copy` for one: a sole reader's gradient is stored, not added."""
        if ln.normalized_shape != (src.c,) or any(p is not None and p.dtype != torch.float32 for p in (ln.weight, ln.bias)):
            raise ValueError("layer norm over %s in %s for %d channels" % (ln.normalized_shape, None if ln.weight is None else ln.weight.dtype, src.c))
        n, h, w, c = src.shape
        stats = torch.empty((2, n * h * w), dtype=torch.float32, device=self.device)
        floats = E.layer_norm_workspace(src, False)
        ws = torch.empty(floats, dtype=torch.float32, device=self.device) if floats else None
        self._ops.append((lambda: E.layer_norm(src, ln, dst, stats, ws), 0, dict(label="layer_norm", flops=8.0 * n * h * w * c, flops_done=8.0 * n * h * w * c,
                                                                              bytes=4 * n * h * w * c)))
        self.records.append(dict(kind="layer_norm", src=src, dst=dst, ln=ln, stats=stats))
        self.norm_params += [p for p in (ln.weight, ln.bias) if p is not None]
        self.keep += [src, dst, ln, stats, ws]

    def dropout(self, view, p, up2=False):
        """F.dropout(view, p, training=True) in place (the dy blocks' dropRate > 0, /root/reference/models/dehaze1113.py:270-274,
        :367-368): a fresh element-wise mask per forward, drawn by torch into a plan-owned fp16 tensor holding 0 or 1 / (1 - p)
        (`refresh_dropout`, called by `launch`), multiplied in by one recorded launch; the reverse walk multiplies the gradient by the
        same tensor.  up2: `view` is already the nearest x2 image of the dropped tensor (TransitionBlockdy)."""
        n, h, w, c = view.shape
        f = 2 if up2 else 1
        mbuf = E.new_act(n, h // f, w // f, (c + 7) // 8 * 8, self.device, zero=True)
        mview = E.View(mbuf, 0, c)
        self.drops.append((mbuf, c, float(p)))
        self._ops.append((lambda: E.mul_mask(mview, view, up2), 0, dict(label="dropout", flops=0.0, flops_done=0.0,
                                                                      bytes=4 * n * h * w * c)))
        self.records.append(dict(kind="dropout", src=view, dst=view, mask=mview, up2=bool(up2)))
        self.keep += [view, mview]

    def refresh_dropout(self, forced=None):
        """New masks for the next launch.  forced: test hook -- a list of NCHW 0 / 1 tensors, one per dropout in plan order (what the
        oracle drew), used instead of the generator."""
        for i, (mbuf, c, p) in enumerate(self.drops):
            if forced is not None:
                m = forced[i].to(mbuf.device).permute(0, 2, 3, 1).to(mbuf.dtype)
                mbuf[..., :c].copy_(m / (1.0 - p))
            else:
                keep = torch.empty(mbuf.shape[:3] + (c,), dtype=torch.float32, device=mbuf.device).bernoulli_(1.0 - p)
                mbuf[..., :c].copy_(keep / (1.0 - p))

    def op(self, fn, record=None, need=0):
        """An arbitrary launch sequence.  record: what the reverse walk needs to know about it (fdgan_hip/backward.py: kinds
        "pyramid", "bn_dropout", "maxpool3" with `src` / `dst` views); need: floats of the shared workspace it uses."""
        self._ops.append((fn, need, dict(label="op", flops=0.0, flops_done=0.0, bytes=0)))
        if record is not None:
            self.records.append(record)

    # ---- build / run ------------------------------------------------------------------
    def finish(self):
        need = max([o[1] for o in self._ops] + [2])
        self.ws = torch.empty(need, dtype=torch.float32, device=self.device)
        self.main = E.Plan()
        self.meta = []             # one entry per op: launch index range + algorithmic work
        with self.main.record():
            for fn, _, meta in self._ops:
                first = len(self.main)
                fn()
                meta = dict(meta)
                meta["launches"] = list(range(first, len(self.main)))
                self.meta.append(meta)
        self._ops = None
        return self

    def _versions(self):
        return tuple(w.param._version for w in self.weights)

    def flipped_weight(self, w):
        """The packed filter image the DATA gradient of conv `w` runs on: flipped taps, in/out channels swapped (a
        ConvTranspose2d 1x1 stores (cin, cout) already).  Created on first use, packed with the forward images from then
        on -- once per parameter update, in the same launch."""
        t = self.flipped.get(id(w))
        if t is None:
            p = w.param.detach()
            t = E.PackedWeight(p, w.cin, w.cout, w.k, transposed=False, flip=not w.transposed, layout=L.WLAYOUT_CHUNK32, grad=True)
            t.pack()
            self.flipped[id(w)] = t
            self.keep.append(t)
            self._table = None
        return t

    def refresh_weights(self, force=False):
        v = self._versions()
        if force or v != self._param_versions:
            if self._table is None:
                self._table = E.PackTable(self.weights + list(self.flipped.values()))
            self._table.launch()
            self._param_versions = v

    def launch(self):
        self.refresh_weights()
        if self.drops:
            self.refresh_dropout(self.forced_dropout)
        self.main.launch()

    def param_ptrs(self):
        return tuple(w.param.data_ptr() for w in self.weights) + tuple(p.data_ptr() for p in self.norm_params)

    def close(self):
        """Deterministic teardown of an evicted plan: its backward walker joins and drains its side stream and
        destroys its tapes, the device finishes whatever still reads this plan's activation set (the plan may have been launched
        from more than one stream: train.py runs the discriminator on a side stream), then the recorded launches and the
        buffers go -- here, not at a random garbage collection of the cycle plan <-> PlanBackward inside later work."""
        if getattr(self, "_closed", False):
            return
        self._closed = True
        bwd = self.__dict__.pop("_bwd", None)
        if bwd is not None:
            bwd.close()
        if self.device is not None and torch.device(self.device).type == "cuda":
            try:
                torch.cuda.synchronize(self.device)
            except Exception:
                pass
        if self.main is not None:
            self.main.close()
        self.main = None
        self.records, self.keep, self.weights, self.drops = [], [], [], []
        self.flipped.clear()
        self._table = self.ws = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def bn_flags(module):
    """Cache key part: the train/eval state of every BatchNorm under `module`.  The list of norms is found once per module
    (walking 800 sub-modules per forward call was 0.4 ms of host time, four times per training step)."""
    bns = module.__dict__.get("_fd_bn_list")
    if bns is None or bns[0] != len(module._modules):
        bns = module.__dict__["_fd_bn_list"] = (len(module._modules), [m for m in module.modules() if isinstance(m, nn.modules.batchnorm._BatchNorm)])
    drops = module.__dict__.get("_fd_drop_list")
    if drops is None or drops[0] != len(module._modules):     # blocks with an F.dropout behind their convs (BottleneckBlockdy, TransitionBlockdy, ...)
        drops = module.__dict__["_fd_drop_list"] = (len(module._modules), [m for m in module.modules() if hasattr(m, "droprate")])
    #  a plan bakes `droprate > 0 and training` of those blocks in: their mode is part of the key like the norms'
    return tuple(m.training for m in bns[1]) + tuple((m.training, float(m.droprate)) for m in drops[1] if m.droprate > 0)
