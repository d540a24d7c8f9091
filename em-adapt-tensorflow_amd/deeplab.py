"""``ADAPT``: the EM-Adapt DeepLab trainer with the reference's class surface (deeplab.py:12-285),
executing on MI355X through libemadapt_hip.so.

What the reference expresses as TF graph nodes is a static plan here:

  create_network / build_block / build_fc   (deeplab.py:35-107)  -> list of fused ops
        conv + bias + relu (+ dropout) = ONE implicit-GEMM launch with a fused epilogue
  e_step                                    (deeplab.py:109-124) -> resize_nearest + device E-step kernel
  getloss                                   (deeplab.py:180-186) -> fused softmax-CE fwd+bwd (+ L2 on demand)
  optimize / pre_train                      (deeplab.py:188-208, network.py:91-102)
        -> hand-written backward (dgrad / wgrad / pool-grad kernels), accumulate, Momentum
  train inner loop                          (deeplab.py:265-270) -> micro_step() / apply_update()

Memory layout (sized for 288 GB HBM: everything stays resident, nothing is recomputed):
  * all 32 parameter tensors live in ONE flat fp32 buffer, ordered fc8 .. conv1_1 (the order in which
    backward produces their gradients), with twin flat buffers for gradients, accumulators and momentum;
    the optimiser is one launch over the flat buffer and data-parallel buckets are contiguous slices;
  * conv1_1's 3 input channels are zero-padded to 4 and fc8's C classes to a multiple of 4 inside the
    buffers so every kernel moves 16-byte vectors; ``weights[layer]`` exposes the reference-shaped views;
  * activations are NHWC fp32, kept for backward (post-ReLU/dropout output of every conv, pool outputs and
    a uint8 arg-max tap per pool output).
"""
import os
import random
import time

import numpy as np
import torch

from . import ops
from .data import dist_rank_world
from .estep import draw_perms
from .network import Network, round_up

_ALIGN = 64  # floats: every layer segment of the flat buffers starts on a 256-byte boundary


class _Op:
    __slots__ = ("name", "kind", "out_name", "k", "rate", "relu", "drop", "cin", "cout", "cin_p", "cout_p",
                 "stride", "in_hw", "out_hw", "seg", "w_pad", "b_pad", "gw_pad", "gb_pad", "index")

    def __init__(self, **kw):
        for s in self.__slots__:
            setattr(self, s, None)
        for k, v in kw.items():
            setattr(self, k, v)


class ADAPT(Network):
    def __init__(self, config):
        Network.__init__(self, config)
        self.stride = {}
        self.stride["input"] = 1
        # different lr for different variable -- kept for surface parity; the reference never applies
        # them (the loop at deeplab.py:194-200 rebinds a local), so neither do we.
        self.lr_1_list = []
        self.lr_2_list = []
        self.lr_10_list = []
        self.lr_20_list = []
        # build-time knobs beyond the reference's config keys
        self.preset = self.config.get("preset", "ref")          # "ref": fc6 4x4 rate 4 (deeplab.py:92,145); "largefov": 3x3 rate 12
        self.width = int(self.config.get("width", 64))          # channel multiplier (64 in the reference)
        fcw = self.config.get("fc_width", None)
        self.fc_width = int(fcw) if fcw is not None else (4096 if self.preset == "ref" else 1024) * self.width // 64
        self.seed = int(self.config.get("seed", 2))
        self.input_channel = int(self.config.get("input_channel", 3))
        # "fp32" (reference numerics, BASELINE configs C1/C2/C5) or "bf16" (C3/C4: bf16 MFMA operands, fp32 accumulation,
        # fp32 master weights / gradients / optimizer state)
        self.compute_dtype = str(self.config.get("compute_dtype", "fp32"))
        # "bf16x6": fp32-grade results on the bf16 matrix pipe (exact 3-way split, six products; all tensors f32)
        if self.compute_dtype not in ("fp32", "bf16", "bf16x6"):
            raise ValueError("compute_dtype must be 'fp32', 'bf16' or 'bf16x6', got %r" % self.compute_dtype)
        # storage type of activations / activation gradients: defaults to the compute type.  bf16 storage holds the very
        # values the bf16 kernels would round an f32 tensor to, at half the bytes (include/emadapt.h "Storage types");
        # the input image, the fc8 logits (E-step / loss input), weights, gradients and optimizer state stay f32.
        act = str(self.config.get("act_dtype", "bf16" if self.compute_dtype == "bf16" else "fp32"))
        if act not in ("fp32", "bf16") or (act == "bf16" and self.compute_dtype != "bf16"):
            raise ValueError("act_dtype must be 'fp32', or 'bf16' together with compute_dtype 'bf16'")
        self.act_dtype = torch.bfloat16 if act == "bf16" else torch.float32
        self._cpad = 8 if act == "bf16" else 4   # channel padding of the buffers (16-byte vectors)
        self._w16_seen = None
        self._plane_fwd = {}   # bf16x6: layer -> its forward pass runs on the plane-image kernel (decided per batch size in _alloc)
        self._plane_dgrad = {}  # ... and its data gradient
        self._plan = []
        self._shapes = {}
        self._dry = False
        self._flat = None
        self._bufs = None
        self._step = 0
        self._micro = 0
        self._estep_cfg = None
        # "momentum" (the reference's), "adamw" or "adamw8" (ops.AdamW with 32- / 8-bit moments over the 32 tensors; config "betas",
        # "adam_eps", "max_grad_norm").  The weight decay of pre_train() is then decoupled, and on the filters alone as before.
        self.optimizer = str(self.config.get("optimizer", "momentum"))
        if self.optimizer not in ("momentum", "adamw", "adamw8"):
            raise ValueError("optimizer must be 'momentum', 'adamw' or 'adamw8', got %r" % self.optimizer)
        self._adamw = None
        self._adamw_source = None
        self._weight_decay = 0.0
        self._momentum = 0.9
        self._gradsync = None
        # config "fused_update": with accum_num == 1 and no gradient exchange the accumulator only carries one micro-batch's gradient
        # from the accumulate kernel to the Momentum kernel; fused, backward() skips the accumulate launches and apply_update() runs
        # accumulate + Momentum + clean as ONE pass per layer (ops.sgd_accumulate_momentum: bit-identical weights, half the bytes).
        # The accumulator then stays zero between the two "ops" of deeplab.py:267-270, so it is opt-in for callers that drive
        # micro_step / apply_update themselves; train(), where nobody looks in between, switches it on.
        self._fused = bool(self.config.get("fused_update", False))
        self._pending_fused = False
        self._bt = {}
        self._tiles_fresh, self._tiles_fresh_ver = set(), None   # layers whose tiled bf16 images the optimizer pass wrote (apply_update)
        self._perm_pool = None
        self._perm_pos = 0
        self.init_model = None

    # ------------------------------------------------------------------------------------------
    # graph construction -- same call sequence as the reference
    # ------------------------------------------------------------------------------------------
    def build(self):
        if "output" not in self.net:
            # placeholders (deeplab.py:27-29): filled by the feed of each step
            self.net["input"] = None
            self.net["label"] = None
            self.net["drop_probe"] = None
            self.net["output"] = self.create_network()
            self.pred()
            bs = self.config.get("batch_size", None)
            if bs:
                self._alloc(int(bs))
        return self.net["output"]

    def create_network(self):
        if "init_model_path" in self.config:
            self.load_init_model()
        fc = None
        # pass 1 (dry) collects shapes so the flat buffers can be laid out; pass 2 binds the views
        for dry in (True, False):
            self._dry = dry
            self._plan = []
            self.stride = {"input": 1}
            self.weights = {}
            self.trainable_list = []
            self.lr_1_list, self.lr_2_list, self.lr_10_list, self.lr_20_list = [], [], [], []
            if not dry:
                self._allocate_flat()
            # build block (deeplab.py:40-45)
            block = self.build_block("input", ["conv1_1", "relu1_1", "conv1_2", "relu1_2", "pool1"])
            block = self.build_block(block, ["conv2_1", "relu2_1", "conv2_2", "relu2_2", "pool2"])
            block = self.build_block(block, ["conv3_1", "relu3_1", "conv3_2", "relu3_2", "conv3_3", "relu3_3", "pool3"])
            block = self.build_block(block, ["conv4_1", "relu4_1", "conv4_2", "relu4_2", "conv4_3", "relu4_3", "pool4"])
            block = self.build_block(block, ["conv5_1", "relu5_1", "conv5_2", "relu5_2", "conv5_3", "relu5_3", "pool5"])
            fc = self.build_fc(block, ["fc6", "relu6", "drop6", "fc7", "relu7", "drop7", "fc8"])
        self._finish_plan()
        # classifier: raw logits, no softmax (deeplab.py:48-49)
        return fc

    def build_block(self, last_layer, layer_lists):
        for layer in layer_lists:
            if layer.startswith("conv"):
                self.stride[layer] = self.stride[last_layer]
                weights, bias = self.get_weights_and_bias(layer)
                rate = 2 if layer[4] == "5" else 1  # atrous_conv2d rate 2 for conv5_x (deeplab.py:60-67)
                self._add_conv(layer, 3, rate)
                self.net[layer] = None  # pre-activation is not materialised: bias+ReLU are fused into the conv
                last_layer = layer
            if layer.startswith("relu"):
                self.stride[layer] = self.stride[last_layer]
                self._fuse(layer, relu=True)
                last_layer = layer
            if layer.startswith("pool"):
                if layer[4] not in ["4", "5"]:
                    self.stride[layer] = 2 * self.stride[last_layer]
                    self._add_pool(layer, 2)  # ksize 3x3, strides 2, SAME (deeplab.py:74-78)
                else:
                    self.stride[layer] = self.stride[last_layer]
                    self._add_pool(layer, 1)  # ksize 3x3, strides 1, SAME (deeplab.py:79-83)
                last_layer = layer
        return last_layer

    def build_fc(self, last_layer, layer_lists):
        for layer in layer_lists:
            if layer.startswith("fc"):
                weights, bias = self.get_weights_and_bias(layer)
                shape = self._shapes[layer]
                if last_layer.startswith("pool"):
                    rate = 4 if self.preset == "ref" else 12  # atrous_conv2d rate 4 on pool5 (deeplab.py:91-92)
                else:
                    rate = 1
                self._add_conv(layer, shape[0], rate)
                self.net[layer] = None
                last_layer = layer
            if layer.startswith("relu"):
                self._fuse(layer, relu=True)
                last_layer = layer
            if layer.startswith("drop"):
                self._fuse(layer, drop=True)  # tf.nn.dropout(x, drop_probe) (deeplab.py:102-105)
                last_layer = layer
        return last_layer

    def e_step(self, last_layer, bg_p, fg_p, num_iter, suppress_others, margin_others):
        """deeplab.py:109-124: resize_nearest(label) -> estep -> argmax, all on the device at run time."""
        self._estep_cfg = dict(layer=last_layer, bg_p=bg_p, fg_p=fg_p, num_iter=num_iter,
                               suppress_others=suppress_others, margin_others=margin_others)
        self.net["e_step"] = None    # float map: only produced on request (want_map)
        self.net["e_argmax"] = self._bufs["labels"] if self._bufs is not None else None  # int64 label map buffer
        return "e_argmax"

    def load_init_model(self):
        """deeplab.py:126-129: a pickled dict {layer: {"w","b"}} stored with np.save."""
        model_path = self.config["init_model_path"]
        self.init_model = np.load(model_path, encoding="latin1", allow_pickle=True).item()
        print("load init model success: %s" % model_path)

    def get_weights_and_bias(self, layer):
        """Shapes exactly as deeplab.py:131-149 (with 64 -> self.width); returns HWIO weight and bias views."""
        if layer.startswith("conv"):
            shape = [3, 3, 0, 0]
            if layer == "conv1_1":
                shape[2] = self.input_channel
            else:
                shape[2] = self.width * self.stride[layer]
                if shape[2] > 8 * self.width:
                    shape[2] = 8 * self.width
                if layer in ["conv2_1", "conv3_1", "conv4_1"]:
                    shape[2] = int(shape[2] / 2)
            shape[3] = self.width * self.stride[layer]
            if shape[3] > 8 * self.width:
                shape[3] = 8 * self.width
        if layer.startswith("fc"):
            if layer == "fc6":
                k = 4 if self.preset == "ref" else 3
                shape = [k, k, 8 * self.width, self.fc_width]
            if layer == "fc7":
                shape = [1, 1, self.fc_width, self.fc_width]
            if layer == "fc8":
                shape = [1, 1, self.fc_width, self.category_num]
        self._shapes[layer] = tuple(shape)
        if self._dry:
            return None, None
        seg = self._segments[layer]
        weights, bias = seg["w"], seg["b"]
        self._init_layer(layer, weights, bias)
        self.weights[layer] = (weights, bias)
        if layer != "fc8":
            self.lr_1_list.append(weights)
            self.lr_2_list.append(bias)
        else:
            self.lr_10_list.append(weights)
            self.lr_20_list.append(bias)
        self.trainable_list.append(weights)
        self.trainable_list.append(bias)
        return weights, bias

    def _init_layer(self, layer, weights, bias):
        gen = torch.Generator(device=self.device)
        gen.manual_seed(self.seed * 1000003 + len(self.trainable_list))
        if self.init_model is None:
            # deeplab.py:150-154: random_normal_initializer(stddev=0.01), zero bias
            weights.copy_(torch.randn(weights.shape, generator=gen, device=self.device) * 0.01)
            bias.zero_()
        elif layer == "fc8":
            # deeplab.py:156-164: xavier_initializer(uniform=True) for the filter AND the bias
            kh, kw, cin, cout = weights.shape
            lim = (6.0 / (kh * kw * cin + kh * kw * cout)) ** 0.5
            weights.copy_((torch.rand(weights.shape, generator=gen, device=self.device) * 2 - 1) * lim)
            blim = (6.0 / (2 * cout)) ** 0.5
            bias.copy_((torch.rand(bias.shape, generator=gen, device=self.device) * 2 - 1) * blim)
        else:
            weights.copy_(torch.as_tensor(np.asarray(self.init_model[layer]["w"], dtype=np.float32)).to(self.device))
            bias.copy_(torch.as_tensor(np.asarray(self.init_model[layer]["b"], dtype=np.float32)).to(self.device))

    # ------------------------------------------------------------------------------------------
    # plan + memory
    # ------------------------------------------------------------------------------------------
    def _add_conv(self, layer, k, rate):
        kh, kw, cin, cout = self._shapes[layer]
        op = _Op(name=layer, kind="conv", out_name=layer, k=k, rate=rate, relu=False, drop=False, cin=cin, cout=cout,
                 cin_p=self._pad_cin(layer, cin), cout_p=round_up(cout, self._cpad), index=len(self._plan))
        if not self._dry:
            seg = self._segments[layer]
            op.seg, op.w_pad, op.b_pad, op.gw_pad, op.gb_pad = seg, seg["w_pad"], seg["b_pad"], seg["gw_pad"], seg["gb_pad"]
        self._plan.append(op)

    def _pad_cin(self, layer, cin):
        # the image keeps its 3 -> 4 padding (conv1_1 always gathers it as f32); every other input is an activation
        return round_up(cin, 4) if layer == "conv1_1" else round_up(cin, self._cpad)

    def _add_pool(self, layer, stride):
        self._plan.append(_Op(name=layer, kind="pool", out_name=layer, stride=stride, index=len(self._plan)))

    def _fuse(self, layer, relu=False, drop=False):
        op = self._plan[-1]
        assert op.kind == "conv", "relu/dropout must follow a conv"
        if relu:
            op.relu = True
        if drop:
            op.drop = True
        op.out_name = layer
        self.net[layer] = None

    def _allocate_flat(self):
        """One flat buffer each for params / grads / accumulators (and momentum, if that is the optimizer), fc8 first (backward order)."""
        order = list(self._shapes.keys())  # build order from the dry pass
        self._segments = {}
        off = 0
        for layer in reversed(order):
            kh, kw, cin, cout = self._shapes[layer]
            cin_p, cout_p = self._pad_cin(layer, cin), round_up(cout, self._cpad)
            nw, nb = kh * kw * cin_p * cout_p, cout_p
            start = off
            self._segments[layer] = dict(start=start, nw=nw, nb=nb, shape=(kh, kw, cin, cout), pshape=(kh, kw, cin_p, cout_p))
            off = round_up(start + nw + nb, _ALIGN)
            self._segments[layer]["end"] = off
        total = off
        dev = self.device
        self._flat = dict(
            params=torch.zeros(total, dtype=torch.float32, device=dev),
            grads=torch.zeros(total, dtype=torch.float32, device=dev),
            accum=torch.zeros(total, dtype=torch.float32, device=dev),
            total=total,
        )
        if self.optimizer == "momentum":   # (AdamW keeps its own states, from optimize() on)
            self._flat["momentum"] = torch.zeros(total, dtype=torch.float32, device=dev)
        for layer, seg in self._segments.items():
            s, nw, nb = seg["start"], seg["nw"], seg["nb"]
            kh, kw, cin, cout = seg["shape"]
            for prefix, buf in (("", "params"), ("g", "grads")):
                wp = self._flat[buf][s:s + nw].view(seg["pshape"])
                bp = self._flat[buf][s + nw:s + nw + nb]
                seg[prefix + "w_pad"], seg[prefix + "b_pad"] = wp, bp
                seg[prefix + "w"], seg[prefix + "b"] = wp[:, :, :cin, :cout], bp[:cout]
        if self.compute_dtype == "bf16x6":
            # k-contiguous f32 image of every filter for the forward pass (include/emadapt.h "bf16x6")
            self._flat["wk32"] = torch.zeros(total, dtype=torch.float32, device=dev)
            for layer, seg in self._segments.items():
                kh, kw, cin_p, cout_p = seg["pshape"]
                seg["wk32"] = self._flat["wk32"][seg["start"]:seg["start"] + seg["nw"]].view(kh * kw, cout_p, cin_p)
            # tiled plane images (csrc/conv_x6p.hip, ops.filter_tiles) for the forward and the data-gradient kernel of the layers
            # the plane kernels can take: a reduction over whole groups of 16 channels and at least 256 output columns
            # (emadapt_conv_x6p_supported's channel rules; its size limits are checked per batch in _alloc).  "kmajor": the layer's
            # forward pass runs on conv_x6.hip's kernel and needs the k-contiguous f32 image (64 or fewer output columns: native).
            for layer, seg in self._segments.items():
                kh, kw, cin_p, cout_p = seg["pshape"]
                # (the images are ALLOCATED in _alloc, for the layers that take the plane kernels at the batch size in use, and
                # refreshed for those alone: by the channel rule alone the ref preset carried ~600 MB of images and rebuilt them
                # after every optimizer step even at batch 1, where no plane kernel runs)
                seg["can_wkp"], seg["can_wp6"] = cout_p >= 256, cin_p >= 256
                seg["wkp"] = seg["wp6"] = None
                seg["kmajor"] = not seg["can_wkp"] and cout_p > 64
            self._w16_seen = None
        if self.compute_dtype == "bf16":
            # bf16 filter images (include/emadapt.h, "bf16-compute variants"), one flat buffer per image kind
            offs, nf, nd = {}, 0, 0
            for layer, seg in self._segments.items():
                kh, kw, cin_p, cout_p = seg["pshape"]
                sf, sd = kh * kw * cout_p * round_up(cin_p, 8), kh * kw * cin_p * round_up(cout_p, 8)
                offs[layer] = (nf, sf, nd, sd)
                nf, nd = round_up(nf + sf, 128), round_up(nd + sd, 128)
            self._flat["wf16"] = torch.zeros(nf, dtype=torch.bfloat16, device=dev)
            self._flat["wd16"] = torch.zeros(nd, dtype=torch.bfloat16, device=dev)
            for layer, seg in self._segments.items():
                kh, kw, cin_p, cout_p = seg["pshape"]
                of, sf, od, sd = offs[layer]
                seg["wf16"] = self._flat["wf16"][of:of + sf].view(kh * kw, cout_p, round_up(cin_p, 8))
                seg["wd16"] = self._flat["wd16"][od:od + sd].view(kh * kw, cin_p, round_up(cout_p, 8))
            self._w16_seen = None

    def _finish_plan(self):
        h, w = self.h, self.w
        for op in self._plan:
            op.in_hw = (h, w)
            if op.kind == "pool":
                h, w = ops.pool_out_size(h, op.stride), ops.pool_out_size(w, op.stride)
            op.out_hw = (h, w)
        self.out_hw = (h, w)
        self.c_pad = round_up(self.category_num, self._cpad)

    def parameter_count(self):
        return sum(int(np.prod(s["shape"])) + s["shape"][3] for s in self._segments.values())

    def flops_per_image(self):
        """Algorithmic FLOPs of one fwd+bwd (bwd = 2x fwd), un-padded shapes."""
        macs = 0
        for op in self._plan:
            if op.kind == "conv":
                macs += op.out_hw[0] * op.out_hw[1] * op.k * op.k * op.cin * op.cout
        return 2.0 * macs, 6.0 * macs

    def _alloc(self, B):
        if self._bufs is not None and self._bufs["B"] == B:
            return self._bufs
        dev = self.device
        f32 = torch.float32
        bufs = {"B": B, "act": {}, "idx": {}}
        bufs["x4"] = torch.zeros((B, self.h, self.w, round_up(self.input_channel, 4)), dtype=f32, device=dev)
        maxn = bufs["x4"].numel()
        c = bufs["x4"].shape[3]
        adt = self.act_dtype
        for op in self._plan:
            oh, ow = op.out_hw
            if op.kind == "conv":
                c = op.cout_p
                dt = f32 if op is self._plan[-1] else adt   # the logits feed the E-step and the loss: always f32
                bufs["act"][op.name] = torch.empty((B, oh, ow, c), dtype=dt, device=dev)
            else:
                bufs["act"][op.name] = torch.empty((B, oh, ow, c), dtype=adt, device=dev)
                bufs["idx"][op.name] = torch.empty((B, oh, ow, c), dtype=torch.uint8, device=dev)
            maxn = max(maxn, bufs["act"][op.name].numel())
            self.net[op.out_name] = bufs["act"][op.name]
        if self.compute_dtype == "bf16x6":
            # which convolutions run on the plane-image kernels (csrc/conv_x6p.hip), their input's plane image (kept from the
            # forward pass for the filter gradient) and one scratch image for the gradient that enters a layer
            xp, dyp_bytes = {}, 0
            for op in self._plan:
                if op.kind != "conv":
                    continue
                ih, iw = op.in_hw
                d = ops.conv_desc(B, ih, iw, op.cin_p, op.cout_p, op.k, op.k, op.rate)
                # config "x6_planes": "auto" (default) = where the plane kernel has enough work to fill the part at this batch
                # size, "always" = wherever it can run and the six-MFMA kernels for every other GEMM with more than 64 columns,
                # however small (the parity tests drive them on small shapes this way)
                take = ops.conv_x6p_supported if self.config.get("x6_planes", "auto") == "always" else ops.conv_x6p_pays
                e = dict(d=d, fwd=op.seg["can_wkp"] and take(d, 0), dgrad=op.seg["can_wp6"] and take(d, 1), wgrad=take(d, 2))
                for key, flag, dg in (("wkp", e["fwd"], False), ("wp6", e["dgrad"], True)):
                    if flag and op.seg[key] is None:
                        kh, kw, cin_p, cout_p = op.seg["pshape"]
                        op.seg[key] = torch.zeros(ops.filter_tiles_bytes(cin_p, cout_p, kh, kw, dg), dtype=torch.uint8, device=dev)
                e["x"] = (torch.empty(B * ih * iw * op.cin_p * 6, dtype=torch.uint8, device=dev) if (e["fwd"] or e["wgrad"]) else None)
                # a GEMM below 3 GFLOP (small maps / narrow nets; at the benchmark shapes none) is launch- and tail-bound: the native
                # fp32 kernels' split-K plans are the faster fp32-grade choice there (scripts/shape_sweep.sh)
                e["small"] = (2.0 * B * ih * iw * op.k * op.k * op.cin_p * op.cout_p < 3e9 and self.config.get("x6_planes", "auto") != "always")
                if e["dgrad"] or e["wgrad"]:
                    dyp_bytes = max(dyp_bytes, B * ih * iw * op.cout_p * 6)
                xp[op.name] = e
            bufs["xp"] = xp
            plane_fwd = {name: e["fwd"] for name, e in xp.items()}
            plane_dgrad = {name: e["dgrad"] for name, e in xp.items()}
            if plane_fwd != self._plane_fwd or plane_dgrad != self._plane_dgrad:   # (first batch, or a batch size that changes which layers the plane kernels take)
                self._plane_fwd, self._plane_dgrad = plane_fwd, plane_dgrad
                self._w16_seen = None
            bufs["dyp"] = torch.empty(max(dyp_bytes, 16), dtype=torch.uint8, device=dev)
        if self.compute_dtype == "bf16":
            # which layers run forward / data gradient on the LDS-DMA kernel (csrc/igemm_b16t.h: 16x16x32 MFMAs, DMA waves) at this
            # batch size -- config "bf16t": "auto" (default: where the library says it pays: fc6 / fc7 at batch 16), "always"
            # (wherever it can run: the parity tests), "never" -- and their tiled filter images (instead of the plain bf16 images)
            mode = str(self.config.get("bf16t", "auto"))
            take = {"auto": ops.conv_bf16t_pays, "always": ops.conv_bf16t_supported, "never": lambda *a, **k: False}[mode]
            bt = {}
            plan = self._plan
            for i, op in enumerate(plan):
                if op.kind != "conv":
                    continue
                ih, iw = op.in_hw
                d = ops.conv_desc(B, ih, iw, op.cin_p, op.cout_p, op.k, op.k, op.rate)
                x_bf16 = i > 0 and adt == torch.bfloat16                     # (the image into conv1_1 is f32)
                y_bf16 = op is not plan[-1] and adt == torch.bfloat16        # (the logits are f32)
                e = dict(fwd=x_bf16 and take(d, "fwd", y_bf16), dgrad=i > 0 and op is not plan[-1] and take(d, "dgrad", True))
                for key, flag, dg in (("wt16", e["fwd"], False), ("wtd16", e["dgrad"], True)):
                    if flag and op.seg.get(key) is None:
                        op.seg[key] = ops.filter_tiles_bf16(op.w_pad, dgrad=dg)
                bt[op.name] = e
            if bt != self._bt:
                self._bt = bt
                self._w16_seen = None
            bufs["bt"] = bt
        bufs["gA"] = torch.empty(maxn, dtype=adt, device=dev)   # activation gradients ping-pong between these two
        bufs["gB"] = torch.empty(maxn, dtype=adt, device=dev)
        S1, S2 = self.out_hw
        bufs["shrink"] = torch.empty((B, S1, S2), dtype=f32, device=dev)
        bufs["labels"] = torch.empty((B, S1, S2), dtype=torch.int64, device=dev)
        bufs["label_full"] = torch.empty((B, self.h, self.w), dtype=f32, device=dev)
        self.net["e_argmax"] = bufs["labels"]
        last = self._plan[-1]
        self.net["output"] = bufs["act"][last.name][..., :self.category_num]
        self._bufs = bufs
        return bufs

    # ------------------------------------------------------------------------------------------
    # execution
    # ------------------------------------------------------------------------------------------
    def _to_dev(self, a, dtype=torch.float32):
        if isinstance(a, torch.Tensor):
            return a.to(device=self.device, dtype=dtype, non_blocking=True).contiguous()
        return torch.as_tensor(np.ascontiguousarray(a)).to(device=self.device, dtype=dtype, non_blocking=True)

    def refresh_bf16_weights(self, force=False):
        """Re-derive the bf16 filter images when the fp32 master weights changed (torch in-place ops bump the flat
        buffer's version counter; the optimizer kernel, which torch does not see, resets ``_w16_seen`` itself)."""
        if self.compute_dtype == "fp32":
            return
        ver = self._flat["params"]._version
        if not force and self._w16_seen == ver:
            return
        # (layers whose two tiled images the optimizer pass itself wrote from the weights as they are now: apply_update)
        fresh = self._tiles_fresh if (not force and self._tiles_fresh_ver == ver) else ()
        plain = []   # (filter, forward image, data-gradient image) of the layers on the register-staged kernel: one launch for all
        for op in self._plan:
            if op.kind == "conv":
                if self.compute_dtype == "bf16":
                    e = self._bt.get(op.name, {"fwd": False, "dgrad": False})
                    if not (e["fwd"] and e["dgrad"]):
                        plain.append((op.w_pad, None if e["fwd"] else op.seg["wf16"], None if e["dgrad"] else op.seg["wd16"]))
                    if e["fwd"] and e["dgrad"] and op.name in fresh:
                        pass
                    elif e["fwd"] and e["dgrad"]:
                        ops.filter_tiles_bf16_both(op.w_pad, op.seg["wt16"], op.seg["wtd16"])   # (one pass over the f32 filter)
                    elif e["fwd"]:
                        ops.filter_tiles_bf16(op.w_pad, dgrad=False, out=op.seg["wt16"])
                    elif e["dgrad"]:
                        ops.filter_tiles_bf16(op.w_pad, dgrad=True, out=op.seg["wtd16"])
                else:
                    if op.seg["kmajor"] or not self._plane_fwd.get(op.name, True):
                        ops.filter_kmajor(op.w_pad, op.seg["wk32"])
                    if self._plane_fwd.get(op.name, False):
                        ops.filter_tiles(op.w_pad, False, out=op.seg["wkp"])
                    if self._plane_dgrad.get(op.name, False):
                        ops.filter_tiles(op.w_pad, True, out=op.seg["wp6"])
        for i in range(0, len(plain), ops.W16_MAX_LAYERS):
            ops.weights_to_bf16_multi(plain[i:i + ops.W16_MAX_LAYERS])
        self._w16_seen = ver
        self._tiles_fresh, self._tiles_fresh_ver = set(), None

    def _pool_gate_in_idx(self, before):
        """A max-pool behind a ReLU layer keeps that layer's ReluGrad gate in its index bytes (ops.maxpool_fwd relu_gate; config
        "pool_gate_idx": False = the gradient reads the pooled tensor as the gate, the A/B)."""
        return bool(before is not None and before.kind == "conv" and before.relu and self.config.get("pool_gate_idx", True))

    def forward(self, images, keep_prob=1.0, drop_masks=None, for_backward=False):
        """The conv stack (deeplab.py:35-49). images [B,H,W,3]; returns the fc8 logits view [B,S,S,C].  for_backward: the pass is
        followed by backward() (micro_step): bf16x6 then also splits the inputs of the layers whose FILTER GRADIENT alone runs on
        the plane kernels; an inference pass skips that work."""
        images = self._to_dev(images)
        bf16 = self.compute_dtype == "bf16"
        x6 = self.compute_dtype == "bf16x6"
        B = images.shape[0]
        bufs = self._alloc(B)
        self.refresh_bf16_weights()
        self.net["input"] = images
        self.net["drop_probe"] = keep_prob
        if images.shape[3] == bufs["x4"].shape[3]:
            x = images
        else:
            x = ops.copy_pad_channels(images, bufs["x4"].shape[3], out=bufs["x4"])
        bufs["x_in"] = x
        prev = None
        for op in self._plan:
            out = bufs["act"][op.name]
            prev, before = op, prev
            if op.kind == "conv":
                kp = keep_prob if op.drop else 1.0
                mask = None
                if op.drop and kp < 1.0 and drop_masks is not None:
                    mask = self._pad_mask(drop_masks[op.name], op)
                seed = self._drop_seed(op)
                if bf16 and bufs["bt"][op.name]["fwd"]:
                    ops.conv_fwd_bf16t(x, op.seg["wt16"], (op.k, op.k), op.cout_p, op.b_pad, op.rate, relu=op.relu, keep_prob=kp,
                                       drop_mask=mask, drop_seed=seed, out=out)
                elif bf16:
                    ops.conv_fwd_bf16(x, op.seg["wf16"], (op.k, op.k), op.b_pad, op.rate, relu=op.relu, keep_prob=kp,
                                      drop_mask=mask, drop_seed=seed, out=out)
                elif x6:
                    e = bufs["xp"][op.name]
                    if e["x"] is not None and (e["fwd"] or for_backward):
                        ops.split_planes(x, out=e["x"])
                    if e["fwd"]:
                        ops.conv_fwd_x6p(e["x"], op.seg["wkp"], e["d"], op.b_pad, relu=op.relu, keep_prob=kp,
                                         drop_mask=mask, drop_seed=seed, out=out)
                    elif op.cout_p <= 64 or e["small"]:
                        # (64 or fewer output columns -- conv1_x, fc8: the native fp32 kernel's 256x64 tiles are the faster
                        # fp32-grade kernel there, measured per layer: profiles/r03_x6_*)
                        ops.conv_fwd(x, op.w_pad, op.b_pad, op.rate, relu=op.relu, keep_prob=kp, drop_mask=mask,
                                     drop_seed=seed, out=out)
                    else:
                        ops.conv_fwd_x6(x, op.seg["wk32"], (op.k, op.k), op.b_pad, op.rate, relu=op.relu, keep_prob=kp,
                                        drop_mask=mask, drop_seed=seed, out=out)
                else:
                    ops.conv_fwd(x, op.w_pad, op.b_pad, op.rate, relu=op.relu, keep_prob=kp, drop_mask=mask,
                                 drop_seed=seed, out=out)
            else:
                # (the index carries the ReluGrad gate of the pooled tensor: backward() then never reads that tensor again)
                ops.maxpool_fwd(x, op.stride, out=out, idx=bufs["idx"][op.name], relu_gate=self._pool_gate_in_idx(before))
            x = out
        bufs["keep_prob"] = keep_prob
        return self.net["output"]

    def _drop_seed(self, op):
        """Seed of the built-in dropout generator for this op and micro-step; ranks of a data-parallel job draw
        different masks (tf.nn.dropout on every tower draws independently)."""
        rank, world = dist_rank_world(self.config)
        return ((self.seed * world + rank) << 32) + self._micro * 64 + op.index

    def _pad_mask(self, m, op):
        m = self._to_dev(m, torch.uint8)
        if m.shape[-1] != op.cout_p:
            mp = torch.zeros(tuple(m.shape[:-1]) + (op.cout_p,), dtype=torch.uint8, device=self.device)
            mp[..., :m.shape[-1]] = m
            m = mp
        return m

    def _next_perms(self):
        cfg = self._estep_cfg
        n_it, C = cfg["num_iter"], self.category_num
        if self._perm_pool is None or self._perm_pos >= self._perm_pool.shape[0]:
            # drawn with the reference's calls on Python's global generator (estep.py:64-66), 64 steps at a time
            host = np.stack([draw_perms(n_it, C, rng=random) for _ in range(64)])
            self._perm_pool = torch.as_tensor(host).to(self.device)
            self._perm_pos = 0
        p = self._perm_pool[self._perm_pos]
        self._perm_pos += 1
        return p

    def run_estep(self, labels, perms=None, want_map=False):
        """deeplab.py:109-124 on the current logits. labels: pixel labels [B,H,W(,1)] f32, or uint8 multi-hot [B,C]."""
        cfg = self._estep_cfg
        bufs = self._bufs
        logits = bufs["act"][self._plan[-1].name]
        if perms is None:
            perms = self._next_perms()
        else:
            perms = self._to_dev(perms, torch.int32)
        if isinstance(labels, torch.Tensor) and labels.dtype == torch.uint8 or (
                isinstance(labels, np.ndarray) and labels.dtype == np.uint8 and labels.ndim == 2):
            lab = self._to_dev(labels, torch.uint8)
            kind = ops.LABEL_MULTIHOT
        else:
            full = self._to_dev(labels)
            self.net["label"] = full
            lab = ops.resize_nearest(full, self.out_hw[0], self.out_hw[1], out=bufs["shrink"])
            kind = ops.LABEL_F32
        labels_out, fmap = ops.estep_device(
            logits, lab, perms, self.category_num, suppress_others=cfg["suppress_others"], num_iter=cfg["num_iter"],
            margin_others=cfg["margin_others"], bg_p=cfg["bg_p"], fg_p=cfg["fg_p"], label_kind=kind,
            want_map=want_map, labels_out=bufs["labels"], map_out=bufs.get("estep_map"))
        if fmap is not None:
            bufs["estep_map"] = fmap
            self.net["e_step"] = fmap
        return labels_out

    def getloss(self, weight_decay):
        weaklabel_layer = self.e_step("fc8", bg_p=0.4, fg_p=0.2, num_iter=5, suppress_others=True, margin_others=1e-5)
        self._weight_decay = float(weight_decay)
        self.loss["norm"] = None   # device scalars, refreshed by micro_step()/eval_loss()
        self.loss["l2"] = None
        self.loss["total"] = None
        return weaklabel_layer

    def optimize(self, base_lr, momentum):
        self.net["lr"] = float(base_lr)
        self._momentum = float(momentum)
        if self.optimizer != "momentum":
            before, params, decay = self._adamw, [], []
            for layer in self._segments:
                s, nw, nb = (self._segments[layer][k] for k in ("start", "nw", "nb"))
                params += [self._flat["params"][s:s + nw], self._flat["params"][s + nw:s + nw + nb]]
                decay += [self._weight_decay, 0.0]
            self._adamw = ops.AdamW(params, self._adamw_grads(self._flat["accum"]), state="u8" if self.optimizer == "adamw8" else "f32",
                                    betas=tuple(self.config.get("betas", (0.9, 0.999))), eps=float(self.config.get("adam_eps", 1e-8)),
                                    weight_decay=decay, seed=self.seed)
            if before is not None:   # (trained before: the moments and steps go on, as the Momentum buffer does)
                for name in ("m", "v") if before.state == "f32" else ("m8", "u8", "powers"):
                    getattr(self._adamw, name).copy_(getattr(before, name))
                self._adamw.steps.copy_(before.steps)
            self._adamw_source = self._flat["accum"]
        # the three "ops" of the reference's loop (deeplab.py:202-205), as callables
        self.net["accum_gradient"] = self._flat["accum"]
        self.net["accum_gradient_accum"] = self.micro_step
        self.net["accum_gradient_update"] = self.apply_update
        self.net["accum_gradient_clean"] = lambda: None  # folded into the update kernel (accum is zeroed there)
        self.net["train_op"] = self.apply_update
        self.net["g"] = 1.0
        if torch.distributed.is_available() and torch.distributed.is_initialized() and \
                (torch.distributed.get_world_size() > 1 or self.config.get("force_gradsync", False)):
            from .dist import GradSync
            # config "allreduce_algo": "allreduce" (RCCL's own) | "direct" (reduce-scatter + all-gather as two all-to-all steps over
            # all xGMI links, on a side stream); "grad_dtype": "fp32" | "bf16" payload (bf16 needs "direct"; dist.py)
            grad_dtype = str(self.config.get("grad_dtype", "fp32"))
            algo = str(self.config.get("allreduce_algo", "direct" if grad_dtype == "bf16" else "allreduce"))
            # (direct exchange: the summed gradients stay in GradSync.gathered, which apply_update's Momentum kernel reads in place)
            # accum_num == 1 with the direct exchange: backward packs (g + wd w) / accum_num straight into the exchange's send buffer
            # (ops.sgd_accumulate_pack) -- no accumulate pass, no accumulator traffic, no pack pass (config "dp_prepack": False = the
            # accumulator path, what accum_num > 1 always takes)
            prepack = self.accum_num == 1 and algo == "direct" and bool(self.config.get("dp_prepack", True))
            # buckets: config "bucket_mb" = equal sizes (the ring all-reduce's default: 32 MB); the direct exchange without it = two buckets
            # cut behind the last fully connected layer (fc8 + fc7 + fc6: 77 % of the bytes, complete a third of the way into backward)
            bounds = None
            if algo == "direct" and self.config.get("bucket_mb", None) is None:
                fcs = [op for op in self._plan if op.kind == "conv" and op.name.startswith("fc")]
                if fcs and len(fcs) < sum(op.kind == "conv" for op in self._plan):
                    bounds = [max(op.seg["end"] for op in fcs)]
            self._gradsync = GradSync(self._flat["accum"], [(s["start"], s["end"]) for s in self._bucket_order()],
                                      bucket_bytes=int(self.config.get("bucket_mb", None) or 32) << 20, algo=algo, payload=grad_dtype,
                                      writeback=False, prepacked=prepack, boundaries=bounds)
            # a failure recorded in ONE rank's device status word must not make that rank alone skip its update: the producers of the
            # exchange turn it into NaNs that travel with the gradient, and every rank's optimiser pass leaves the same elements alone
            # and raises its own word (include/emadapt.h, emadapt_status_collective)
            ops.status_collective(True)

    def _adamw_grads(self, flat):
        """The 32 tensors' gradients in a buffer laid out like the flat parameters (accumulators, one micro-batch's gradients, the exchange's payload)."""
        got = []
        for seg in self._segments.values():
            s, nw, nb = seg["start"], seg["nw"], seg["nb"]
            got += [flat[s:s + nw], flat[s + nw:s + nw + nb]]
        return got

    def _adamw_update(self, scale):
        """apply_update() with AdamW: the gradients are read where the mode leaves them, the accumulators zeroed (the clean op)."""
        f, gs = self._flat, self._gradsync
        clean = False
        if self._pending_fused:
            source, scale = f["grads"], scale / float(self.accum_num)
            self._pending_fused = False
        elif gs is not None and not gs.writeback:
            source = gs.gathered
            if not gs.prepacked:
                f["accum"].zero_()
        else:
            source, clean = f["accum"], True
        if source is not self._adamw_source:
            self._adamw.set_grads(self._adamw_grads(source))
            self._adamw_source = source
        self._adamw.step(self.net["lr"], grad_scale=scale, max_norm=float(self.config.get("max_grad_norm", 0.0)), zero_grads=clean)

    def _bucket_order(self):
        return [self._segments[op.name] for op in reversed(self._plan) if op.kind == "conv"]

    def _ce(self, want_grad=True):
        bufs = self._bufs
        logits = bufs["act"][self._plan[-1].name]
        M = logits.numel() // logits.shape[-1]
        dl = bufs["gA"][:logits.numel()].view(logits.shape) if want_grad else None
        loss_sum, dl = ops.softmax_ce(logits, bufs["labels"], self.category_num, grad_scale=1.0 / M,
                                      want_grad=want_grad, want_loss=True, dlogits=dl)
        self.loss["norm"] = loss_sum / M
        return dl

    def backward(self, dlogits, last_micro=True):
        """Hand-written autodiff of deeplab.py:192 (fc8 .. conv1_1), accumulating as deeplab.py:202."""
        bufs = self._bufs
        B = bufs["B"]
        keep = bufs.get("keep_prob", 1.0)
        d = dlogits
        cur, other = bufs["gA"], bufs["gB"]
        inv_accum = 1.0 / float(self.accum_num)
        decay = self._weight_decay if self._adamw is None else 0.0   # (AdamW's decay is not a part of the gradient)
        plan = self._plan
        bf16 = self.compute_dtype == "bf16"
        x6 = self.compute_dtype == "bf16x6"
        # data parallel: every bucket's all-reduce is launched as soon as its gradients are final (default), or -- opt-in,
        # config "allreduce_release_at": a layer name -- held until backward reaches that layer (dist.py: a policy to be
        # chosen by measurement on a multi-GPU node; bench.py reports the exposed time of either)
        sync = self._gradsync if last_micro else None
        fused = self._fused and self.accum_num == 1 and self._gradsync is None   # (see __init__: apply_update does the accumulate)
        self._pending_fused = fused
        release_at = self.config.get("allreduce_release_at", None)
        if sync is not None and release_at is not None and any(o.name == release_at for o in plan):
            sync.hold()
        for i in range(len(plan) - 1, -1, -1):
            op = plan[i]
            prev = plan[i - 1] if i > 0 else None
            if sync is not None and op.name == release_at:
                sync.release()
            if op.kind == "conv":
                x_in = bufs["act"][prev.name] if prev is not None else bufs["x_in"]
                if bf16:
                    # (the bias gradient rides in the filter-gradient launch: its loader waves see every dy piece anyway)
                    ops.conv_wgrad_bf16(x_in, d, op.k, op.k, op.rate, out=op.gw_pad, bias_out=op.gb_pad)
                elif x6:
                    e = bufs["xp"][op.name]
                    if e["wgrad"] or (e["dgrad"] and prev is not None):
                        ops.split_planes(d, out=bufs["dyp"])
                    if e["wgrad"]:
                        ops.conv_wgrad_x6p(e["x"], bufs["dyp"], e["d"], out=op.gw_pad)
                    elif e["small"]:
                        ops.conv_wgrad(x_in, d, op.k, op.k, op.rate, out=op.gw_pad, bias_out=op.gb_pad)
                    else:
                        ops.conv_wgrad_x6(x_in, d, op.k, op.k, op.rate, out=op.gw_pad)
                    if e["wgrad"] or not e["small"]:
                        ops.bias_grad(d, out=op.gb_pad)
                else:
                    # (the bias gradient rides in the filter-gradient launch where the library fuses it: conv1_x .. conv3_1, fc8)
                    ops.conv_wgrad(x_in, d, op.k, op.k, op.rate, out=op.gw_pad, bias_out=op.gb_pad)
                seg = op.seg
                s, n = seg["start"], seg["nw"] + seg["nb"]
                if sync is not None and sync.prepacked:
                    ops.sgd_accumulate_pack(self._flat["grads"][s:s + n], self._flat["params"][s:s + n], seg["nw"], decay,
                                            inv_accum, out=sync.sendfull[s:s + n])
                elif not fused:
                    ops.sgd_accumulate(self._flat["accum"][s:s + n], self._flat["grads"][s:s + n],
                                       self._flat["params"][s:s + n], seg["nw"], decay, inv_accum)
                if last_micro and self._gradsync is not None:
                    self._gradsync.segment_ready(seg["start"], seg["end"])
                if prev is None:
                    break
                out = other[:x_in.numel()].view(x_in.shape)
                gate, scale = None, 1.0
                if prev.kind == "conv" and prev.relu:
                    gate = x_in
                    scale = (1.0 / keep) if (prev.drop and keep < 1.0) else 1.0
                if bf16 and bufs["bt"][op.name]["dgrad"]:
                    d = ops.conv_dgrad_bf16t(d, op.seg["wtd16"], (op.k, op.k), op.cin_p, op.rate, gate=gate, gate_scale=scale, out=out)
                elif bf16:
                    d = ops.conv_dgrad_bf16(d, op.seg["wd16"], (op.k, op.k), op.rate, gate=gate, gate_scale=scale, out=out)
                elif x6:
                    if bufs["xp"][op.name]["dgrad"]:
                        d = ops.conv_dgrad_x6p(bufs["dyp"], op.seg["wp6"], bufs["xp"][op.name]["d"], gate=gate, gate_scale=scale, out=out)
                    elif op.cin_p <= 64 or bufs["xp"][op.name]["small"]:
                        d = ops.conv_dgrad(d, op.w_pad, op.rate, gate=gate, gate_scale=scale, out=out)
                    else:
                        d = ops.conv_dgrad_x6(d, op.w_pad, op.rate, gate=gate, gate_scale=scale, out=out)
                else:
                    d = ops.conv_dgrad(d, op.w_pad, op.rate, gate=gate, gate_scale=scale, out=out)
            else:
                x_in = bufs["act"][prev.name]
                gate = x_in if (prev.kind == "conv" and prev.relu and not self._pool_gate_in_idx(prev)) else None
                out = other[:x_in.numel()].view(x_in.shape)
                d = ops.maxpool_bwd(d, bufs["idx"][op.name], tuple(x_in.shape), op.stride, gate=gate, out=out)
            cur, other = other, cur
        del B

    def micro_step(self, images, labels, keep_prob=0.5, perms=None, drop_masks=None):
        """sess.run(net["accum_gradient_accum"], feed) of deeplab.py:267: fwd + E-step + bwd + accumulate."""
        self.forward(images, keep_prob, drop_masks, for_backward=True)
        self.run_estep(labels, perms)
        dl = self._ce(want_grad=True)
        last = (self._micro % self.accum_num) == self.accum_num - 1
        self.backward(dl, last_micro=last)
        self._micro += 1
        return self.loss["norm"]

    # -- training on rewards and preferences (beside micro_step: the same forward, backward and update) -----------------------
    def _own_loss(self, images, keep_prob, loss):
        """One micro-batch with a loss of its own over the logits: loss(logits, dlogits) fills dlogits."""
        self.forward(images, keep_prob, for_backward=True)
        logits = self._bufs["act"][self._plan[-1].name]
        dl = self._bufs["gA"][:logits.numel()].view(logits.shape)
        out = loss(logits, dl)
        self.backward(dl, last_micro=(self._micro % self.accum_num) == self.accum_num - 1)
        self._micro += 1
        return out

    def label_logp(self, images, labels, keep_prob=1.0):
        """Log-probability f32 [B,S,S] of the label maps int64 [B,S,S] (S = the logits' size, 255 = void: 0) under the network as it is: what
        policy_step takes as old_logp / ref_logp."""
        self.forward(images, keep_prob)
        return ops.label_logp(self._bufs["act"][self._plan[-1].name], self._to_dev(labels, torch.int64), self.category_num)[0]

    def policy_step(self, images, labels, old_logp, advantages, ref_logp=None, weights=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, keep_prob=1.0):
        """One micro-batch of the clipped policy loss (ops.policy_loss, mean over the pixels) on sampled label maps int64 [B,S,S]: forward, loss, backward,
        accumulate.  advantages (and weights): f32 [B,S,S], or one per image [B].  Returns (sums, logp)."""
        lab = self._to_dev(labels, torch.int64)

        def rows(v):
            if v is None:
                return None
            v = self._to_dev(v)
            return v.view(-1, 1, 1).expand(lab.shape).contiguous() if v.dim() == 1 else v

        old, adv, ref, w = (rows(v) for v in (old_logp, advantages, ref_logp, weights))
        sums, logp = self._own_loss(images, keep_prob, lambda z, dl: ops.policy_loss(
            z, lab, old, adv, self.category_num, ref_logp=ref, weights=w, clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, dlogits=dl)[:2])
        self.loss["norm"] = sums[:1] / max(lab.numel(), 1)
        return sums, logp

    def preference_step(self, images, labels, ref_logp, beta=0.1, label_smoothing=0.0, keep_prob=1.0):
        """One micro-batch of the preference loss (ops.preference_loss, mean over the pairs): images [2P,H,W,3] with label maps int64 [2P,S,S], entry 2j
        preferred to entry 2j + 1; ref_logp f32 [2P]: the maps' summed log-probabilities under the reference network.  Returns (loss [P], map_logp [2P])."""
        lab = self._to_dev(labels, torch.int64)
        if lab.shape[0] % 2:
            raise ValueError("preference_step takes pairs: %d label maps" % lab.shape[0])
        at = torch.arange(lab.shape[0] + 1, device=self.device) * (lab.numel() // max(lab.shape[0], 1))
        ref = self._to_dev(ref_logp)
        loss, seq = self._own_loss(images, keep_prob, lambda z, dl: ops.preference_loss(z, lab, at, ref, self.category_num, beta=beta,
                                                                                      label_smoothing=label_smoothing, dlogits=dl)[:2])
        self.loss["norm"] = loss.mean()
        return loss, seq

    def apply_update(self):
        """accum_gradient_update + accum_gradient_clean (deeplab.py:203-205,268-270)."""
        scale = 1.0
        f = self._flat
        gs = self._gradsync
        if gs is not None:
            gs.wait()
            scale = 1.0 / gs.world_size
        fresh = set()
        if self._adamw is not None:
            self._adamw_update(scale)
        elif self._pending_fused:
            tiles = self.compute_dtype == "bf16" and self.config.get("fused_tiles", True)
            rest = []   # (start, n, n_decay) of the layers without a pass of their own: one launch for all of them
            for op in self._plan:   # accumulate + apply_gradients + clean of the one micro-batch
                if op.kind == "conv":
                    s, n = op.seg["start"], op.seg["nw"] + op.seg["nb"]
                    e = self._bt.get(op.name, {"fwd": False, "dgrad": False})
                    if (tiles and e["fwd"] and e["dgrad"] and op.seg.get("wt16") is not None and op.seg.get("wtd16") is not None
                            and ops.sgd_accumulate_momentum_tiles_supported(*op.seg["pshape"])):
                        # (the pass also writes the layer's two tiled bf16 images: the next forward's refresh skips them)
                        ops.sgd_accumulate_momentum_tiles(f["params"][s:s + n], f["momentum"][s:s + n], f["grads"][s:s + n], tuple(op.seg["pshape"]),
                                                          self._weight_decay, 1.0 / float(self.accum_num), self.net["lr"], self._momentum, scale,
                                                          op.seg["wt16"], op.seg["wtd16"])
                        fresh.add(op.name)
                    elif s % 4 == 0 and n % 4 == 0 and op.seg["nw"] % 4 == 0 and self.config.get("fused_update_multi", True):
                        rest.append((s, n, op.seg["nw"]))
                    else:
                        ops.sgd_accumulate_momentum(f["params"][s:s + n], f["momentum"][s:s + n], f["grads"][s:s + n], op.seg["nw"],
                                                    self._weight_decay, 1.0 / float(self.accum_num), self.net["lr"], self._momentum, scale)
            for i in range(0, len(rest), ops.SGD_MAX_SEGS):
                ops.sgd_accumulate_momentum_multi(f["params"], f["momentum"], f["grads"], rest[i:i + ops.SGD_MAX_SEGS], self._weight_decay,
                                                  1.0 / float(self.accum_num), self.net["lr"], self._momentum, scale)
            self._pending_fused = False
        elif gs is not None and not gs.writeback:
            # the exchanged sum lives in the gathered payload (f32 or bf16); the accumulator is only zeroed (the clean op)
            acc = None if gs.prepacked else f["accum"]
            tiled = []   # layers whose pass also writes their two tiled bf16 images (as in the fused update above)
            if self.compute_dtype == "bf16" and self.config.get("fused_tiles", True):
                for op in self._plan:
                    if op.kind == "conv":
                        e = self._bt.get(op.name, {"fwd": False, "dgrad": False})
                        if (e["fwd"] and e["dgrad"] and op.seg.get("wt16") is not None and op.seg.get("wtd16") is not None
                                and ops.sgd_accumulate_momentum_tiles_supported(*op.seg["pshape"])):
                            tiled.append(op)
            if not tiled:
                ops.sgd_momentum_payload(f["params"], f["momentum"], acc, gs.gathered, self.net["lr"], self._momentum, scale)
            else:
                at = 0   # the flat buffer in order: a tiled layer's own pass, one plain pass per run of other layers in between
                for op in sorted(tiled, key=lambda o: o.seg["start"]) + [None]:
                    s = f["total"] if op is None else op.seg["start"]
                    if s > at:
                        ops.sgd_momentum_payload(f["params"][at:s], f["momentum"][at:s], None if acc is None else acc[at:s], gs.gathered[at:s],
                                                 self.net["lr"], self._momentum, scale)
                    if op is not None:
                        n = op.seg["nw"] + op.seg["nb"]
                        ops.sgd_momentum_payload_tiles(f["params"][s:s + n], f["momentum"][s:s + n], None if acc is None else acc[s:s + n],
                                                       gs.gathered[s:s + n], tuple(op.seg["pshape"]), self.net["lr"], self._momentum, scale,
                                                       op.seg["wt16"], op.seg["wtd16"])
                        fresh.add(op.name)
                        # the next plain run starts at the segment's aligned end, not at s + n: the gap is padding nobody's gradient
                        # touches, and a run that started inside it would lose the 16-byte alignment of its bf16 payload pointer
                        # and fall back to the scalar kernel without a word
                        at = op.seg["end"]
        else:
            ops.sgd_momentum(f["params"], f["momentum"], f["accum"], self.net["lr"], self._momentum, scale)
        self._w16_seen = None  # the master weights moved: the bf16 images are refreshed by the next forward
        self._tiles_fresh, self._tiles_fresh_ver = fresh, f["params"]._version
        self._step += 1

    def eval_loss(self, images, labels, keep_prob=0.5, perms=None, drop_masks=None):
        """sess.run(loss["total"], feed) of deeplab.py:274: a forward + E-step + CE + L2, no gradients."""
        self.forward(images, keep_prob, drop_masks)
        self.run_estep(labels, perms)
        self._ce(want_grad=False)
        l2 = None
        for op in self._plan:
            if op.kind == "conv":
                t = ops.l2_loss(op.w_pad.reshape(-1))  # padding entries are exactly zero
                l2 = t if l2 is None else l2 + t
        self.loss["l2"] = l2
        self.loss["total"] = self.loss["norm"] + self._weight_decay * l2
        return float(self.loss["total"])

    # ------------------------------------------------------------------------------------------
    # training loop (deeplab.py:210-285)
    # ------------------------------------------------------------------------------------------
    def train(self, base_lr, weight_decay, momentum, batch_size, epoches, max_iterations=None, log=print):
        """deeplab.py:210-285.  In a data-parallel job (torch.distributed initialised, one process per GPU) every rank
        runs this loop on its own shard: `batch_size` is per rank, an epoch is data_len // (batch_size * world)
        iterations, the data source hands each rank its slice of every global batch (data.py), rank 0 alone writes
        checkpoints and logs, and all ranks meet at a barrier after each save."""
        assert self.data is not None, "data is None"
        rank, world = dist_rank_world(self.config)
        if rank != 0:
            log = lambda *a, **k: None  # noqa: E731
        # (config "start_epoch": the epoch a resumed run continues in; None = behind the epochs this data object has handed out)
        train_iter = self.data.next_batch(category="train", batch_size=batch_size, epoches=-1,
                                          start_epoch=self.config.get("start_epoch", None))
        self.config.setdefault("batch_size", batch_size)
        self.build()
        self.pre_train(base_lr, weight_decay, momentum, batch_size,
                       save_layers=["input", "output", "label", "pred", "is_training", "drop_probe"])
        if self.config.get("model_path", False) is not False:
            log("start to load model: %s" % self.config.get("model_path"))
            self.restore_from_model(self.saver["norm"], self.config.get("model_path"), checkpoint=False)
            log("model loaded ...")
        start_time = time.time()
        log("start_time: %f" % start_time)
        log("config -- lr:%f weight_decay:%f momentum:%f batch_size:%f epoches:%f" % (
            base_lr, weight_decay, momentum, batch_size, epoches))
        epoch, i = 0.0, 0
        if "fused_update" not in self.config:
            self._fused = True   # (takes effect where accum_num == 1 and there is no gradient exchange: backward())
        iterations_per_epoch_train = max(self.data.get_data_len() // (batch_size * world), 1)
        saver_dir = self.config.get("saver_path", "saver")

        def save(which, name, step):
            # never write a checkpoint behind a recorded device failure (the optimiser kernels have been skipping updates since it was
            # raised; in a data-parallel job every rank's word is raised by then -- emadapt_status_collective -- so every rank raises here)
            ops.status_poll(clear=True, raise_on_error=True)
            path = self.saver[which].save(None, os.path.join(saver_dir, name), global_step=step)
            if world > 1 and torch.distributed.is_available() and torch.distributed.is_initialized():
                torch.distributed.barrier()   # (rank / world given by the config alone: nothing to meet at)
            return path

        while epoch < epoches and (max_iterations is None or i < max_iterations):
            if i == 0:
                self.net["lr"] = base_lr
            for mult, new_lr in ((10, 1e-4), (20, 1e-5), (30, 1e-6)):  # deeplab.py:245-262
                if i == mult * iterations_per_epoch_train:
                    log("save model before new_lr:%f" % new_lr)
                    save("lr", "lr-%f" % base_lr, i)
                    self.net["lr"] = new_lr
                    base_lr = new_lr
            batch = next(train_iter)   # (images, labels) or the dataset class's (images, labels, ids)
            data_x, data_y = batch[0], batch[1]
            self.net["accum_gradient_accum"](data_x, data_y, 0.5)
            if i % self.accum_num == self.accum_num - 1:
                self.net["accum_gradient_update"]()
                self.net["accum_gradient_clean"]()
            if i % 500 == 10:
                loss = self.eval_loss(data_x, data_y, 0.5)
                log("epoch:%f, iteration:%f, lr:%f, loss:%f" % (epoch, i, self.net["lr"], loss))
                # once per logging interval (the loop synchronises here anyway): a failure a kernel recorded in the device status
                # word (a stream-K wait that ran out: the optimiser kernels have been skipping their updates since) raises
                # EmadaptDeviceError, and a loss that is no longer finite stops the run -- TF's session.run would have raised
                ops.status_poll(clear=True, raise_on_error=True)
                if not np.isfinite(loss):
                    raise FloatingPointError("loss is %r at iteration %d (lr %g)" % (loss, i, self.net["lr"]))
            if i % 6000 == 5999:
                save("norm", "norm", i)
            i += 1
            epoch = i / iterations_per_epoch_train
        torch.cuda.synchronize(self.device)
        ops.status_poll(clear=True, raise_on_error=True)   # (whether or not anything is saved)
        if self.config.get("save_final", True):
            save("norm", "norm", i)
        end_time = time.time()
        log("end_time:%f" % end_time)
        log("duration time:%f" % (end_time - start_time))
        return i
