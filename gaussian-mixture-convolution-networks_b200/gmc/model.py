"""The GMCN classifier: per layer convolution -> 1/Cin -> ReLU fit -> normalisation, then integrate -> BatchNorm1d
(-> MLP) -> log_softmax. Counterpart of the reference's src/gmc/model.py (Layer, Config, Net)."""
import time
import typing

import torch
from torch import Tensor
import torch.nn as nn
import torch.nn.functional as F

import gmc.classification
import gmc.mixture as gm
import gmc.modules


class Layer:
    def __init__(self, n_feature_maps, kernel_radius, n_convolution_fittiong_components, n_fitting_components):
        self.n_feature_layers = n_feature_maps
        self.kernel_radius = kernel_radius
        self.n_convolution_fittiong_components = n_convolution_fittiong_components
        self.n_fitting_components = n_fitting_components


class Config:
    BN_CONSTANT_COMPUTATION_ZERO = 0
    BN_CONSTANT_COMPUTATION_MEAN_IN_CONST = 1
    BN_CONSTANT_COMPUTATION_INTEGRAL = 2
    BN_CONSTANT_COMPUTATION_WEIGHTED = 3

    BIAS_TYPE_NONE = 0
    BIAS_TYPE_NORMAL = 1
    BIAS_TYPE_NEGATIVE_SOFTPLUS = 2

    BN_TYPE_STD = "Std"
    BN_TYPE_COVARIANCE = "Cov"
    BN_TYPE_COVARIANCE_STD = "CovStd"

    BN_PLACE_NOWHERE = "None"
    BN_PLACE_AFTER_GMC = "aCn"
    BN_PLACE_AFTER_RELU = "aRl"

    def __init__(self, n_dims):
        self.n_dims = n_dims
        self.n_classes = 10
        self.n_kernel_components = 5
        self.layers: typing.List[Layer] = [Layer(8, 1, 32, 32), Layer(16, 1, 16, 16), Layer(10, 1, 8, 8)]
        self.bias_type = Config.BIAS_TYPE_NONE
        self.mlp: typing.Optional[typing.List[int]] = None
        self.bn_place = Config.BN_PLACE_AFTER_RELU
        self.bn_type = Config.BN_TYPE_COVARIANCE
        self.dropout = 0.0
        self.relu_config: gmc.modules.ReLUFittingConfig = gmc.modules.ReLUFittingConfig()
        self.convolution_config: gmc.modules.ConvolutionConfig = gmc.modules.ConvolutionConfig()

    def produce_gmc_layers_description(self) -> str:
        name = "L"
        for l in self.layers:
            fit = ""
            if isinstance(l.n_fitting_components, (list, tuple)):
                fit = "-" + "-".join(str(x) for x in l.n_fitting_components)
            elif l.n_fitting_components > 0:
                fit = f"-{l.n_fitting_components}"
            name = f"{name}_{l.n_feature_layers}f_{int(l.kernel_radius * 10)}r_{int(l.n_convolution_fittiong_components)}{fit}c"
        return name

    def produce_description(self):
        mlp = "" if self.mlp is None else "_MLP" + "".join(f"_{l}" for l in self.mlp)
        return f"BN{self.bn_place}{self.bn_type}_Drp{int(self.dropout * 100)}_nK{self.n_kernel_components}_" \
               f"{self.produce_gmc_layers_description()}{mlp}_"


class Net(nn.Module):
    def __init__(self, learn_positions: bool = True, learn_covariances: bool = True, config: Config = Config):
        super(Net, self).__init__()
        self.config = config
        bias_0 = -0.1 if config.bias_type == Config.BIAS_TYPE_NEGATIVE_SOFTPLUS else 0.0

        self.norm0 = nn.Sequential(gmc.modules.CovScaleNorm(1, batch_norm=False), gmc.modules.BatchNorm(1, batch_norm=False))
        self.biases = torch.nn.ParameterList()
        self.gmcs = torch.nn.modules.ModuleList()
        self.relus = torch.nn.modules.ModuleList()
        self.norms = torch.nn.modules.ModuleList()
        self.dropout = gmc.modules.Dropout(config.dropout)

        n_in = 1
        for i, l in enumerate(config.layers):
            self.gmcs.append(gmc.modules.Convolution(
                config.convolution_config, n_layers_in=n_in, n_layers_out=l.n_feature_layers,
                n_kernel_components=config.n_kernel_components, position_range=l.kernel_radius,
                covariance_range=(l.kernel_radius / 3) ** 2, learn_positions=learn_positions,
                learn_covariances=learn_covariances, weight_sd=1.0, weight_mean=0.1, n_dims=config.n_dims,
                n_fitting_components=l.n_convolution_fittiong_components))
            self.biases.append(torch.nn.Parameter(torch.zeros(1, l.n_feature_layers) + bias_0))
            self.relus.append(gmc.modules.ReLUFitting(config.relu_config, n_layers=l.n_feature_layers,
                                                      n_output_gaussians=l.n_fitting_components, convolution_layer=f"{i}"))
            if config.bn_type == Config.BN_TYPE_COVARIANCE_STD:
                norm = nn.Sequential(gmc.modules.CovScaleNorm(n_layers=l.n_feature_layers),
                                     gmc.modules.BatchNorm(n_layers=l.n_feature_layers))
            elif config.bn_type == Config.BN_TYPE_COVARIANCE:
                norm = gmc.modules.CovScaleNorm(n_layers=l.n_feature_layers)
            elif config.bn_type == Config.BN_TYPE_STD:
                norm = gmc.modules.BatchNorm(n_layers=l.n_feature_layers)
            else:
                norm = nn.Module()
            self.norms.append(norm)
            n_in = l.n_feature_layers

        self.normX = nn.BatchNorm1d(num_features=n_in)
        if config.mlp is not None:
            mlp = []
            for l in config.mlp:
                if l == -1:
                    mlp.append(nn.Dropout(p=0.5))
                else:
                    mlp += [nn.Linear(n_in, l), nn.ReLU(), nn.BatchNorm1d(l)]
                    n_in = l
            self.mlp = nn.Sequential(*mlp)
        else:
            self.mlp = None
        self.timings = dict()
        self.last_time = time.time()

    def reset_timer(self):
        self.last_time = time.perf_counter()

    def time_lap(self, name: str):
        now = time.perf_counter()
        self.timings[name] = now - self.last_time
        self.last_time = now

    def set_position_learning(self, flag: bool):
        for g in self.gmcs:
            g.learn_positions = flag

    def set_covariance_learning(self, flag: bool):
        for g in self.gmcs:
            g.learn_covariances = flag

    def matrix_parameters(self) -> typing.List[torch.nn.Parameter]:
        """The parameters that mix features, as gmc.optimisation.Muon takes them: the kernel weights of the convolutions
        ([n_out, n_in, n_kernel_components, 1], a matrix of n_out rows) and the matrices of the head's linear layers. Kernel
        positions, covariance factors, normalisations and biases are not matrices of this kind: give them to another
        optimiser."""
        return ([g.weights for g in self.gmcs]
                + ([m.weight for m in self.mlp if isinstance(m, nn.Linear)] if self.mlp is not None else []))

    def weight_decay_loss(self) -> Tensor:
        loss = torch.zeros(1, device=next(self.parameters()).device, dtype=torch.float)
        for g in self.gmcs:
            loss = loss + g.weight_decay_loss()
        return loss

    def _fused_inference_layers(self, in_x: Tensor) -> bool:
        """True when a layer can run as convolution fit + one fused kernel (weight division, ReLU fixed-point fit,
        covariance-scale normalisation): evaluation mode without autograd, no bias, fixed-point-only ReLU fit,
        covariance normalisation after the ReLU, and a fitted convolution. Anything else takes the general path."""
        cfg = self.config
        return (not self.training and not torch.is_grad_enabled() and in_x.is_cuda and in_x.dtype == torch.float32
                and cfg.bias_type == Config.BIAS_TYPE_NONE and cfg.bn_place == Config.BN_PLACE_AFTER_RELU
                and cfg.bn_type == Config.BN_TYPE_COVARIANCE
                and cfg.relu_config.fitting_method is gmc.fitting.fixed_point_only
                and all(isinstance(n, gmc.modules.CovScaleNorm) and n.batch_norm for n in self.norms)
                and all(g.n_fitting_components > 0 for g in self.gmcs)
                and all(0 < g.n_fitting_components <= gmc.fitting.FUSED_FIXED_POINT_MAX_COMPONENTS for g in self.gmcs))

    def _input_normalisation(self, in_x: Tensor) -> Tensor:
        """norm0 on the inference path: one kernel when it is the pair of per-sample normalisations on one channel that
        this class builds (a replaced norm0, e.g. one that replays stored values, is called as it is)."""
        n0 = self.norm0
        if (isinstance(n0, nn.Sequential) and len(n0) == 2 and isinstance(n0[0], gmc.modules.CovScaleNorm)
                and isinstance(n0[1], gmc.modules.BatchNorm) and not n0[0].batch_norm and not n0[1].batch_norm
                and gm.n_layers(in_x) == 1 and gm.n_components(in_x) <= 2048):
            return gmc.modules.fused_input_normalisation(in_x, n0[1].learnable_scaling)[0]
        return self.norm0((in_x, None))[0]

    def _features_inference(self, in_x: Tensor) -> Tensor:
        """The layer stack of features() for the case _fused_inference_layers() describes: per layer the two
        convolution-fit kernels and one fused kernel; same values as the general path."""
        import gmc.cpp.extensions.convolution_fitting.binding as cpp_convolution_fitting
        x = self._input_normalisation(in_x)
        for i in range(len(self.config.layers)):
            n_in = gm.n_layers(x)
            conv = self.gmcs[i]
            fitted = cpp_convolution_fitting.forward(x.contiguous(), conv.kernels(), conv.n_fitting_components)[0]
            # the convolved constant is dropped (no bias: the constant restarts at zero, as in the general path)
            x, _ = gmc.fitting.fused_relu_layer(fitted, None, float(n_in), self.norms[i].inference_scale(gm.n_dimensions(x)))
        return gm.integrate(x)

    def features(self, in_x: Tensor, tensorboard=None) -> Tensor:
        """Everything up to and including the integration of the last layer: [n_batch, n_feature_maps]."""
        if tensorboard is None and self._fused_inference_layers(in_x):
            return self._features_inference(in_x)
        x, x_const = self.norm0((in_x, None))
        n_batch = gm.n_batch(x)
        for i in range(len(self.config.layers)):
            if gm.n_layers(x) > 8:
                x, x_const = self.dropout((x, x_const))
            n_in = gm.n_layers(x)
            x, x_const = self.gmcs[i](x, x_const)
            x = gm.pack_mixture(gm.weights(x) / n_in, gm.positions(x), gm.covariances(x))
            x_const = x_const / n_in
            if self.config.bn_place == Config.BN_PLACE_AFTER_GMC:
                x, x_const = self.norms[i]((x, torch.zeros_like(x_const)))
            if self.config.bias_type == Config.BIAS_TYPE_NEGATIVE_SOFTPLUS:
                x_const = x_const - F.softplus(self.biases[i], beta=20)
            elif self.config.bias_type == Config.BIAS_TYPE_NORMAL:
                x_const = x_const + self.biases[i]
            else:
                assert self.config.bias_type == Config.BIAS_TYPE_NONE
                x_const = torch.zeros(n_batch, gm.n_layers(x), device=in_x.device)
            self.reset_timer()
            x, x_const = self.relus[i](x, x_const, tensorboard)
            self.time_lap(f"relu{i}")
            if self.config.bn_place == Config.BN_PLACE_AFTER_RELU:
                x, x_const = self.norms[i]((x, x_const))
        return gm.integrate(x)

    def logits(self, in_x: Tensor, tensorboard=None) -> Tensor:
        """The class scores [n_batch, n_classes] that forward() normalises."""
        x = self.normX(self.features(in_x, tensorboard))
        if self.mlp is not None:
            x = self.mlp(x)
        return x

    def forward(self, in_x: Tensor, tensorboard=None) -> Tensor:
        return F.log_softmax(self.logits(in_x, tensorboard), dim=1).view(in_x.shape[0], self.config.n_classes)

    def log_probabilities(self, in_x: Tensor, targets: typing.Optional[Tensor] = None, n_top: int = 0,
                          temperature: float = 1.0) -> gmc.classification.LogProbabilities:
        """Log-probability of each sample's target class, entropy of its distribution and its n_top likeliest classes in
        one pass (gmc.classification.log_probabilities). -result.target.mean() is the loss that nll_loss(forward(x), targets)
        computes."""
        return gmc.classification.log_probabilities(self.logits(in_x), targets, n_top, temperature)
