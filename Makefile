# Builds the MI355X (gfx950) shared library behind include/sv2n.h (the
# oracle is Python and needs no build).  `python -c "import __graft_entry__ as g; g.build()"`
# runs the same recipe.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH ?= gfx950
HIPFLAGS ?= -O3 -std=c++17 -fPIC --offload-arch=$(ARCH) -Iinclude -Wall -Wno-unused-result
# no packed fp32 instructions (v_pk_*_f32): the compiler forms them from plain
# float code, and some of their forms are not reliable on this hardware
HIPFLAGS += -Xclang -target-feature -Xclang -packed-fp32-ops
BUILD ?= build
# EXTRA: extra compiler flags for diagnostic A/B builds (into their own BUILD / LIB)
HIPFLAGS += $(EXTRA)
LIB ?= spotv2net_amd/libsv2n.so
ifeq ($(STAMPS),1)
HIPFLAGS += -DSV2N_STAMPS   # diagnostic phase stamps (tools/stamps.py)
endif
# diagnostic bound checks (SV2N_CHK, sv2n_check_hits): make CHECK=1 builds
# build_check/ -> spotv2net_amd/libsv2n_check.so; tests load it with
# SV2N_LIB=spotv2net_amd/libsv2n_check.so (tools/measure.sh check)
ifeq ($(CHECK),1)
HIPFLAGS += -DSV2N_CHECK
BUILD = build_check
LIB = spotv2net_amd/libsv2n_check.so
endif
SRC := $(wildcard spotv2net_amd/csrc/*.hip)
OBJ := $(patsubst spotv2net_amd/csrc/%.hip,$(BUILD)/%.o,$(SRC))

# the operators whose host side is C++ (host code only; the C++ compiler torch's
# headers and libraries were built for)
TORCH_LIB ?= spotv2net_amd/libsv2n_torch.so
PYTHON ?= python3
TORCH_DIR = $(shell $(PYTHON) -c "import importlib.util as u; print(u.find_spec('torch').submodule_search_locations[0])")
ROCM ?= /opt/rocm
CXX = g++
CXXFLAGS ?= -O2 -std=c++17 -fPIC -Wall

all: $(LIB) $(TORCH_LIB)

$(TORCH_LIB): spotv2net_amd/csrc/sv2n_torch.cpp include/sv2n.h
	$(CXX) $(CXXFLAGS) -D__HIP_PLATFORM_AMD__=1 -DUSE_ROCM -Iinclude -isystem $(TORCH_DIR)/include \
	  -isystem $(TORCH_DIR)/include/torch/csrc/api/include -isystem $(ROCM)/include -shared -o $@ $< \
	  -L$(TORCH_DIR)/lib -ltorch -ltorch_cpu -lc10 -lc10_hip

$(BUILD)/%.o: spotv2net_amd/csrc/%.hip $(wildcard spotv2net_amd/csrc/*.h) include/sv2n.h
	@mkdir -p $(BUILD)
	$(HIPCC) $(HIPFLAGS) -c $< -o $@

$(LIB): $(OBJ)
	$(HIPCC) $(HIPFLAGS) -shared -o $@ $(OBJ)

clean:
	rm -rf build $(LIB) $(TORCH_LIB)

.PHONY: all clean
