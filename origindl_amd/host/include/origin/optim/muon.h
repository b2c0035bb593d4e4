// The Muon optimizer; everything lives in origin/nn.h.
#pragma once
#include "origin/nn.h"
