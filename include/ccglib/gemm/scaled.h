// Forwarding header: ccglib::mma::ScaledGEMM is defined in <ccglib/b200_api.hpp>.
#pragma once
#include <ccglib/b200_api.hpp>
